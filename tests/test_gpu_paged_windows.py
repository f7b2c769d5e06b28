"""Prompts behind attention windows whose pages go back while they are read."""
import pytest

from joshua_b200._lib import JoshuaB200Error
from tests.test_gpu_paged_decoder import ids, make
from tests.test_gpu_paged_extend import near

pytestmark = pytest.mark.gpu


def windowed(batch, n_pages=None):
    dec = make(batch, max_ctx=2000, n_pages=n_pages, attention_window=100, attention_sinks=4)
    dec.prompt_rows = 120
    return dec


@pytest.mark.parametrize("n,pages", [(1500, 8), (1536, 6), (30, 3)])   # ends within a page, at a page's end, in the first one
def test_a_long_shared_prompt_through_a_small_pool(n, pages):
    small, wide = windowed(3, pages), windowed(3)
    for dec in (small, wide):
        dec.share_prompt(ids(n, 3))
        assert dec.held == [n] * 3
    near(small.logits, wide.logits)
    for _ in range(2):
        wide.token.copy_(small.token)
        if n == 1500:
            small.step(), wide.step()
            near(small.logits, wide.logits)
    for i in range(3):
        small.release(i)
    assert sorted(small.free) == list(range(pages))
    small.check_flags(), wide.check_flags()


def test_one_that_does_not_fit_is_refused_whole():
    dec = windowed(3, 6)
    for bad in (1500, 1996, 2001):    # one page too few for the others' ends; past max_ctx
        free, table = list(dec.free), dec.table.clone()
        with pytest.raises(JoshuaB200Error):
            dec.share_prompt(ids(bad, 3))
        assert dec.held == [0] * 3 and dec.free == free and bool((dec.table == table).all()) and dec.owned == [[], [], []]
    dec.share_prompt(ids(1472, 3))    # a page's end: nothing is copied
    assert dec.held == [1472] * 3
    dec.check_flags()


def test_reserved_pages_go_back_for_the_common_ones():
    dec = windowed(3, 9)
    dec.reserve(1, 128), dec.reserve(2, 64)
    dec.share_prompt(ids(1472, 3))
    assert dec.held == [1472] * 3 and dec.owned[1] == dec.owned[2] == dec.owned[0]
    for i in range(3):
        dec.release(i)
    assert sorted(dec.free) == list(range(9))
    dec.check_flags()


@pytest.mark.parametrize("window", [0, 100])
def test_one_scratch_for_all_layers_of_a_pass(window):
    import torch

    from tests.test_gpu_paged_decoder import config

    dec = make(2, cfg=config(layers=6), attention_window=window)
    need = dec.layers[0]["cache"].scratch_bytes(2, 8, rows=200)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    dec.extend({0: ids(150, 1), 1: ids(50, 2)}), dec.prefill(ids(90, 3)), dec.step()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before < 2 * need   # 20 MB; of every layer's own, six times that
    dec.check_flags()


def test_ids_from_the_host_and_the_device():
    import torch

    a, b = make(3), make(3)
    prompts = {0: ids(70, 1), 1: ids(5, 2), 2: ids(33, 3)}
    want = a.extend(prompts, scores=2)
    got = b.extend({0: torch.tensor(prompts[0], device="cuda"), 1: prompts[1], 2: torch.tensor(prompts[2])}, scores=2)
    assert bool((a.logits == b.logits).all()) and a.held == b.held == [70, 5, 33]
    assert all(bool((x == y).all()) for i in want for x, y in zip(want[i], got[i]))


def test_the_serving_command_gives_pages_back():
    """The pages that a run behind a window holds at its end: those of the sinks and of the window, fewer than without one."""
    from joshua_b200.llama import LlamaConfig
    from joshua_b200.serve import run

    cfg = LlamaConfig(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, ffn=2048, vocab=2048)
    more = dict(batch=3, prompt=500, tokens=200, kv="q8_0", layers=2, cfg=cfg)
    plain = run(**more)
    assert plain["pages_used"] == 7 + 3 * 4        # 448 positions in common, reserved up to 701
    for window, sinks in ((64, 2), (130, 0)):
        used = run(**more, window=window, sinks=sinks)["pages_used"]
        # a step has made room for itself before it takes its page
        assert used <= 3 * (-(-sinks // 64) + (window - 1) // 64 + 2) < plain["pages_used"]


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("rows", [150, 64, 40, 7])
def test_scores_of_a_prompt_in_parts(monkeypatch, window, rows):
    """The serving command's prompts that are longer than a pass: what is scored does not depend on the parts, but for the rounding of
    passes of other row counts (tests/test_gpu_paged_extend.py derives 2^-6 of a logit's size where the cache was filled otherwise): log
    probabilities are off by twice that."""
    from joshua_b200 import serve

    once, parts = (make(3, attention_window=window) for _ in range(2))
    prompt = ids(150, 1)
    want = serve.score_prompts(once, prompt, 2)
    monkeypatch.setattr(serve, "PASS_ROWS", rows)
    got = serve.score_prompts(parts, prompt, 2)
    assert parts.held == once.held == [150] * 3 and sorted(got) == [0, 1, 2]
    spread = 2 * 2.0**-6 * float(once.logits.abs().max())
    for i in range(3):
        assert [list(t.shape) for t in got[i]] == [[149], [149], [149, 2], [149, 2]]
        assert float((got[i][0] - want[i][0]).abs().max()) <= spread and float((got[i][3] - want[i][3]).abs().max()) <= spread
