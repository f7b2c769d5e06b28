"""Several sequences' next tokens in one pass, attention windows and scores of the decoders over the paged cache, against the same tokens
taken another way and against a CPU attention over what the caches hold.

Tolerance: passes of other row counts take other routes of the linears, of which that of a row or two (int8 planes) is held to 7e-5 of
max(|value|, 1) by its own tests.  Nine linears follow one another here (two layers of four, the head): 9 * 7e-5 = 6.3e-4 if every
error were carried on whole; the attentions' (2e-5 of a value each) bring it to 6.7e-4, below 1e-3 of a logit's size.
  Where the cache itself was filled by other routes, its codes may differ by a step: a value off by 7e-5 of its size rounds to the next code
where it lies that near a border, a share of 2 * 7e-5 * 127 = 1.8% of the codes in eight bits.  A step is 1/127 of the block's largest, so
values are off by sqrt(0.018) / 127 = 1.1e-3 of it in the mean square, keys and so scores alike; two layers of both: 4.4e-3, below 2^-6
(halves: steps of 2^-11, less).
"""
import torch
import numpy as np
import pytest

from joshua_b200._lib import JoshuaB200Error
from tests.test_gpu_paged_decoder import ids, make
from tests.test_gpu_paged_decoder import near as near_by

pytestmark = pytest.mark.gpu


FILLED_OTHERWISE = 2.0**-6


def near(a, b, tol=1e-3):
    near_by(a, b, tol)


@pytest.mark.parametrize("kv", ["f16", "q8_0", "q4_0"])
@pytest.mark.parametrize("qk_norm", [False, True])
def test_extend_is_prefill(kv, qk_norm):
    a, b = make(4, kv, qk_norm=qk_norm), make(4, kv, qk_norm=qk_norm)
    prompts = {0: ids(70, 1), 2: ids(1, 2), 3: ids(131, 3)}
    a.extend(prompts)
    for i, p in prompts.items():
        b.prefill(p, sequence=i)
    rows = list(prompts)
    near(a.logits[rows], b.logits[rows])
    assert a.pos[rows].tolist() == b.pos[rows].tolist() == [70, 1, 131] and a.token[rows].tolist() == b.token[rows].tolist()
    assert a.held == b.held and [len(o) for o in a.owned] == [len(o) for o in b.owned]
    # parts of prompts behind earlier ones, of other sequences, one token of another
    more = {0: ids(40, 4), 1: ids(65, 5), 2: ids(3, 6), 3: ids(1, 7)}
    a.extend(more)
    for i, p in more.items():
        b.prefill(p, sequence=i)
    near(a.logits, b.logits)
    for _ in range(3):
        b.token.copy_(a.token)
        a.step(), b.step()
        near(a.logits, b.logits)
    a.check_flags(), b.check_flags()


def test_extend_is_steps_after_one_another():
    a, b = make(2), make(2)
    prompt, tail = ids(100, 1), ids(9, 2)
    a.extend({0: prompt, 1: prompt[:50]}), b.extend({0: prompt, 1: prompt[:50]})
    a.extend({0: tail})
    for t in tail:
        b.extend({0: [t]})
    near(a.logits[0], b.logits[0])
    assert a.pos.tolist() == b.pos.tolist() == [109, 50]
    a.check_flags()


def test_scores():
    """Log probabilities of a prompt's tokens: the same whether it is read in one pass or token by token, and sums to one."""
    import torch

    from joshua_b200.sampling import log_probs

    dec, steps = make(3), make(3)
    dec.score_rows = 32   # several slices
    prompt, other = ids(80, 1), ids(2, 2)
    got = dec.extend({0: prompt, 1: other, 2: [5]}, scores=7)
    assert sorted(got) == [0, 1, 2] and [len(g[0]) for g in got.values()] == [79, 1, 0]
    assert [list(t.shape) for t in got[0]] == [[79], [79], [79, 7], [79, 7]] and [list(t.shape) for t in got[2]] == [[0], [0], [0, 7], [0, 7]]
    for k in range(len(prompt) - 1):
        steps.extend({0: [prompt[k]]})
        lp, entropy, top, top_lp = log_probs(steps.logits[:1], torch.tensor([prompt[k + 1]], dtype=torch.int32, device="cuda"), top=7)
        # logits differ by 1e-3 of their size, log probabilities by twice that
        spread = 2e-3 * float(steps.logits[0].abs().max())
        assert abs(float(lp) - float(got[0][0][k])) <= spread and abs(float(entropy) - float(got[0][1][k])) <= 8 * spread
        assert float((top_lp[0] - got[0][3][k]).abs().max()) <= spread
    near(dec.logits[0], (steps.extend({0: [prompt[-1]]}), steps.logits[0])[1])
    assert dec.extend({1: [3, 4]}, scores=0)[1][2].shape == (1, 0)


@pytest.mark.parametrize("kv", ["f16", "q8_0"])
@pytest.mark.parametrize("window,sinks", [(64, 0), (100, 4), (30, 70), (1, 1), (400, 3)])
def test_a_window_by_parts_by_steps_and_in_one_pass(kv, window, sinks):
    """The same tokens read in one pass, in parts and token by token, with pages given back on the way."""
    more = dict(kv=kv, max_ctx=400, attention_window=window, attention_sinks=sinks)
    once, parts, single = make(2, **more), make(2, **more), make(2, **more)
    parts.prompt_rows = 37
    prompt = ids(250, 9)
    once.prefill(prompt, sequence=1), parts.prefill(prompt, sequence=1)
    near(once.logits[1], parts.logits[1], FILLED_OTHERWISE)
    single.prefill(prompt[:200], sequence=1)
    for t in prompt[200:]:
        single.extend({1: [t]})
    near(once.logits[1], single.logits[1], FILLED_OTHERWISE)
    for dec in (once, parts, single):
        dec.prefill(prompt[:90], sequence=0)
    for step in range(70):
        for dec in (parts, single):
            dec.token.copy_(once.token)
        for dec in (once, parts, single):
            dec.step()
        near(once.logits, parts.logits, FILLED_OTHERWISE), near(once.logits, single.logits, FILLED_OTHERWISE)
    sink_pages = -(-sinks // 64)
    for dec in (once, parts, single):
        dec.check_flags()
        live = [sum(p is not None for p in o) for o in dec.owned]
        for i, n in enumerate(live):
            assert n <= min(-(-dec.held[i] // 64), sink_pages + (window - 1) // 64 + 2), (live, dec.held)
        assert len(dec.free) == dec.n_pages - sum(live)
        table = dec.table.cpu().numpy()
        for i, o in enumerate(dec.owned):
            assert table[i, :len(o)].tolist() == [-1 if p is None else p for p in o]


def test_a_wide_window_is_none():
    a, b = make(2, attention_window=320), make(2)
    prompt = ids(150, 1)
    a.prefill(prompt), b.prefill(prompt)
    a.prefill(prompt[:20], sequence=1), b.prefill(prompt[:20], sequence=1)
    near(a.logits, b.logits)
    for _ in range(5):
        b.token.copy_(a.token)
        a.step(), b.step()
        near(a.logits, b.logits)


def test_a_long_prompt_through_a_small_pool():
    """A prompt of more pages than the pool has, in parts; one that does not fit is refused whole."""
    dec = make(2, max_ctx=2000, n_pages=6, attention_window=100, attention_sinks=4)
    dec.prompt_rows = 120
    dec.prefill(ids(1500, 3), sequence=1)
    assert dec.held == [0, 1500]
    wide = make(2, max_ctx=2000, attention_window=100, attention_sinks=4)
    wide.prompt_rows = 120
    wide.prefill(ids(1500, 3), sequence=1)
    near(dec.logits[1], wide.logits[1])
    free, table = list(dec.free), dec.table.clone()
    dec.prompt_rows = 512
    with pytest.raises(JoshuaB200Error):
        dec.prefill(ids(450, 4), sequence=1)
    assert dec.held == [0, 1500] and dec.free == free and bool((dec.table == table).all())
    dec.release(1)
    assert sorted(dec.free) == list(range(6))
    dec.reset()
    assert sorted(dec.free) == list(range(6)) and dec.kept_from == [0, 0]


def test_a_shared_prompt_behind_a_window():
    shared, own = (make(3, attention_window=80, attention_sinks=2) for _ in range(2))
    prompt = ids(200, 5)
    shared.share_prompt(prompt)
    for i in range(3):
        own.prefill(prompt, sequence=i)
    near(shared.logits, own.logits)
    for _ in range(80):
        own.token.copy_(shared.token)
        shared.step(), own.step()
        near(shared.logits, own.logits)
    for i in range(3):
        shared.release(i)
    assert sorted(shared.free) == list(range(shared.n_pages))
    shared.check_flags()


def test_a_captured_step_with_a_window():
    """A caller's graph, its pages reserved, between host steps and parts of prompts; the host call too."""
    import torch

    more = dict(attention_window=70, attention_sinks=3)
    a, b = make(2, **more), make(2, **more)
    for dec in (a, b):
        dec.extend({0: ids(100, 1), 1: ids(30, 2)})
    a.reserve(0, 200), a.reserve(1, 200)
    a.step(), b.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.step()
    for _ in range(60):
        g.replay()
        b.step()
    near(a.logits, b.logits)
    assert a.pos.tolist() == b.pos.tolist()
    for dec in (a, b):
        dec.extend({1: ids(10, 3)})
    near(a.logits, b.logits)
    for _ in range(3):
        a.step(), b.step()
    near(a.logits, b.logits)
    a.check_flags()
    tokens = b.token.cpu()
    out = a.forward_host(tokens)
    b.token.copy_(tokens)
    b.step()
    near(torch.as_tensor(out), b.logits)


def test_routed_experts():
    import torch

    from joshua_b200.moe_decoder import MoeDecoderConfig
    from joshua_b200.paged import PagedMoeDecoder

    cfg = MoeDecoderConfig(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, n_expert=8, n_used=2, moe_inter=256, vocab=2048)
    a, b = (PagedMoeDecoder(cfg, torch.device("cuda", 0), batch=2, max_ctx=320, kv_type="q8_0", seed=1) for _ in range(2))
    a.extend({0: ids(40, 1), 1: ids(33, 2)})
    b.prefill(ids(40, 1), sequence=0), b.prefill(ids(33, 2), sequence=1)
    near(a.logits, b.logits, tol=2.0**-6)   # batches of other sizes round differently, and experts in a near tie may change places


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_drafts_that_are_not_taken(window, sinks):
    a, b = (make(2, "f16", attention_window=window, attention_sinks=sinks) for _ in range(2))
    for dec in (a, b):
        dec.extend({0: ids(100, 1), 1: ids(61, 2)})
    scores = a.extend({0: ids(6, 3), 1: ids(4, 4)}, scores=1)   # the second sequence's pass a page's end
    assert scores[0][0].shape == (5,) and a.pos.tolist() == [106, 65]
    a.rewind(0, 102), a.rewind(1, 62)
    assert a.pos.tolist() == a.held == [102, 62]
    b.extend({0: ids(6, 3)[:2], 1: ids(4, 4)[:1]})
    for dec in (a, b):
        dec.extend({0: ids(3, 5), 1: ids(70, 6)})
    near(a.logits, b.logits)
    assert a.pos.tolist() == b.pos.tolist() == [105, 132]
    a.rewind(0, 104)
    a.token[0] = ids(3, 5)[2]
    b.token.copy_(a.token)
    a.rewind(1, 131), b.rewind(1, 131)
    a.step()                       # the same token again, by a step
    b.rewind(0, 104), b.step()
    near(a.logits, b.logits)
    a.check_flags(), b.check_flags()


def test_where_there_is_no_way_back():
    dec = make(3)
    dec.share_prompt(ids(150, 1))                      # two common pages and 22 positions
    dec.extend({0: ids(5, 2)})
    dec.rewind(0, 151), dec.rewind(0, 128)
    for n in (127, 64, 0, -1, 129):                    # 129: no longer held
        with pytest.raises(JoshuaB200Error):
            dec.rewind(0, n)
    with pytest.raises(JoshuaB200Error):
        dec.rewind(3, 10)
    win = make(1, attention_window=64, n_pages=4)
    for part in range(5):
        win.extend({0: ids(50, part)})
    win.extend({0: [1]})                               # position 250; what is in front of 187 is gone, page 0 and 1 with it
    win.rewind(0, 200)
    with pytest.raises(JoshuaB200Error):
        win.rewind(0, 150)
    assert win.held == [200]
    win.extend({0: ids(9, 9)})
    win.check_flags(), dec.check_flags()


def test_refusals():
    dec = make(2)
    for bad in ({}, {0: []}, {0: [1], 1: []}):
        with pytest.raises(JoshuaB200Error):
            dec.extend(bad)
    for bad in ({2: [1]}, {-1: [1]}):
        with pytest.raises(JoshuaB200Error):
            dec.extend(bad)
    with pytest.raises(JoshuaB200Error):
        dec.extend({0: [1, 2]}, scores=33)
    with pytest.raises(JoshuaB200Error):
        dec.extend({0: ids(321)})
    with pytest.raises(JoshuaB200Error):
        dec.extend({0: ids(20), 1: ids(400)})
    assert dec.held == [0, 0] and len(dec.free) == dec.n_pages
    for more in (dict(attention_window=-1), dict(attention_sinks=4), dict(attention_window=5, attention_sinks=-1)):
        with pytest.raises(JoshuaB200Error):
            make(1, **more)


def test_serving_a_batch():
    """The command's run: a prompt of every sequence's own in one pass with its scores, windows, log probabilities of what is sampled."""
    from joshua_b200.llama import LlamaConfig
    from joshua_b200.serve import run

    cfg = LlamaConfig(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, ffn=2048, vocab=2048)
    more = dict(batch=3, prompt=150, tokens=70, kv="q8_0", layers=2, cfg=cfg)
    plain, scored = run(**more), run(**more, logprobs=5)
    assert bool((plain["tokens"] == scored["tokens"]).all()) and plain["log_probs"] is None
    lp = scored["log_probs"]
    assert list(lp.shape) == [3, 70] and bool((lp <= 0).all()) and bool(lp.isfinite().all())
    own = run(**more, own_prompts=True, logprobs=0)
    assert own["prompt_log_prob"] < 0 and list(own["tokens"].shape) == [3, 70]
    windowed = run(**more, window=64, sinks=2, logprobs=1)
    assert windowed["pages_used"] < plain["pages_used"] + 6 and bool(windowed["log_probs"].isfinite().all())
