"""The decoders over the paged cache: against themselves in other orders of work, and against the dense decoder.

Tolerances.  The same cache contents reached another way (shared or own pages, prompt or single steps) leave the matmuls' and the
attention's own f32-level differences, at most some 1e-6 of an activation per layer and 1e-4 of a logit's size at the end (the
bound of this repository's fused-against-separate tests is 1e-3).  Against the dense f32 cache, a cache of halves rounds keys and
values by 2^-11: a score by 2^-11 of itself, 2^-8 with the scores of these inputs (below 8), and so the attention's output;
two layers: 2^-6 of the logits' spread.
"""
import numpy as np
import pytest

from joshua_b200 import synth
from joshua_b200._lib import JoshuaB200Error

pytestmark = pytest.mark.gpu


def config(**more):
    from joshua_b200.llama import LlamaConfig

    return LlamaConfig(**{**dict(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, ffn=2048, vocab=2048), **more})


def make(batch, kv="q8_0", max_ctx=320, cfg=None, **more):
    import torch

    from joshua_b200.paged import PagedLlamaDecoder

    return PagedLlamaDecoder(cfg or config(), torch.device("cuda", 0), batch=batch, max_ctx=max_ctx, kv_type=kv, wtype=synth.Q8_0, seed=3, **more)


def ids(n, seed=0):
    return np.random.RandomState(seed).randint(0, 2048, n).tolist()


def near(a, b, tol=1e-4):
    a, b = (np.asarray(x.cpu().numpy(), dtype=np.float64) for x in (a, b))
    assert np.abs(a - b).max() <= tol * np.abs(b).max(), np.abs(a - b).max() / np.abs(b).max()


@pytest.mark.parametrize("kv", ["f16", "q8_0", "q4_0"])
def test_a_shared_prompt_is_every_sequences_own(kv):
    import torch

    prompt = ids(150)
    shared, own = make(5, kv), make(5, kv)
    shared.share_prompt(prompt)
    assert shared.shared_pages == 2 and len(shared.free) == own.n_pages - 2 - 5
    for i in range(5):
        own.prefill(prompt, sequence=i)
    near(shared.logits, own.logits)
    follow = torch.tensor([[7, 100, 2000, 5, 90], [1, 2, 3, 4, 5], [900, 800, 700, 600, 500]], dtype=torch.int32, device="cuda")
    for row in follow:
        for dec in (shared, own):
            dec.token.copy_(row)
            dec.step()
        near(shared.logits, own.logits)
    assert shared.pos.tolist() == own.pos.tolist() == [153] * 5
    shared.check_flags(), own.check_flags()


def test_a_prompt_in_one_pass_and_token_by_token():
    prompt = ids(70, 1)
    whole, steps, parts = make(1), make(1), make(1)
    whole.prefill(prompt)
    for t in prompt:
        steps.force_token(t)
        steps.step()
    parts.prefill(prompt[:30])
    parts.prefill(prompt[30:])
    # a step rounds rows that differ in their last bits: now and then a code moves by one of 127
    near(steps.logits, whole.logits, 2e-2)
    near(parts.logits, whole.logits, 2e-2)
    assert whole.pos.tolist() == steps.pos.tolist() == parts.pos.tolist() == [70]


@pytest.mark.parametrize("qk_norm", [False, True])
def test_halves_against_the_dense_cache(qk_norm):
    import torch

    from joshua_b200.llama import LlamaDecoder

    prompt = ids(100, 2)
    dense = LlamaDecoder(config(), torch.device("cuda", 0), batch=1, max_ctx=320, wtype=synth.Q8_0, seed=3, qk_norm=qk_norm)
    paged = make(1, "f16", qk_norm=qk_norm)
    for dec in (dense, paged):
        dec.prefill(prompt)
    near(paged.logits, dense.logits, 2.0**-6)
    for t in ids(5, 3):
        for dec in (dense, paged):
            dec.force_token(t)
            dec.step()
        near(paged.logits, dense.logits, 2.0**-6)


def test_sequences_of_their_own_lengths_in_a_graph():
    import torch

    prompts = [ids(n, n) for n in (5, 64, 130)]
    dec, alone = make(3), [make(1) for _ in range(3)]
    for i, p in enumerate(prompts):
        dec.prefill(p, sequence=i)
        alone[i].prefill(p)
        dec.reserve(i, 200)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dec.step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            dec.step()
        graph.replay()
        side.synchronize()
    for i in range(3):
        alone[i].step(), alone[i].step()
        near(dec.logits[i], alone[i].logits[0], 2e-2)
    assert dec.pos.tolist() == [len(p) + 2 for p in prompts]


def test_sampling_penalty_and_greedy_rows():
    import torch

    dec = make(4)
    dec.sampling = dict(temperature=torch.tensor([0.0, 0.7, 1.0, 0.0], device="cuda"), top_k=torch.tensor([0, 20, 5, 0], dtype=torch.int32, device="cuda"))
    dec.uniform.copy_(torch.tensor([0.1, 0.2, 0.3, 0.4]))
    dec.share_prompt(ids(90, 4))
    best = dec.logits[0].argmax()
    assert dec.token[0] == best and dec.token[3] == best and dec.pos.tolist() == [90] * 4
    top = dec.logits[0].topk(20).indices.tolist()
    assert int(dec.token[1]) in top and int(dec.token[2]) in top[:5]
    dec.repetition_penalty = 1.3
    dec.seed_window(ids(90, 4))
    dec.step()
    assert dec.window_state[:, 0].tolist() == [64] * 4


def test_pages_come_and_go():
    dec = make(2, max_ctx=256, n_pages=5)
    dec.prefill(ids(130), sequence=0)
    with pytest.raises(JoshuaB200Error):
        dec.prefill(ids(130), sequence=1)   # three pages wanted, two are free
    dec.release(0)
    assert len(dec.free) == 5
    dec.prefill(ids(130), sequence=1)
    with pytest.raises(JoshuaB200Error):
        dec.reserve(1, 257)
    with pytest.raises(JoshuaB200Error):
        dec.share_prompt(ids(10))
    dec.reset()
    dec.share_prompt(ids(64))
    assert dec.shared_pages == 1 and len(dec.free) == 4
    dec.release(0)
    assert len(dec.free) == 4               # sequence 1 still has the common page
    dec.release(1)
    assert len(dec.free) == 5


def test_routed_experts_over_pages():
    import torch

    from joshua_b200.moe_decoder import MoeDecoder, MoeDecoderConfig
    from joshua_b200.paged import PagedMoeDecoder

    cfg = MoeDecoderConfig(layers=2, hidden=512, q_heads=4, kv_heads=2, head_dim=128, vocab=1024, n_expert=8, n_used=2, moe_inter=256)
    dense = MoeDecoder(cfg, torch.device("cuda", 0), batch=2, max_ctx=128, seed=1)
    paged = PagedMoeDecoder(cfg, torch.device("cuda", 0), batch=2, max_ctx=128, seed=1, kv_type="f16")
    for t in (3, 900, 17):
        for dec in (dense, paged):
            dec.force_token(t)
            dec.step()
    near(paged.logits, dense.logits, 2.0**-6)


def test_the_example_runs():
    from joshua_b200 import serve

    a = serve.run(3, 100, 4, "q8_0", 2, cfg=config())
    b = serve.run(3, 100, 4, "q8_0", 2, cfg=config(), own_prompts=True)
    assert a["tokens"].shape == (3, 4) and a["pages_used"] < b["pages_used"]
    assert serve.run(2, 40, 3, "q4_0", 2, yarn=4.0, cfg=config())["tokens"].shape == (2, 3)
