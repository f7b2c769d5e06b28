"""Serves a batch of requests behind one long prompt, on random weights: the paged cache, its attention, the rotary table and the
sampler together.

    python -m joshua_b200.serve --batch 32 --prompt 2000 --tokens 64 --kv q8_0 [--layers 8] [--yarn 4] [--own-prompts]
        [--window 1024 --sinks 4] [--logprobs 5]

Prints what the cache takes and the time of a step.  With --own-prompts every sequence reads the prompt for itself; with --window a token
sees so many positions back, and the first --sinks; with --logprobs every sampled token's log probability comes with that many others, and
prompts of the sequences' own go through the model several at a time, their log probabilities printed.
"""
from __future__ import annotations

import argparse
import time

import torch

from .llama import LlamaConfig
from .paged import PagedLlamaDecoder
from .rope import Rope, rope_table
from .sampling import log_probs

PASS_ROWS = 16384   # prompt tokens of several sequences in one pass


def score_prompts(dec, ids: list, alternatives: int) -> dict:
    """Reads one prompt into every sequence, several at a time, one longer than PASS_ROWS in parts; by sequence, what `sampling.log_probs`
    gives for its tokens but the first."""
    scores: dict = {}
    some = max(1, PASS_ROWS // len(ids))
    for i in range(0, dec.batch, some):
        sequences = range(i, min(dec.batch, i + some))
        for at in range(0, len(ids), PASS_ROWS):
            part = ids[at:at + PASS_ROWS]
            if at:   # its first token, by the logits that the part before it has left
                first = torch.tensor(part[:1], dtype=torch.int32, device=dec.dev)
                for k in sequences:
                    scores[k].append(log_probs(dec.logits[k:k + 1], first, top=alternatives))
            for k, got in dec.extend({k: part for k in sequences}, scores=alternatives).items():
                scores.setdefault(k, []).append(got)
    return {k: tuple(torch.cat(t) for t in zip(*parts)) for k, parts in scores.items()}


def run(batch: int, prompt: int, tokens: int, kv: str, layers: int, yarn: float = 1.0, own_prompts: bool = False, cfg=None, window: int = 0,
        sinks: int = 0, logprobs: int | None = None) -> dict:
    cfg = cfg or LlamaConfig(layers=layers)
    dev = torch.device("cuda", 0)
    max_ctx = prompt + tokens + 1
    scaled = dict(scaling="yarn", factor=yarn, orig_ctx=max(1, int(max_ctx / yarn))) if yarn > 1 else {}
    rope = Rope(rope_table(cfg.rope_theta, cfg.head_dim, max_ctx, dev, **scaled))
    dec = PagedLlamaDecoder(cfg, dev, batch=batch, max_ctx=max_ctx, kv_type=kv, rope=rope, attention_window=window,
                            attention_sinks=sinks)
    gen = torch.Generator(device=dev).manual_seed(1)
    ids = torch.randint(0, cfg.vocab, (prompt,), generator=torch.Generator().manual_seed(2)).tolist()
    dec.sampling = dict(temperature=torch.full((batch,), 0.8, device=dev), top_p=torch.full((batch,), 0.95, device=dev),
                        top_k=torch.full((batch,), 100, dtype=torch.int32, device=dev))
    dec.uniform.uniform_(generator=gen)
    scores = {}
    if own_prompts and logprobs is None:
        for i in range(batch):
            dec.prefill(ids, sequence=i)
    elif own_prompts:
        scores = score_prompts(dec, ids, logprobs)
    else:
        dec.share_prompt(ids)
    if not window:   # steps take a page now and then otherwise, and give one back
        for i in range(batch):
            dec.reserve(i, max_ctx)

    def score():
        return log_probs(dec.logits, dec.token, top=logprobs)[0].clone() if logprobs is not None else None

    out, given, steps = [dec.token.clone()], [score()], []
    for _ in range(tokens - 1):
        dec.uniform.uniform_(generator=gen)
        torch.cuda.synchronize()
        t = time.perf_counter()
        dec.step()
        given.append(score())
        torch.cuda.synchronize()
        steps.append(time.perf_counter() - t)
        out.append(dec.token.clone())
    dec.check_flags()
    used = dec.n_pages - len(dec.free)
    return {"tokens": torch.stack(out, 1).cpu(), "ms_per_step": 1e3 * sorted(steps)[len(steps) // 2] if steps else 0.0,
            "log_probs": torch.stack(given, 1).cpu() if logprobs is not None else None,
            "prompt_log_prob": float(scores[0][0].mean()) if scores else None,
            "pages_used": used, "cache_mib": used * dec.layers[0]["cache"].page_bytes * cfg.layers / 2**20}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=2000)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--kv", default="q8_0", choices=("f16", "q8_0", "q4_0"))
    ap.add_argument("--layers", type=int, default=8)
    ap.add_argument("--yarn", type=float, default=1.0, help="stretch the positions by this factor")
    ap.add_argument("--own-prompts", action="store_true")
    ap.add_argument("--window", type=int, default=0, help="positions that a token sees (0: all)")
    ap.add_argument("--sinks", type=int, default=0, help="first positions that stay visible behind the window")
    ap.add_argument("--logprobs", type=int, default=None, help="log probabilities of the tokens, with so many others")
    a = ap.parse_args()
    r = run(a.batch, a.prompt, a.tokens, a.kv, a.layers, a.yarn, a.own_prompts, window=a.window, sinks=a.sinks, logprobs=a.logprobs)
    print(f"{a.batch} sequences behind {a.prompt} tokens, {a.kv} cache: {r['pages_used']} pages, {r['cache_mib']:.0f} MiB; "
          f"{r['ms_per_step']:.2f} ms a step, {1e3 * a.batch / max(r['ms_per_step'], 1e-9):.0f} tokens/s")
    if r["log_probs"] is not None:
        print(f"mean log probability of a sampled token {float(r['log_probs'].mean()):.3f}"
              + (f", of the prompt's {r['prompt_log_prob']:.3f}" if r["prompt_log_prob"] is not None else ""))


if __name__ == "__main__":
    main()
