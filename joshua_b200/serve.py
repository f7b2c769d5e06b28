"""Serves a batch of requests behind one long prompt, on random weights: the paged cache, its attention, the rotary table and the
sampler together.

    python -m joshua_b200.serve --batch 32 --prompt 2000 --tokens 64 --kv q8_0 [--layers 8] [--yarn 4] [--own-prompts]

Prints what the cache takes and the time of a step; with --own-prompts every sequence reads the prompt for itself.
"""
from __future__ import annotations

import argparse
import time

import torch

from .llama import LlamaConfig
from .paged import PagedLlamaDecoder
from .rope import Rope, rope_table


def run(batch: int, prompt: int, tokens: int, kv: str, layers: int, yarn: float = 1.0, own_prompts: bool = False, cfg=None) -> dict:
    cfg = cfg or LlamaConfig(layers=layers)
    dev = torch.device("cuda", 0)
    max_ctx = prompt + tokens + 1
    scaled = dict(scaling="yarn", factor=yarn, orig_ctx=max(1, int(max_ctx / yarn))) if yarn > 1 else {}
    rope = Rope(rope_table(cfg.rope_theta, cfg.head_dim, max_ctx, dev, **scaled))
    dec = PagedLlamaDecoder(cfg, dev, batch=batch, max_ctx=max_ctx, kv_type=kv, rope=rope)
    gen = torch.Generator(device=dev).manual_seed(1)
    ids = torch.randint(0, cfg.vocab, (prompt,), generator=torch.Generator().manual_seed(2)).tolist()
    dec.sampling = dict(temperature=torch.full((batch,), 0.8, device=dev), top_p=torch.full((batch,), 0.95, device=dev),
                        top_k=torch.full((batch,), 100, dtype=torch.int32, device=dev))
    dec.uniform.uniform_(generator=gen)
    if own_prompts:
        for i in range(batch):
            dec.prefill(ids, sequence=i)
    else:
        dec.share_prompt(ids)
    for i in range(batch):
        dec.reserve(i, max_ctx)
    out, steps = [dec.token.clone()], []
    for _ in range(tokens - 1):
        dec.uniform.uniform_(generator=gen)
        torch.cuda.synchronize()
        t = time.perf_counter()
        dec.step()
        torch.cuda.synchronize()
        steps.append(time.perf_counter() - t)
        out.append(dec.token.clone())
    dec.check_flags()
    used = dec.n_pages - len(dec.free)
    return {"tokens": torch.stack(out, 1).cpu(), "ms_per_step": 1e3 * sorted(steps)[len(steps) // 2] if steps else 0.0,
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
    a = ap.parse_args()
    r = run(a.batch, a.prompt, a.tokens, a.kv, a.layers, a.yarn, a.own_prompts)
    print(f"{a.batch} sequences behind {a.prompt} tokens, {a.kv} cache: {r['pages_used']} pages, {r['cache_mib']:.0f} MiB; "
          f"{r['ms_per_step']:.2f} ms a step, {1e3 * a.batch / max(r['ms_per_step'], 1e-9):.0f} tokens/s")


if __name__ == "__main__":
    main()
