"""Attention of chunks of new tokens over the paged cache, a sliding window with sinks, and log probabilities, as cases whose time is
measured.

Families (`what` of a case):

  chunk   some new tokens of each sequence (a part of a prompt, a draft to check, a decode step beside a prompt) over what the cache
          holds of it, the new tokens included, each token up to its own position (`PagedCache.attend_chunk`).
  window  one new token of every sequence over its last `window` positions and the first `sinks` ones (`PagedCache.attend`).  Pages
          that no token sees any more are not in the table.
  score   log probability of a given token of every row of logits, the entropy of the row, the likeliest tokens (`log_probs`).

A page holds 64 positions of every kv head.  In memory a head's part of a page is keys, scales of keys, values, scales of values;
the order inside is that of the matrix instructions that read it, spelt out in `_decode` below.

Head counts and sizes are those of the decoders of this repository (32 / 8 and 32 / 4 heads of 128, 64-wide ones of its tests,
vocabularies of 128256, 151936 and 32000), lengths and batches generic.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 64
BITS = {"f16": 16, "q8_0": 8, "q4_0": 4}
HEADS = [(32, 8), (32, 4), (8, 8), (16, 2), (24, 8), (14, 2), (32, 32)]
VOCABS = [128256, 151936, 32000]


def listed():
    return [
        # the next 512 tokens of a prompt behind its first 3584
        {"name": "chunk_q8_512", "what": "chunk", "kind": "q8_0", "hd": 128, "n_q": 32, "n_kv": 8, "batch": 1, "rows": 512, "split": "even", "ctx": 4096, "window": 0, "sinks": 0},
        # four short prompts from their beginning, together
        {"name": "chunk_f16_4x500", "what": "chunk", "kind": "f16", "hd": 64, "n_q": 32, "n_kv": 8, "batch": 4, "rows": 2000, "split": "even", "ctx": 500, "window": 0, "sinks": 0},
        # a draft of four tokens of every sequence of a batch, to be checked
        {"name": "chunk_q8_b32_draft", "what": "chunk", "kind": "q8_0", "hd": 128, "n_q": 32, "n_kv": 8, "batch": 32, "rows": 128, "split": "even", "ctx": 4000, "window": 0, "sinks": 0},
        # a decode step of 23 sequences with a part of another one's prompt beside it, four bits
        {"name": "chunk_q4_b24_mixed", "what": "chunk", "kind": "q4_0", "hd": 128, "n_q": 32, "n_kv": 4, "batch": 24, "rows": 700, "split": "mixed", "ctx": 8000, "window": 0, "sinks": 0},
        # a long part of a prompt, the largest call
        {"name": "chunk_q8_4096", "what": "chunk", "kind": "q8_0", "hd": 128, "n_q": 32, "n_kv": 8, "batch": 1, "rows": 4096, "split": "even", "ctx": 12288, "window": 0, "sinks": 0},
        # parts of unlike prompts of a model whose layers see 1024 positions back and four sinks
        {"name": "chunk_q8_window", "what": "chunk", "kind": "q8_0", "hd": 128, "n_q": 32, "n_kv": 4, "batch": 3, "rows": 1999, "split": "ragged", "ctx": 9001, "window": 1024, "sinks": 4},
        # one user far behind the beginning: latency
        {"name": "window_q8_b1", "what": "window", "kind": "q8_0", "hd": 128, "n_q": 32, "n_kv": 8, "batch": 1, "ctx": 30000, "window": 1024, "sinks": 4},
        # a full batch, a long window
        {"name": "window_q8_b64", "what": "window", "kind": "q8_0", "hd": 128, "n_q": 32, "n_kv": 8, "batch": 64, "ctx": 32768, "window": 4096, "sinks": 16},
        # a large batch of 64-wide heads, a window that no page begins with
        {"name": "window_f16_b128", "what": "window", "kind": "f16", "hd": 64, "n_q": 32, "n_kv": 8, "batch": 128, "ctx": 5000, "window": 700, "sinks": 100},
        # a sampled token's probability and five others, one user
        {"name": "score_b1", "what": "score", "rows": 1, "vocab": 128256, "top": 5, "peak": 6.0},
        # the same of a batch, as many others as a server offers
        {"name": "score_b64", "what": "score", "rows": 64, "vocab": 151936, "top": 20, "peak": 3.0},
        # the tokens of a prompt
        {"name": "score_prompt", "what": "score", "rows": 1000, "vocab": 128256, "top": 0, "peak": 5.0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(["chunk", "chunk", "chunk", "window", "window", "score"])
    if what == "score":
        vocab = rng.choice(VOCABS) - rng.randrange(0, 500)
        return {"what": what, "rows": _log_int(rng, 1, 1000 * 128256 // vocab), "vocab": vocab, "top": rng.choice([0, 1, 5, 8, 20, 32]),
                "peak": rng.uniform(1.0, 8.0)}
    hd, kind, (n_q, n_kv) = rng.choice([64, 128, 128]), rng.choice(sorted(BITS)), rng.choice(HEADS)
    bounded = what == "window" or rng.random() < 0.4
    window, sinks = (_log_int(rng, 1, 4096), rng.choice([0, 0, 1, 4, rng.randrange(1, 200)])) if bounded else (0, 0)
    if what == "window":
        batch, hd = _log_int(rng, 1, 128), rng.choice([64, 128, 256])
        most = 2.0**28 / (batch * n_kv * hd)  # positions a sequence, so that the largest listed one stays it
        window = min(window, int(most))
        return {"what": what, "kind": kind, "hd": hd, "n_q": n_q, "n_kv": n_kv, "batch": batch, "ctx": _log_int(rng, 1, 32768), "window": window,
                "sinks": sinks}
    batch = _log_int(rng, 1, 32)
    split = rng.choice(["even", "ragged", "mixed"])
    rows = _log_int(rng, batch, 4096)
    if split == "even":
        rows = max(1, rows // batch) * batch
    longest = max(_counts(split, batch, rows))
    most = 2.0**37 / (rows * n_q * hd)  # positions, so that the largest listed one stays it
    ctx = _log_int(rng, longest, max(longest, min(16384, int(most))))
    return {"what": what, "kind": kind, "hd": hd, "n_q": n_q, "n_kv": n_kv, "batch": batch, "rows": rows, "split": split, "ctx": ctx,
            "window": window, "sinks": sinks}


# ── the cache's pages ───────────────────────────────────────────────────
# Orders inside a head's part of a page.  Axes of position (a: 16-position groups; h: upper half of a group; r8, c: eighths and
# pairs within a half; e: one of a pair) and of dimension (b: 32-wide blocks; s: halves of a fragment; u, m: rest).
def _orders(kind, hd):
    """(shape of the key codes, axes order to [position, dimension]), the same of the values."""
    a, b = PAGE // 16, hd // 32
    if kind == "f16":
        return (((a, b, 2, 8, 4, 2, 4), (0, 5, 3, 1, 4, 2, 6)), ((a, b, 2, 8, 4, 2, 2, 2), (0, 5, 4, 7, 1, 3, 2, 6)))
    if kind == "q8_0":
        return (((a, b, 8, 4, 2, 8), (0, 4, 2, 1, 3, 5)), ((a, b, 8, 4, 2, 2, 2, 2), (0, 5, 3, 7, 1, 2, 4, 6)))
    # the last axis of both: low and high half of a byte
    return (((a, b // 2, 8, 4, 2, 2, 2, 2, 2), (0, 7, 2, 1, 4, 3, 5, 8, 6)),
            ((a, b // 2, 8, 4, 2, 2, 2, 2, 2), (0, 7, 3, 6, 1, 4, 2, 5, 8)))


def _sizes(kind, hd):
    """Bytes of a head's codes in a page (keys or values) and of their scales."""
    return PAGE * hd * BITS[kind] // 8, 0 if kind == "f16" else PAGE * (hd // 32) * 2


def _decode(pages, kind, hd):
    """uint8 [..., bytes of a head in a page] -> keys, values f32 [..., PAGE, hd]."""
    lead, (nc, ns), at, out = pages.shape[:-1], _sizes(kind, hd), 0, []
    for shape, order in _orders(kind, hd):
        raw = pages[..., at:at + nc]
        if kind == "f16":
            v = raw.contiguous().view(torch.float16).float()
        elif kind == "q8_0":
            v = raw.float() - 128.0
        else:
            v = torch.stack((raw & 15, raw >> 4), dim=-1).float() - 8.0
        n = len(lead)
        v = v.reshape(*lead, *shape).permute(*range(n), *(n + i for i in order)).reshape(*lead, PAGE, hd)
        at += nc
        if ns:
            d = pages[..., at:at + ns].contiguous().view(torch.float16).float().reshape(*lead, 2, 8, hd // 32, 4)
            d = d.permute(*range(n), n, n + 3, n + 1, n + 2).reshape(*lead, PAGE, hd // 32)
            v = (v.reshape(*lead, PAGE, hd // 32, 32) * d.unsqueeze(-1)).reshape(*lead, PAGE, hd)
            at += ns
        out.append(v)
    return out


def _quantise(x, kind):
    """f32 [..., hd] -> (codes, scales) of blocks of 32, or halves and None."""
    if kind == "f16":
        return x.clamp(-65504.0, 65504.0).half(), None
    x = x.reshape(*x.shape[:-1], -1, 32)
    if kind == "q8_0":
        d = (x.abs().amax(-1) * (1.0 / 127.0)).clamp(max=65504.0).half()
    else:
        hi, lo = x.amax(-1), x.amin(-1)
        d = (torch.where(hi > -lo, hi, lo) * -0.125).clamp(-65504.0, 65504.0).half()
    f = d.float()
    inv = torch.where(f != 0, 1.0 / f, torch.zeros_like(f))
    c = (x * inv.unsqueeze(-1)).round()
    c = c.clamp(-127, 127) + 128 if kind == "q8_0" else (c + 8).clamp(0, 15)
    return c.to(torch.uint8).reshape(*x.shape[:-2], -1), d


def _encode(k, v, kind, hd):
    """f32 [..., PAGE, hd] twice -> uint8 [..., bytes of a head in a page]."""
    lead, parts = k.shape[:-2], []
    for x, (shape, order) in zip((k, v), _orders(kind, hd)):
        c, d = _quantise(x, kind)
        n, back = len(lead), [0] * len(order)
        for i, o in enumerate(order):
            back[o] = i
        c = c.reshape(*lead, *(shape[o] for o in order)).permute(*range(n), *(n + i for i in back))
        if kind == "q4_0":
            c = c[..., 0] | (c[..., 1] << 4)
        parts.append(c.contiguous().reshape(*lead, -1).view(torch.uint8))
        if d is not None:
            d = d.reshape(*lead, 2, 4, 8, hd // 32).permute(*range(n), n, n + 2, n + 3, n + 1)
            parts.append(d.contiguous().reshape(*lead, -1).view(torch.uint8))
    return torch.cat(parts, dim=-1)


def _pages(kind, hd, n_kv, count, gen, dev):
    """Pages of N(0, 1) keys and values, some dimensions larger, as keys of trained models have them."""
    wide = torch.ones(n_kv, 1, hd, device=dev)
    wide[:, :, :: 32] = 4.0
    nc, ns = _sizes(kind, hd)
    pages = torch.empty(count, n_kv, 2 * (nc + ns), dtype=torch.uint8, device=dev)
    step = max(1, 2**25 // (n_kv * PAGE * hd))
    for i in range(0, count, step):
        n = min(step, count - i)
        k = torch.randn(n, n_kv, PAGE, hd, device=dev, generator=gen) * wide
        v = torch.randn(n, n_kv, PAGE, hd, device=dev, generator=gen)
        pages[i:i + n] = _encode(k, v, kind, hd)
    return pages


# ── inputs ──────────────────────────────────────────────────────────────
def _counts(split, batch, rows):
    """New tokens of each sequence: as many of all, one of all but the first, or some of each."""
    if split == "even":
        return [rows // batch] * batch
    if split == "mixed":
        return [rows - (batch - 1)] + [1] * (batch - 1)
    cuts = sorted(np.random.RandomState(31 * rows + batch).randint(0, rows - batch + 1, size=batch - 1).tolist())
    return [b - a + 1 for a, b in zip([0] + cuts, cuts + [rows - batch])]


def _spans(case):
    """(new tokens, positions with them) of every sequence: the longest has `ctx`, others less, of none less than its tokens."""
    if case["what"] == "window":
        counts = [1] * case["batch"]
    else:
        counts = _counts(case["split"], case["batch"], case["rows"])
    rng = np.random.RandomState((1009 * case["ctx"] + 7 * case["batch"] + sum(counts)) % 2**32)
    lens = [n + int((case["ctx"] - n) * u) for n, u in zip(counts, rng.uniform(size=len(counts)))]
    lens[int(np.argmax(counts))] = case["ctx"]
    return counts, lens


def _seen_pages(count, length, window, sinks):
    """Numbers of the pages of a sequence that its new tokens see."""
    pages = np.arange(-(-length // PAGE))
    if not window:
        return pages
    return pages[(pages * PAGE < sinks) | ((pages + 1) * PAGE > length - count + 1 - window)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    what = case["what"]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    if what == "score":
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab) * 2.5
        some = torch.randint(0, vocab, (rows, 20), device=dev, generator=gen)
        logits.scatter_add_(1, some, normal(rows, 20).abs() * case["peak"])
        token = torch.where(torch.rand(rows, device=dev, generator=gen) < 0.7, some[:, 0], torch.randint(0, vocab, (rows,), device=dev, generator=gen))
        return {"case": case, "logits": logits, "token": token.int()}
    kind, hd, n_q, n_kv = case["kind"], case["hd"], case["n_q"], case["n_kv"]
    counts, lens = _spans(case)
    seen = [_seen_pages(n, length, case["window"], case["sinks"]) for n, length in zip(counts, lens)]
    total = sum(len(p) for p in seen)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).int().numpy()
    table = np.full((len(lens), -(-case["ctx"] // PAGE)), -1, dtype=np.int32)
    at = 0
    for i, p in enumerate(seen):
        table[i, p] = order[at:at + len(p)]
        at += len(p)
    state = {"case": case, "q": normal(sum(counts), n_q * hd), "pages": _pages(kind, hd, n_kv, total, gen, dev),
             "table": torch.from_numpy(table).to(dev), "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "counts": counts, "spans": lens}
    if what == "chunk" and case["split"] != "even":  # where each sequence's rows begin; even ones need no telling
        state["first"] = torch.tensor([0, *np.cumsum(counts).tolist()], dtype=torch.int32, device=dev)
    return state


# ── one pass ────────────────────────────────────────────────────────────
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    case = state["case"]
    if case["what"] == "score":
        from joshua_b200.sampling import log_probs

        return log_probs(state["logits"], state["token"], top=case["top"])
    if "cache" not in state:  # what a program builds once around its pages
        from joshua_b200.kv_cache import PagedCache

        state["cache"] = PagedCache(case["kind"], case["n_kv"], case["hd"], pages=state["pages"])
    cache, q, lens, table = state["cache"], state["q"], state["lens"], state["table"]
    if case["what"] == "window":
        return cache.attend(q, lens, table, n_q=case["n_q"], window=case["window"], sinks=case["sinks"])
    return cache.attend_chunk(q, lens, table, n_q=case["n_q"], first=state.get("first"), window=case["window"], sinks=case["sinks"])


def _softmax(s):
    e = (s - s.amax(-1, keepdim=True)).exp()
    return e / e.sum(-1, keepdim=True)


def _run_plain(state):
    what = state["case"]["what"]
    return {"score": _plain_score, "window": _plain_window, "chunk": _plain_chunk}[what](state)


def _plain_chunk(state):
    case = state["case"]
    kind, hd, n_q, n_kv, window, sinks = (case[n] for n in ("kind", "hd", "n_q", "n_kv", "window", "sinks"))
    dev, g, out, row = state["q"].device, n_q // n_kv, torch.empty_like(state["q"]), 0
    for i, (n, length) in enumerate(zip(state["counts"], state["spans"])):
        seen = torch.from_numpy(_seen_pages(n, length, window, sinks)).to(dev)
        t = (seen[:, None] * PAGE + torch.arange(PAGE, device=dev)).reshape(-1)
        pos = torch.arange(length - n, length, device=dev)
        hidden = t[None, :] > pos[:, None]
        if window:
            hidden |= (pos[:, None] - t[None, :] >= window) & (t[None, :] >= sinks)
        held = state["pages"][state["table"][i, seen].long()]
        q = state["q"][row:row + n].reshape(n, n_kv, g, hd) / math.sqrt(hd)
        for h in range(n_kv):  # one at a time: the scores of all heads are many
            k, v = (x.reshape(-1, hd) for x in _decode(held[:, h], kind, hd))
            s = torch.matmul(q[:, h].reshape(n * g, hd), k.t()).reshape(n, g, -1)
            s = s.masked_fill_(hidden[:, None, :], float("-inf"))
            o = torch.matmul(_softmax(s).reshape(n * g, -1), v)
            out[row:row + n].view(n, n_kv, g * hd)[:, h] = o.reshape(n, g * hd)
        row += n
    return out


def _plain_window(state):
    case = state["case"]
    kind, hd, n_q, n_kv, batch = case["kind"], case["hd"], case["n_q"], case["n_kv"], case["batch"]
    window, sinks = case["window"], case["sinks"]
    lens, dev = state["lens"].long(), state["q"].device
    # the pages seen, those of the sinks first, as many a sequence as any may need
    full, low = (lens + PAGE - 1) // PAGE, (lens - window).clamp(min=0) // PAGE
    head = torch.minimum(low, torch.tensor(-(-sinks // PAGE), device=dev))
    j = torch.arange(min(-(-case["ctx"] // PAGE), -(-sinks // PAGE) + (window - 1) // PAGE + 2), device=dev)[None, :]
    number = torch.where(j < head[:, None], j, j - head[:, None] + low[:, None])
    there = number < full[:, None]
    held = state["table"].long().gather(1, torch.where(there, number, 0)).clamp(min=0)
    t = (number[:, :, None] * PAGE + torch.arange(PAGE, device=dev)).reshape(batch, -1)
    visible = (t < lens[:, None]) & ((t >= lens[:, None] - window) | (t < sinks))
    q = state["q"].reshape(batch, n_kv, n_q // n_kv, hd) / math.sqrt(hd)
    out = torch.empty_like(q)
    step = max(1, 2**27 // (held.shape[1] * PAGE * n_kv * hd))
    for i in range(0, batch, step):  # some sequences at a time: their keys in 32 bits are many
        k, v = (x.transpose(1, 2).reshape(x.shape[0], n_kv, -1, hd) for x in _decode(state["pages"][held[i:i + step]], kind, hd))
        s = torch.matmul(q[i:i + step], k.transpose(-1, -2))
        s = torch.where(visible[i:i + step, None, None, :], s, float("-inf"))
        out[i:i + step] = torch.matmul(_softmax(s), v)
    return out.reshape(batch, -1)


def _plain_score(state):
    l, n = state["logits"], state["case"]["top"]
    d = l - l.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    logs = d - total.log()
    entropy = total.log().reshape(-1) - (e * d).sum(-1) / total.reshape(-1)
    given = logs.gather(1, state["token"].long()[:, None]).reshape(-1)
    if not n:
        return given, entropy, torch.empty(l.shape[0], 0, dtype=torch.int32, device=l.device), l.new_empty(l.shape[0], 0)
    best = l.sort(dim=-1, descending=True, stable=True).indices[:, :n]
    return given, entropy, best.int(), logs.gather(1, best)


# ── how much of it there is, and what it is exactly ─────────────────────
def work(case):
    if case["what"] == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    kind, hd, n_q, n_kv, window, sinks = (case[n] for n in ("kind", "hd", "n_q", "n_kv", "window", "sinks"))
    held = 2 * n_kv * sum(_sizes(kind, hd)) // PAGE  # bytes of a position
    pairs = positions = 0
    counts, lens = _spans(case)
    for n, length in zip(counts, lens):
        p = np.arange(length - n, length, dtype=np.int64)
        low = np.maximum(p + 1 - window, 0) if window else np.zeros_like(p)
        pairs += int((p + 1 - low + np.minimum(low, sinks)).sum())
        positions += length - int(low[0]) + min(int(low[0]), sinks)
    return {"bytes": positions * held + 8 * sum(counts) * n_q * hd, "flops": 4 * pairs * n_q * hd}


def _exact_values(pages, kind, hd):
    """Values of pages [count, n_kv, bytes] in 64 bits, place by place: keys, values [n_kv, positions, hd]."""
    pos, dim = np.meshgrid(np.arange(PAGE), np.arange(hd), indexing="ij")
    a, h, r, b, d, nb = pos // 16, pos % 16 // 8, pos % 8, dim // 32, dim % 32, hd // 32
    vr, vm, vx, vc, ve = d // 4, d % 4 // 2, d % 2, pos % 8 // 2, pos % 2  # values: row, tile, half of the tile; column, one of a pair
    kc, kd = d // 8, d % 8
    nc, ns = _sizes(kind, hd)

    def take(t, at):
        return t[..., torch.from_numpy(at.reshape(-1)).to(t.device)].double()

    out = []
    for which in (0, 1):
        codes = pages[..., which * (nc + ns):which * (nc + ns) + nc].contiguous()
        if kind == "f16":
            at = (((a * nb + b) * 2 + kd // 4) * 32 + r * 4 + kc) * 8 + h * 4 + kd % 4 if which == 0 else \
                (((a * nb + b) * 2 + vm) * 32 + vr * 4 + vc) * 8 + h * 4 + vx * 2 + ve
            value = take(codes.view(torch.float16), at)
        else:
            if kind == "q8_0":
                at = ((a * nb + b) * 32 + r * 4 + kc) * 16 + h * 8 + kd if which == 0 else \
                    ((a * nb + b) * 32 + vr * 4 + vc) * 16 + vm * 8 + h * 4 + vx * 2 + ve
                code = take(codes, at) - 128
            else:
                lane = (a * (nb // 2) + b // 2) * 32
                at = (lane + r * 4 + kc) * 16 + b % 2 * 8 + kd // 4 * 4 + kd % 2 * 2 + h if which == 0 else \
                    (lane + vr * 4 + vc) * 16 + b % 2 * 8 + vm * 4 + ve * 2 + h
                unit = torch.from_numpy(16.0 ** (kd % 4 // 2 if which == 0 else vx).reshape(-1)).to(pages.device)
                code = (take(codes, at) / unit).floor() % 16 - 8
            scales = pages[..., which * (nc + ns) + nc:(which + 1) * (nc + ns)].contiguous().view(torch.float16)
            value = code * take(scales, ((pos // 32 * 8 + r) * nb + b) * 4 + pos % 32 // 8)
        out.append(value.reshape(*pages.shape[:2], PAGE, hd).transpose(0, 1).reshape(pages.shape[1], -1, hd))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["what"] == "score":
        return _exact_score(st)
    kind, hd, n_q, n_kv, window, sinks = (case[n] for n in ("kind", "hd", "n_q", "n_kv", "window", "sinks"))
    g, out, row = n_q // n_kv, torch.empty(st["q"].shape, dtype=torch.float64, device=st["q"].device), 0
    for i, (n, length) in enumerate(zip(st["counts"], st["spans"])):
        seen = torch.from_numpy(_seen_pages(n, length, window, sinks)).to(out.device)
        t = (seen[:, None] * PAGE + torch.arange(PAGE, device=out.device)).reshape(-1)
        q = st["q"][row:row + n].double().reshape(n, n_kv, g, hd)
        held = st["pages"][st["table"][i, seen].long()]
        for h in range(n_kv):
            k, v = (x[0] for x in _exact_values(held[:, h:h + 1], kind, hd))
            for j in range(0, n, 1024):  # some of the rows at a time
                p = torch.arange(length - n + j, length - n + min(n, j + 1024), device=out.device)
                fine = t[None, :] <= p[:, None]
                if window:
                    fine &= (t[None, :] > p[:, None] - window) | (t[None, :] < sinks)
                s = torch.einsum("rgd,td->rgt", q[j:j + 1024, h], k) / math.sqrt(hd)
                s.masked_fill_(~fine[:, None, :], float("-inf"))
                o = torch.einsum("rgt,td->rgd", torch.softmax(s, dim=-1), v)
                out[row + j:row + j + len(p), h * g * hd:(h + 1) * g * hd] = o.reshape(len(p), -1)
        row += n
    return out


def _exact_score(st):
    n, parts = st["case"]["top"], []
    for l, t in zip(st["logits"].split(64), st["token"].long().split(64)):
        x = l.double()
        logs = torch.log_softmax(x, dim=-1)
        order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :n] if n else x.new_empty(x.shape[0], 0).long()
        parts.append((logs[torch.arange(len(t)), t], -(logs.exp() * logs).sum(-1), order.int(), logs.gather(1, order)))
    return tuple(torch.cat(p) for p in zip(*parts))
