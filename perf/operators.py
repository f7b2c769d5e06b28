"""What serving many sequences asks of the paged cache, its attention, the rotary positions and the sampler, as cases whose time
is measured.

Families (`what` of a case):

  rope    rotary positions of the heads of some tokens, out of place (`Rope.apply`).
  append  new tokens' keys and values into the cache's pages, keys rotated, and the queries rotated on the way
          (`PagedCache.append`), then a run of positions read back as f32 rows (`PagedCache.read`), which is how a prompt's
          attention sees what earlier tokens left.
  attend  one new token of every sequence over its pages (`PagedCache.attend`); with `shared` pages, the leading ones are the
          same for the whole batch.
  sample  one token of every row of logits from a given random number (`sample`).

A page holds 64 positions of every kv head.  In memory a head's part of a page is keys, scales of keys, values, scales of values;
the order inside is that of the matrix instructions that read it, spelt out in `_decode` below.

Head counts and sizes are those of the decoders of this repository (32 / 8 and 32 / 4 heads of 128, 64-wide ones of its tests,
vocabularies of 128256 and 151936), lengths and batches generic.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 64
BITS = {"f16": 16, "q8_0": 8, "q4_0": 4}
HEADS = [(32, 8), (32, 4), (8, 8), (16, 2), (24, 8), (32, 32)]
VOCABS = [128256, 151936, 32000]


def listed():
    return [
        # the smallest call: one token's queries and keys in the half layout
        {"name": "rope_b1", "what": "rope", "rows": 1, "heads": 40, "hd": 128, "rot": 128, "inter": False, "scaled": False, "ctx": 4096},
        # a prompt in the interleaved layout, half of each head rotated, positions scaled for a long context
        {"name": "rope_2048_interleaved", "what": "rope", "rows": 2048, "heads": 40, "hd": 128, "rot": 64, "inter": True, "scaled": True, "ctx": 32768},
        # a decode step of a batch: a token for each of 32 sequences
        {"name": "append_q8_b32", "what": "append", "kind": "q8_0", "hd": 128, "n_q": 32, "n_kv": 8, "rows": 32, "prompt": False, "ctx": 2048, "back": 32, "inter": False},
        # a prompt of odd length behind an earlier one, and all of both back for its attention
        {"name": "append_q4_1000", "what": "append", "kind": "q4_0", "hd": 128, "n_q": 32, "n_kv": 4, "rows": 1000, "prompt": True, "ctx": 3001, "back": 3001, "inter": True},
        # a long prompt of 64-wide heads into a cache of halves
        {"name": "append_f16_4096", "what": "append", "kind": "f16", "hd": 64, "n_q": 32, "n_kv": 8, "rows": 4096, "prompt": True, "ctx": 4096, "back": 4096, "inter": False},
        # one user, a short conversation: latency
        {"name": "attend_q8_b1", "what": "attend", "kind": "q8_0", "hd": 128, "n_q": 32, "n_kv": 8, "batch": 1, "ctx": 1000, "shared": 0},
        # a batch of very unlike lengths in the smallest cache
        {"name": "attend_q4_b24_ragged", "what": "attend", "kind": "q4_0", "hd": 128, "n_q": 32, "n_kv": 4, "batch": 24, "ctx": 16384, "shared": 0},
        # a full batch of long sequences, 8 bits
        {"name": "attend_q8_b64", "what": "attend", "kind": "q8_0", "hd": 128, "n_q": 32, "n_kv": 8, "batch": 64, "ctx": 8192, "shared": 0},
        # a batch behind one long system prompt, short tails of their own
        {"name": "attend_q8_b32_shared", "what": "attend", "kind": "q8_0", "hd": 128, "n_q": 32, "n_kv": 8, "batch": 32, "ctx": 4600, "shared": 64},
        # many requests on one document, halves of 64-wide heads
        {"name": "attend_f16_b128_shared", "what": "attend", "kind": "f16", "hd": 64, "n_q": 32, "n_kv": 8, "batch": 128, "ctx": 8500, "shared": 128},
        # one user's next token under all four rules
        {"name": "sample_b1", "what": "sample", "rows": 1, "vocab": 128256, "peak": 6.0},
        # a batch whose requests each have rules of their own, a vocabulary of another size
        {"name": "sample_b64", "what": "sample", "rows": 64, "vocab": 151936, "peak": 3.0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(["rope", "append", "append", "attend", "attend", "attend", "sample"])
    hd = rng.choice([64, 128, 128, 256])
    if what == "rope":
        rows = _log_int(rng, 1, 2048)
        return {"what": what, "rows": rows, "heads": rng.choice([1, 5, 10, 40]), "hd": hd,
                "rot": rng.choice([hd, hd // 2, hd // 4]), "inter": rng.random() < 0.5, "scaled": rng.random() < 0.5,
                "ctx": _log_int(rng, max(rows, 512), 32768)}
    kind, (n_q, n_kv) = rng.choice(sorted(BITS)), rng.choice(HEADS)
    if what == "append":
        prompt = rng.random() < 0.6
        most = 2**25 // ((n_q + 2 * n_kv) * hd)
        rows = _log_int(rng, 2, min(4096, most)) if prompt else _log_int(rng, 1, 128)
        ctx = _log_int(rng, max(rows, 16), 4096)
        return {"what": what, "kind": kind, "hd": hd, "n_q": n_q, "n_kv": n_kv, "rows": rows, "prompt": prompt, "ctx": ctx,
                "back": rng.randrange(1, ctx + 1) if prompt else rows, "inter": rng.random() < 0.5}
    if what == "attend":
        batch = _log_int(rng, 1, 128)
        most = 2.0**29 / (batch * n_kv * hd)  # positions a sequence, so that the largest listed one stays it
        ctx = _log_int(rng, 1, int(min(65536, max(64, most))))
        shared = 0
        if ctx > PAGE and rng.random() < 0.5:
            shared = rng.randrange(1, (ctx - 1) // PAGE + 1)
        return {"what": what, "kind": kind, "hd": hd, "n_q": n_q, "n_kv": n_kv, "batch": batch, "ctx": ctx, "shared": shared}
    return {"what": what, "rows": _log_int(rng, 1, 96), "vocab": rng.choice(VOCABS) - rng.randrange(0, 500),
            "peak": rng.uniform(1.0, 8.0)}


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
def _rope_table(rot, n_pos, scaled, dev):
    """(cos, sin) of every position and pair, as a decoder keeps them; scaled: positions stretched by 8, the fast ones less."""
    f = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    if scaled:
        wave = 2 * math.pi / f
        mix = ((8192 / wave - 1) / 3).clamp(0, 1)
        f = f * (mix + (1 - mix) / 8)
    angle = torch.arange(n_pos, dtype=torch.float64, device=dev)[:, None] * f
    return torch.stack((angle.cos(), angle.sin()), dim=-1).float()


def _lengths(case):
    """Positions each sequence holds: spread from the shared part, or from one, to the longest, which the first one has."""
    least, n = case["shared"] * PAGE + 1, case["batch"]
    rng = np.random.RandomState((1009 * case["ctx"] + n) % 2**32)
    ctx = case["ctx"]
    spread = rng.uniform(size=n) ** (2.0 if ctx > 8192 else 1.0)
    lens = (least + (ctx - least) * spread).astype(np.int64)
    lens[0] = ctx
    return lens


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    what = case["what"]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    if what == "rope":
        start = int(torch.randint(0, case["ctx"] - case["rows"] + 1, (1,), device=dev, generator=gen))
        return {"case": case, "x": normal(case["rows"], case["heads"] * case["hd"]),
                "pos": torch.arange(start, start + case["rows"], dtype=torch.int32, device=dev),
                "table": _rope_table(case["rot"], case["ctx"], case["scaled"], dev)}
    if what == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab) * 2.5
        some = torch.randint(0, vocab, (rows, 20), device=dev, generator=gen)
        logits.scatter_add_(1, some, normal(rows, 20).abs() * case["peak"])
        pick = torch.rand(4, rows, device=dev, generator=gen)
        return {"case": case, "logits": logits, "u": torch.rand(rows, device=dev, generator=gen),
                "temperature": 0.5 + pick[0], "top_k": torch.where(pick[1] < 0.5, 40, 1000).int(),
                "top_p": torch.where(pick[2] < 0.7, 0.95, 1.0), "min_p": torch.where(pick[3] < 0.5, 0.0, 0.02)}
    kind, hd, n_q, n_kv = case["kind"], case["hd"], case["n_q"], case["n_kv"]
    if what == "append":
        rows, ctx = case["rows"], case["ctx"]
        seqs = 1 if case["prompt"] else rows
        per = -(-ctx // PAGE)
        if case["prompt"]:  # the last rows of one sequence; `back` positions up to the last are read
            pos = torch.arange(ctx - rows, ctx, dtype=torch.int32, device=dev)
            back = torch.arange(ctx - case["back"], ctx, dtype=torch.int32, device=dev)
            seq, back_seq = torch.zeros(rows, dtype=torch.int32, device=dev), torch.zeros(case["back"], dtype=torch.int32, device=dev)
        else:  # a row of each sequence, and the same rows back
            pos = torch.randint(0, ctx, (rows,), dtype=torch.int32, device=dev, generator=gen)
            seq = back_seq = torch.arange(rows, dtype=torch.int32, device=dev)
            back = pos
        return {"case": case, "qkv": normal(rows, (n_q + 2 * n_kv) * hd), "pos": pos, "seq": seq, "back": back, "back_seq": back_seq,
                "pages": _pages(kind, hd, n_kv, seqs * per, gen, dev), "rope": _rope_table(hd, ctx, False, dev),
                "table": torch.randperm(seqs * per, device=dev, generator=gen).int().reshape(seqs, per)}
    lens = _lengths(case)
    shared, batch = case["shared"], case["batch"]
    per = -(-case["ctx"] // PAGE)
    used = [-(-int(n) // PAGE) - shared for n in lens]  # pages of a sequence's own
    count = shared + sum(used)
    order = torch.randperm(count, device=dev, generator=gen).int()
    table = torch.zeros(batch, per, dtype=torch.int32, device=dev)
    table[:, :shared] = order[:shared]
    at = shared
    for i, n in enumerate(used):
        table[i, shared:shared + n] = order[at:at + n]
        at += n
    return {"case": case, "q": normal(batch, n_q * hd), "pages": _pages(kind, hd, n_kv, count, gen, dev), "table": table,
            "lens": torch.from_numpy(lens).int().to(dev)}


# ── one pass ────────────────────────────────────────────────────────────
def run(state):
    return (_run_own if own else _run_plain)(state)


def _handles(state):
    """What a program builds once around its tensors."""
    from joshua_b200.kv_cache import PagedCache
    from joshua_b200.rope import Rope

    case, made = state["case"], {}
    if case["what"] == "rope":
        made["rope"] = Rope(state["table"], interleaved=case["inter"])
    elif case["what"] == "append":
        made["rope"] = Rope(state["rope"], interleaved=case["inter"])
    if "pages" in state:
        made["cache"] = PagedCache(case["kind"], case["n_kv"], case["hd"], pages=state["pages"])
    return made


def _run_own(state):
    case = state["case"]
    if "handles" not in state:
        state["handles"] = _handles(state)
    made = state["handles"]
    if case["what"] == "rope":
        return made["rope"].apply(state["x"], state["pos"], case["heads"], case["hd"])
    if case["what"] == "append":
        q = made["cache"].append(state["qkv"], state["pos"], state["table"], n_q=case["n_q"], seq=state["seq"], rope=made["rope"])
        return q, *made["cache"].read(state["back"], state["table"], seq=state["back_seq"])
    if case["what"] == "attend":
        return made["cache"].attend(state["q"], state["lens"], state["table"], n_q=case["n_q"], shared_pages=case["shared"])
    from joshua_b200.sampling import sample

    return sample(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                  min_p=state["min_p"])


def _rotate(x, table, pos, rot, inter):
    """Rotary positions of [rows, heads, hd]."""
    cs = table[pos.long()].unsqueeze(1)
    c, s = cs[..., 0], cs[..., 1]
    y = x.clone()
    if inter:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, a * s + b * c
    return y


def _place(codes, scales, kind, hd, which):
    """Bytes that one position's codes and scales take in its page: (place of each byte in a head's part [PAGE, ...], bytes)."""
    nc, ns = _sizes(kind, hd)
    shape, order = _orders(kind, hd)[which]
    dev = codes.device
    at = torch.arange(PAGE * hd, device=dev).reshape(shape).permute(order).reshape(PAGE, hd)
    if kind == "f16":
        at = torch.stack((2 * at, 2 * at + 1), dim=-1).reshape(PAGE, -1)
        data = codes.contiguous().view(torch.uint8)
    elif kind == "q8_0":
        data = codes
    else:  # pairs of codes in a byte: `at` counts halves of bytes
        low = at.reshape(PAGE, hd)
        first = (low[0] & 1 == 0).nonzero().reshape(-1)
        partner = (low[0][:, None] == low[0][first][None, :] + 1).float().argmax(0)
        at = low[:, first] // 2
        data = codes[..., first] | (codes[..., partner] << 4)
    at = at + which * (nc + ns)
    if ns:
        sat = torch.arange(ns // 2, device=dev).reshape(2, 8, hd // 32, 4).permute(0, 3, 1, 2).reshape(PAGE, hd // 32)
        sat = torch.stack((2 * sat, 2 * sat + 1), dim=-1).reshape(PAGE, -1) + which * (nc + ns) + nc
        at = torch.cat((at, sat), dim=-1)
        data = torch.cat((data, scales.contiguous().view(torch.uint8)), dim=-1)
    return at, data


def _run_plain(state):
    case, what = state["case"], state["case"]["what"]
    if what == "rope":
        x = state["x"].reshape(case["rows"], case["heads"], case["hd"])
        return _rotate(x, state["table"], state["pos"], case["rot"], case["inter"]).reshape(case["rows"], -1)
    if what == "append":
        return _plain_append(state, case)
    if what == "attend":
        return _plain_attend(state, case)
    return _plain_sample(state)


def _plain_append(state, case):
    kind, hd, n_q, n_kv, rows = case["kind"], case["hd"], case["n_q"], case["n_kv"], case["rows"]
    x = state["qkv"].reshape(rows, n_q + 2 * n_kv, hd)
    qk = _rotate(x[:, :n_q + n_kv], state["rope"], state["pos"], hd, case["inter"])
    pos = state["pos"].long()
    page = state["table"][state["seq"].long(), pos // PAGE].long()
    head = torch.arange(n_kv, device=x.device)
    for which, rowsof in enumerate((qk[:, n_q:], x[:, n_q + n_kv:])):
        codes, scales = _quantise(rowsof, kind)
        at, data = _place(codes, scales, kind, hd, which)
        at = at[pos % PAGE]  # [rows, bytes]
        state["pages"][page[:, None, None], head[None, :, None], at[:, None, :]] = data
    back = state["back"].long()
    held = state["table"][0] if case["prompt"] else state["table"][state["back_seq"].long(), back // PAGE]
    k, v = _decode(state["pages"][held.long()], kind, hd)  # [pages, n_kv, PAGE, hd]
    if case["prompt"]:
        first = case["ctx"] - case["back"]
        k, v = (t.transpose(0, 1).reshape(n_kv, -1, hd)[:, first:case["ctx"]] for t in (k, v))
    else:
        i = torch.arange(rows, device=x.device)
        k, v = (t[i, :, back % PAGE].transpose(0, 1) for t in (k, v))
    return qk[:, :n_q].reshape(rows, -1), k.contiguous(), v.contiguous()


def _softmax(s):
    e = (s - s.amax(-1, keepdim=True)).exp()
    return e / e.sum(-1, keepdim=True)


def _plain_attend(state, case):
    kind, hd, n_q, n_kv, batch = case["kind"], case["hd"], case["n_q"], case["n_kv"], case["batch"]
    g, lens, table = n_q // n_kv, state["lens"].long(), state["table"].long()
    q = state["q"].reshape(batch, n_kv, g, hd) / math.sqrt(hd)
    shared = case["shared"]
    own_k, own_v = _decode(state["pages"][table[:, shared:]], kind, hd)  # [batch, pages, n_kv, PAGE, hd]
    own_k, own_v = (t.transpose(1, 2).reshape(batch, n_kv, -1, hd) for t in (own_k, own_v))
    s = torch.matmul(q, own_k.transpose(-1, -2))
    at = shared * PAGE + torch.arange(s.shape[-1], device=s.device)
    s = torch.where((at[None, :] < lens[:, None])[:, None, None, :], s, float("-inf"))
    if not shared:
        return torch.matmul(_softmax(s), own_v).reshape(batch, -1)
    k, v = _decode(state["pages"][table[0, :shared]], kind, hd)  # [pages, n_kv, PAGE, hd]
    k, v = (t.transpose(0, 1).reshape(n_kv, -1, hd) for t in (k, v))
    rows = q.transpose(0, 1).reshape(n_kv, batch * g, hd)
    first = torch.matmul(rows, k.transpose(-1, -2)).reshape(n_kv, batch, g, -1).transpose(0, 1)
    p = _softmax(torch.cat((first, s), dim=-1))
    n = shared * PAGE
    out = torch.matmul(p[..., :n].transpose(0, 1).reshape(n_kv, batch * g, n), v).reshape(n_kv, batch, g, hd).transpose(0, 1)
    return (out + torch.matmul(p[..., n:], own_v)).reshape(batch, -1)


def _plain_sample(state):
    l, k = state["logits"], state["top_k"].long()
    rows, vocab = l.shape
    best = l.amax(-1, keepdim=True)
    e = ((l - best) / state["temperature"][:, None]).exp()
    w = (e * 4294967296.0).round().to(torch.int64)  # weights in fixed point: their sums are exact
    order = l.sort(dim=-1, descending=True, stable=True).indices
    w, e = w.gather(1, order), e.gather(1, order)
    rank = torch.arange(vocab, device=l.device)[None, :]
    kept = (rank < k[:, None]) | (k[:, None] <= 0)
    w = torch.where(kept, w, 0)
    before = w.cumsum(-1) - w
    total = w.sum(-1, keepdim=True)
    p = state["top_p"][:, None].double()
    most = torch.where(p < 1, (p * total.double()).to(torch.int64).clamp(min=1), total)
    kept = kept & (before < most) & (e >= state["min_p"][:, None])
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0))  # by token again
    cum = w.cumsum(-1)
    total = cum[:, -1:]
    r = torch.minimum((state["u"][:, None].double() * total.double()).to(torch.int64), total - 1)
    token = (cum <= r).sum(-1)
    prob = (w.gather(1, token[:, None]).double() / total.double()).float().reshape(-1)
    return token.int(), prob


# ── how much of it there is, and what it is exactly ─────────────────────
def work(case):
    what = case["what"]
    if what == "rope":
        n = case["rows"] * case["heads"] * case["hd"]
        return {"bytes": 8 * n + case["rows"] * (4 + 4 * case["rot"]), "flops": 3 * case["rows"] * case["heads"] * case["rot"]}
    if what == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    kind, hd, n_q, n_kv = case["kind"], case["hd"], case["n_q"], case["n_kv"]
    held = 2 * n_kv * sum(_sizes(kind, hd)) // PAGE  # bytes of a position
    if what == "append":
        rows = case["rows"]
        io = 4 * rows * (n_q + 2 * n_kv) * hd + 4 * rows * n_q * hd + rows * (8 + 4 * hd) + rows * held
        return {"bytes": io + case["back"] * (held + 8 * n_kv * hd), "flops": rows * hd * (3 * (n_q + n_kv) + 8 * n_kv) + 2 * case["back"] * n_kv * hd}
    lens = [int(n) for n in _lengths(case)]
    alone = sum(n - case["shared"] * PAGE for n in lens)
    return {"bytes": (alone + case["shared"] * PAGE) * held + 8 * case["batch"] * n_q * hd, "flops": 4 * sum(lens) * n_q * hd}


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


def _exact_rope(x, pos, rot, inter, table):
    """Rotation of [rows, heads, hd] in 64 bits, by complex numbers of the table's entries."""
    t = table[pos].astype(np.float64)
    turn = (t[..., 0] + 1j * t[..., 1])[:, None, :]
    y = x.astype(np.float64).copy()
    half = rot // 2
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, half), slice(half, rot))
    z = (y[..., first] + 1j * y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    what, st = case["what"], prepare(case, seed)
    if what == "rope":
        x = st["x"].cpu().numpy().reshape(case["rows"], case["heads"], case["hd"])
        y = _exact_rope(x, st["pos"].cpu().numpy(), case["rot"], case["inter"], st["table"].cpu().numpy())
        return y.reshape(case["rows"], -1)
    if what == "sample":
        return _exact_sample(st)
    kind, hd, n_q, n_kv = case["kind"], case["hd"], case["n_q"], case["n_kv"]
    if what == "append":
        rows = case["rows"]
        x = st["qkv"].cpu().numpy().reshape(rows, n_q + 2 * n_kv, hd)
        y = _exact_rope(x, st["pos"].cpu().numpy(), hd, case["inter"], st["rope"].cpu().numpy())
        y[:, n_q + n_kv:] = x[:, n_q + n_kv:]
        fresh = [_exact_held(y[:, i:i + n_kv], kind).transpose(1, 0, 2) for i in (n_q, n_q + n_kv)]
        if not case["prompt"]:
            return y[:, :n_q].reshape(rows, -1), *fresh
        k, v = (t.cpu().numpy() for t in _exact_values(st["pages"][st["table"][0].long()], kind, hd))
        k, v = (np.concatenate((t[:, :case["ctx"] - rows], f), axis=1)[:, case["ctx"] - case["back"]:] for t, f in zip((k, v), fresh))
        return y[:, :n_q].reshape(rows, -1), k, v
    q, out = st["q"].double().reshape(case["batch"], n_kv, n_q // n_kv, hd), []
    for b, n in enumerate(st["lens"].tolist()):
        k, v = (t[:, :n] for t in _exact_values(st["pages"][st["table"][b, :-(-n // PAGE)].long()], kind, hd))
        s = torch.einsum("hgd,hnd->hgn", q[b], k) / math.sqrt(hd)
        out.append(torch.einsum("hgn,hnd->hgd", torch.softmax(s, dim=-1), v).reshape(-1))
    return torch.stack(out)


def _exact_held(x, kind):
    """What the cache holds of f64 rows [..., hd]."""
    if kind == "f16":
        return x.astype(np.float16).astype(np.float64)
    y = x.reshape(*x.shape[:-1], -1, 32)
    if kind == "q8_0":
        d = (np.abs(y).max(-1) / 127).astype(np.float16).astype(np.float64)[..., None]
        return (np.rint(y / d).clip(-127, 127) * d).reshape(x.shape)
    top = np.take_along_axis(y, np.abs(y).argmax(-1)[..., None], -1)
    d = (top / -8).astype(np.float16).astype(np.float64)
    return (np.rint(y / d).clip(-8, 7) * d).reshape(x.shape)


def _exact_sample(st):
    logits, u = st["logits"].cpu().numpy().astype(np.float64), st["u"].cpu().numpy().astype(np.float64)
    rules = [st[n].cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p")]
    tokens, probs = [], []
    for l, x, t, k, p, m in zip(logits, u, *rules):
        e = np.exp((l - l.max()) / np.float64(t))
        order = np.argsort(-l, kind="stable")
        if k > 0:
            order = order[:k]
        mass = e[order]
        if p < 1:
            order = order[np.cumsum(mass) - mass < np.float64(p) * mass.sum()]
        order = np.sort(order[e[order] >= m])
        cum = np.cumsum(e[order])
        i = min(int(np.searchsorted(cum, x * cum[-1], side="right")), len(order) - 1)
        tokens.append(order[i])
        probs.append(e[order[i]] / cum[-1])
    return np.array(tokens, dtype=np.int32), np.array(probs)
