"""The paged cache: positions rounded into their pages and read back, against the rounding stated in f32 operations.

No tolerance stands on keys and values: the library states each operation of the rounding, so what is read back is equal to the
statement's values (a code times its scale is exact in f32: 8 + 11 bits).  Rotated rows are compared through the device's own
rotation (`Rope.apply`, tested by itself), which the cache has to match bit for bit.
"""
import numpy as np
import pytest

from joshua_b200 import _lib
from joshua_b200._lib import JoshuaB200Error
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu
KINDS = ["f16", "q8_0", "q4_0"]


def i32(values):
    import torch

    return torch.tensor(list(map(int, values)), dtype=torch.int32, device="cuda")


def make(kind, n_kv, hd, seqs, per, seed=0, spare=3):
    """A cache of pages full of rubbish (NaN bit patterns among it), handed out in random order."""
    import torch

    from joshua_b200.kv_cache import PagedCache

    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = PagedCache(kind, n_kv, hd, n_pages=seqs * per + spare, device="cuda")
    cache.pages.copy_(torch.randint(0, 256, cache.pages.shape, dtype=torch.uint8, device="cuda", generator=g))
    table = torch.randperm(seqs * per + spare, device="cuda", generator=g)[:seqs * per].int().reshape(seqs, per)
    return cache, table


def split(qkv, n_q, n_kv, hd):
    x = np.asarray(qkv).reshape(len(qkv), n_q + 2 * n_kv, hd)
    return x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,n_q,n_kv", [(64, 6, 3), (128, 8, 2), (256, 2, 1), (128, 4, 4), (64, 1, 1)])
def test_append_and_read(kind, hd, n_q, n_kv):
    import torch

    rng = np.random.RandomState(hd + n_q)
    cache, table = make(kind, n_kv, hd, 4, 3)
    want_k, want_v, places = {}, {}, []
    # three calls: a prompt of one sequence, rows of several in no order, a step of all
    for call, (seq, pos) in enumerate([([2] * 70, range(5, 75)), ([0, 3, 0, 1, 3], [191, 0, 7, 64, 63]), (None, [100, 15, 75, 128])]):
        rows = len(pos)
        x = rng.randn(rows, (n_q + 2 * n_kv) * hd).astype(np.float32) * np.float32(10.0 ** rng.uniform(-3, 3, (rows, 1)))
        out = cache.append(torch.from_numpy(x).cuda(), i32(pos), table, n_q=n_q, seq=None if seq is None else i32(seq))
        q, k, v = split(x, n_q, n_kv, hd)
        assert np.array_equal(out.cpu().numpy().reshape(q.shape), q)
        for i, p in enumerate(pos):
            at = (seq[i] if seq else i, p)
            want_k[at], want_v[at] = ref.held(k[i], kind), ref.held(v[i], kind)
    at = sorted(want_k, key=lambda a: (a[1] * 7919 + a[0]) % 101)
    k, v = cache.read(i32(p for _, p in at), table, seq=i32(s for s, _ in at))
    assert np.array_equal(k.cpu().numpy(), np.stack([want_k[a] for a in at], 1))
    assert np.array_equal(v.cpu().numpy(), np.stack([want_v[a] for a in at], 1))
    cache.check_flags()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,start", [(1, 0), (1, 63), (15, 1), (16, 16), (17, 47), (64, 0), (65, 63), (200, 30), (130, 63), (128, 16), (300, 7)])
def test_prompts_of_all_lengths(kind, rows, start):
    """Runs that begin and end inside pages and groups of 16 leave their neighbours as they were."""
    import torch

    n_q, n_kv, hd = 2, 2, 128
    cache, table = make(kind, n_kv, hd, 2, 5)
    rng = np.random.RandomState(rows)
    before = rng.randn(320, (n_q + 2 * n_kv) * hd).astype(np.float32)
    cache.append(torch.from_numpy(before).cuda(), i32(range(320)), table, n_q=n_q, seq=i32([1] * 320))
    x = rng.randn(rows, (n_q + 2 * n_kv) * hd).astype(np.float32)
    cache.append(torch.from_numpy(x).cuda(), i32(range(start, start + rows)), table, n_q=n_q, seq=i32([1] * rows))
    whole = before.copy()
    whole[start:start + rows] = x
    k, v = cache.read(i32(range(320)), table, seq=i32([1] * 320))
    _, wk, wv = split(whole, n_q, n_kv, hd)
    assert np.array_equal(k.cpu().numpy(), ref.held(wk, kind).transpose(1, 0, 2))
    assert np.array_equal(v.cpu().numpy(), ref.held(wv, kind).transpose(1, 0, 2))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_rows_of_several_sequences(kind, hd):
    """Hundreds of rows in one call: prompts of three sequences one behind another, then the same rows in another order, and read
    back in a third; rows without a place among them."""
    import torch

    n_q, n_kv = 3, 3
    cache, table = make(kind, n_kv, hd, 3, 4, seed=hd)
    rng = np.random.RandomState(hd)
    seq = np.repeat([2, 0, 1], [150, 97, 120])
    pos = np.concatenate([np.arange(150) + 31, np.arange(97), np.arange(120) + 64])
    for order in (np.arange(len(pos)), rng.permutation(len(pos))):
        x = rng.randn(len(pos), (n_q + 2 * n_kv) * hd).astype(np.float32)
        q = cache.append(torch.from_numpy(x).cuda(), i32(pos[order]), table, n_q=n_q, seq=i32(seq[order]))
        wq, wk, wv = split(x, n_q, n_kv, hd)
        assert np.array_equal(q.cpu().numpy().reshape(wq.shape), wq)
        back = rng.permutation(len(pos))
        for again in (np.arange(len(pos)), back):
            k, v = cache.read(i32(pos[order][again]), table, seq=i32(seq[order][again]))
            assert np.array_equal(k.cpu().numpy(), ref.held(wk, kind)[again].transpose(1, 0, 2))
            assert np.array_equal(v.cpu().numpy(), ref.held(wv, kind)[again].transpose(1, 0, 2))
    cache.check_flags()
    lost = pos.copy()
    lost[40], lost[200] = -1, 4 * 64
    x = rng.randn(len(pos), (n_q + 2 * n_kv) * hd).astype(np.float32)
    out = torch.full((len(pos), n_q * hd), 7.0, device="cuda")
    cache.append(torch.from_numpy(x).cuda(), i32(lost), table, n_q=n_q, seq=i32(seq), out=out)
    assert bool((out[[40, 200]] == 7).all()) and int(cache.bad_pos) == 1
    k, v = cache.read(i32(lost), table, seq=i32(seq))
    want = ref.held(split(x, n_q, n_kv, hd)[1], kind).transpose(1, 0, 2)
    want[:, [40, 200]] = np.nan
    assert np.array_equal(k.cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,n_q,n_kv,rot,interleaved", [(64, 5, 5, 64, False), (128, 6, 3, 64, True), (128, 2, 2, 12, False), (256, 2, 1, 256, False)])
def test_a_thousand_rows(kind, hd, n_q, n_kv, rot, interleaved):
    """Whole prompts of two sequences in one call, rotated and normed on the way as the same rows a few at a time, in order and out
    of it; their neighbours stay; rows without a place among them."""
    import torch

    from joshua_b200.rope import Rope, rope_table

    rope = Rope(rope_table(10000.0, rot, 960, "cuda"), interleaved=interleaved)
    (cache, table), (other, _) = make(kind, n_kv, hd, 2, 15), make(kind, n_kv, hd, 2, 15)
    width = (n_q + 2 * n_kv) * hd
    rng = np.random.RandomState(hd + rot)
    norm = torch.from_numpy(rng.uniform(0.5, 2.0, hd).astype(np.float32)).cuda()
    every = i32(list(range(960)) * 2), i32([0] * 960 + [1] * 960)
    before = torch.from_numpy(rng.randn(1920, width).astype(np.float32)).cuda()
    for c in (cache, other):
        c.append(before, every[0], table, n_q=n_q, seq=every[1])
    seq = np.repeat([1, 0], [603, 411])
    pos = np.concatenate([np.arange(603) + 47, np.arange(411) + 500])
    x = torch.from_numpy(rng.randn(len(pos), width).astype(np.float32)).cuda()
    for order in (np.arange(len(pos)), rng.permutation(len(pos))):
        kw = dict(n_q=n_q, rope=rope, q_norm=norm, k_norm=norm, eps=1e-5)
        q = cache.append(x, i32(pos[order]), table, seq=i32(seq[order]), **kw)
        few = torch.cat([other.append(x[i:i + 100], i32(pos[order][i:i + 100]), table, seq=i32(seq[order][i:i + 100]), **kw)
                         for i in range(0, len(pos), 100)])
        assert torch.equal(q, few)
        read = cache.read(*every[:1], table, seq=every[1])
        parts = [other.read(every[0][i:i + 100], table, seq=every[1][i:i + 100]) for i in range(0, 1920, 100)]
        for i in range(2):
            assert torch.equal(read[i], torch.cat([part[i] for part in parts], 1))
        _, _, wv = split(x.cpu().numpy(), n_q, n_kv, hd)
        assert np.array_equal(cache.read(i32(pos[order]), table, seq=i32(seq[order]))[1].cpu().numpy(), ref.held(wv, kind).transpose(1, 0, 2))
    cache.check_flags()
    lost = pos.copy()
    lost[[40, 1000]] = -1, 15 * 64
    out = torch.full((len(pos), n_q * hd), 7.0, device="cuda")
    q = cache.append(x, i32(pos), table, seq=i32(seq), **kw)
    cache.append(x, i32(lost), table, seq=i32(seq), out=out, **kw)
    q[[40, 1000]] = 7.0
    assert torch.equal(q, out) and int(cache.bad_pos) == 1
    k, v = cache.read(i32(lost), table, seq=i32(seq))
    assert bool(k[:, [40, 1000]].isnan().all()) and int(torch.cat([k, v]).isnan().any(2).sum()) == 4 * n_kv


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [40, 170])
@pytest.mark.parametrize("hd,rot,interleaved", [(128, 128, False), (128, 64, True), (64, 64, True), (256, 96, False), (64, 2, False)])
def test_rotation_on_the_way(kind, rows, hd, rot, interleaved):
    import torch

    from joshua_b200.rope import Rope, rope_table

    n_q, n_kv = 3, 3
    rope = Rope(rope_table(500000.0, rot, 900, "cuda"), interleaved=interleaved)
    cache, table = make(kind, n_kv, hd, 1, 13)
    torch.manual_seed(rot)
    x = torch.randn(rows, 9 * hd, device="cuda")
    pos = torch.arange(655, 655 + rows, dtype=torch.int32, device="cuda")
    seq = torch.zeros(rows, dtype=torch.int32, device="cuda")
    q = cache.append(x, pos, table, n_q=n_q, seq=seq, rope=rope)
    turned = rope.apply(x[:, :6 * hd], pos, 6, hd)
    assert torch.equal(q, turned[:, :3 * hd])
    k, v = cache.read(pos, table, seq=seq)
    assert np.array_equal(k.cpu().numpy(), ref.held(turned[:, 3 * hd:].cpu().numpy().reshape(rows, 3, hd), kind).transpose(1, 0, 2))
    assert np.array_equal(v.cpu().numpy(), ref.held(x[:, 6 * hd:].cpu().numpy().reshape(rows, 3, hd), kind).transpose(1, 0, 2))


@pytest.mark.parametrize("hd,rows", [(64, 9), (128, 9), (256, 9), (64, 130), (128, 130), (256, 130)])
def test_norms_on_the_way(hd, rows):
    """The per-head norm in front of the rotation.  Its sum of squares is rounded (hd products and sums, the root, two products:
    under (hd + 8) roundings of 2^-24 in all) and a key then by at most 2^-11 (halves)."""
    import torch

    from joshua_b200.rope import Rope, rope_table

    n_q, n_kv = 4, 2
    table_np = rope_table(10000.0, hd, 64, "cuda")
    rope = Rope(table_np)
    cache, table = make("f16", n_kv, hd, rows, 1)
    rng = np.random.RandomState(hd)
    x = rng.randn(rows, 8 * hd).astype(np.float32)
    qw, kw = (rng.uniform(0.5, 2.0, hd).astype(np.float32) for _ in range(2))
    pos = rng.randint(0, 64, rows)
    q = cache.append(torch.from_numpy(x).cuda(), i32(pos), table, n_q=n_q, rope=rope, q_norm=torch.from_numpy(qw).cuda(),
                     k_norm=torch.from_numpy(kw).cuda(), eps=1e-6)
    k, v = cache.read(i32(pos), table)

    def normed(t, w):
        t = t.astype(np.float64)
        return ref.rope(t / np.sqrt((t * t).mean(-1, keepdims=True) + 1e-6) * w, table_np.cpu().numpy(), pos, hd, False)

    wq, wk, wv = split(x, n_q, n_kv, hd)
    tol = (hd + 8) * 2.0**-24
    top = lambda t: np.abs(t).max(-1, keepdims=True)  # noqa: E731
    want = normed(wq, qw)
    assert np.all(np.abs(q.cpu().numpy().reshape(want.shape) - want) <= 2 * tol * top(want))
    want = normed(wk, kw)
    assert np.all(np.abs(k.cpu().numpy().transpose(1, 0, 2) - want) <= (2 * tol + 2.0**-11) * top(want))
    assert np.array_equal(v.cpu().numpy().transpose(1, 0, 2), ref.held(wv, "f16"))


@pytest.mark.parametrize("kind", KINDS)
def test_extreme_values(kind):
    import torch

    hd = 64
    cache, table = make(kind, 1, hd, 12, 1)
    x = np.zeros((12, 3 * hd), dtype=np.float32)
    k = x[:, hd:2 * hd]
    k[0, 0] = np.nan            # a block with a NaN reads as NaN, the other block of the head does not
    k[1, 5], k[1, 40] = np.inf, 1.0
    k[2, 33] = -np.inf
    k[3] = 1e30                 # past what a scale (a half) holds
    k[4, ::2], k[4, 1::2] = -3e38, 3e38
    k[5] = 1e-30                # a scale of zero
    k[6] = 1e-7                 # a subnormal scale
    k[7, 3], k[7, 9] = -2.5, 2.5  # equal magnitudes of both signs
    k[8, 3], k[8, 9] = 2.5, -2.5
    k[9] = -0.0
    k[10] = 65504.0
    k[11] = np.linspace(-65520, 65520, hd)
    x[:, 2 * hd:] = k
    cache.append(torch.from_numpy(x).cuda(), i32([7] * 12), table, n_q=1)
    got = cache.read(i32([7] * 12), table)
    for t in got:
        assert np.array_equal(t.cpu().numpy()[0], ref.held(k, kind).astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
def test_strided_rows_and_given_outputs(kind):
    import torch

    n_q, n_kv, hd, rows = 4, 2, 128, 33
    cache, table = make(kind, n_kv, hd, rows, 1)
    x = torch.randn(rows, 8 * hd, device="cuda")
    wide = torch.randn(rows, 8 * hd + 132, device="cuda")
    wide[:, 64:64 + 8 * hd] = x
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    out = torch.empty(rows, n_q * hd, device="cuda")
    q = cache.append(wide[:, 64:64 + 8 * hd], pos, table, n_q=n_q, out=out)
    assert q is out and torch.equal(q, x[:, :n_q * hd])
    into = torch.full((n_kv, rows + 7, hd), 3.0, device="cuda"), torch.full((n_kv, rows + 7, hd), 3.0, device="cuda")
    k, v = cache.read(pos, table, out=into)
    _, wk, wv = split(x.cpu().numpy(), n_q, n_kv, hd)
    for t, w in ((k, wk), (v, wv)):
        assert np.array_equal(t[:, :rows].cpu().numpy(), ref.held(w, kind).transpose(1, 0, 2)) and bool((t[:, rows:] == 3).all())


def test_rows_without_a_place():
    import torch

    n_q, n_kv, hd = 1, 1, 64
    cache, table = make("q8_0", n_kv, hd, 2, 2)
    table[1, 1] = cache.pages.shape[0]    # ids outside the cache
    table[0, 1] = -1
    before = cache.pages.clone()
    x = torch.randn(6, 3 * hd, device="cuda")
    pos, seq = i32([-1, 128, 64, 70, 0, 5]), i32([0, 0, 1, 0, 2, -1])
    out = torch.full((6, hd), 9.0, device="cuda")
    cache.append(x, pos, table, n_q=n_q, seq=seq, out=out)
    assert bool((out == 9).all()) and torch.equal(cache.pages, before)
    with pytest.raises(JoshuaB200Error):
        cache.check_flags()
    cache.check_flags()
    k, v = cache.read(pos, table, seq=seq)
    assert bool(k.isnan().all()) and bool(v.isnan().all()) and int(cache.bad_pos) == 1
    from joshua_b200.rope import Rope, rope_table

    cache.bad_pos.zero_()   # a position that the rope table does not have
    cache.append(x[:1], i32([60]), table, n_q=n_q, seq=i32([1]), rope=Rope(rope_table(1e4, hd, 60, "cuda")), out=out[:1])
    assert int(cache.bad_pos) == 1 and torch.equal(cache.pages, before)


def test_refusals():
    import torch

    from joshua_b200.kv_cache import PagedCache

    cache, table = make("q8_0", 2, 64, 2, 2)
    x, pos = torch.zeros(2, 8 * 64, device="cuda"), i32([0, 0])
    for bad in (lambda: PagedCache("q5_0", 2, 64, n_pages=1, device="cuda"), lambda: PagedCache("q8_0", 2, 96, n_pages=1, device="cuda"),
                lambda: PagedCache("q8_0", 0, 64, n_pages=1, device="cuda"), lambda: PagedCache("q8_0", 2, 64, pages=cache.pages[:, 1:]),
                lambda: PagedCache("q8_0", 2, 64, pages=cache.pages[:0]),
                lambda: cache.append(x, pos, table, n_q=3), lambda: cache.append(x[:, :256], pos, table, n_q=4),
                lambda: cache.append(x, pos[:1], table, n_q=4), lambda: cache.append(x.double(), pos, table, n_q=4),
                lambda: cache.append(x, pos, table.long(), n_q=4), lambda: cache.append(x, pos, table[:, :1], n_q=4),
                lambda: cache.append(x, pos, table, n_q=4, q_norm=torch.ones(64, device="cuda")),
                lambda: cache.append(x, pos, table, n_q=4, out=torch.empty(2, 255, device="cuda")),
                lambda: cache.append(x, pos, table, n_q=4, seq=pos[:1]),
                lambda: cache.read(pos.long(), table), lambda: cache.read(pos, table, out=(x, x)),
                lambda: cache.read(pos, table, out=(torch.empty(2, 2, 64, device="cuda"), torch.empty(2, 3, 64, device="cuda")))):
        with pytest.raises(JoshuaB200Error):
            bad()
    assert cache.append(x[:0], pos[:0], table, n_q=4).shape == (0, 256)
    assert cache.read(pos[:0], table)[0].shape == (2, 0, 64)
