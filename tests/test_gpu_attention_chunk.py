"""Attention of chunks of new tokens over the paged cache, and with a window and sinks, against softmax in 64 bits over the values that
the cache reads back.

Tolerance: as for one token per sequence (tests/test_gpu_attention_paged.py): products of 16-bit terms carry 22 bits of a query or
probability and every bit of a code; a score is off by less than 1.5e-5 for the scores of these inputs (below 40), sums are f32: 2e-5 of
the largest value.
"""
import numpy as np
import pytest

from tests.test_gpu_attention_paged import TOL, fill, queries
from tests.test_gpu_kv_cache import KINDS, i32, make

pytestmark = pytest.mark.gpu


def sees(p, window, sinks):
    """Positions that the token at position p sees."""
    t = np.arange(p + 1)
    return t if not window else t[(t > p - window) | (t < sinks)]


def plain(q, k, v, pos, window=0, sinks=0, scale=None):
    """q [rows, n_q, hd] at positions pos; k, v [n_kv, n, hd] -> [rows, n_q, hd] in 64 bits."""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    rows, n_q, hd = q.shape
    g, out = n_q // k.shape[0], np.zeros(q.shape)
    for r, p in enumerate(pos):
        t = sees(p, window, sinks)
        kk, vv, x = k[:, t], v[:, t], q[r].reshape(-1, g, hd)
        s = np.einsum("hgd,htd->hgt", x, kk) * (scale if scale is not None else 1 / np.sqrt(hd))
        e = np.exp(s - s.max(-1, keepdims=True))
        out[r] = np.einsum("hgt,htd->hgd", e / e.sum(-1, keepdims=True), vv).reshape(n_q, hd)
    return out


def starts(counts):
    return i32(np.concatenate(([0], np.cumsum(counts))).astype(np.int32))


def compare(got, q, kv, counts, lens, n_q, hd, window=0, sinks=0, scale=None, tol=TOL, first=0):
    got, q, row = got.cpu().numpy().reshape(-1, n_q, hd), q.cpu().numpy().reshape(-1, n_q, hd), first
    for b, (n, length, (k, v)) in enumerate(zip(counts, lens, kv)):
        if n and length:
            want = plain(q[row:row + n], k, v, range(length - n, length), window, sinks, scale)
            err = np.abs(got[row:row + n] - want).max() / np.abs(v).max()
            assert err <= tol, (b, n, length, err)
        elif n:
            assert (got[row:row + n] == 0).all()
        row += n


LENGTHS = [(1, 1), (1, 64), (5, 5), (3, 130), (64, 64), (1, 65), (17, 257), (0, 0), (40, 190), (2, 63), (1, 0), (129, 200)]  # new, in all


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n_q,n_kv", [(4, 4), (8, 2), (6, 2), (8, 1), (20, 1), (14, 2)])
def test_lengths_and_heads(kind, hd, n_q, n_kv):
    counts, lens = zip(*LENGTHS)
    cache, table = make(kind, n_kv, hd, len(lens), 5, seed=n_q)
    kv = fill(cache, table, lens, seed=hd)
    q = queries(sum(counts), n_q, hd, 1)
    got = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts))
    compare(got, q, kv, counts, lens, n_q, hd)
    for _ in range(3):  # the scratch is left as it has to be, and nothing depends on who comes last
        assert bool((cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts)) == got).all())
    cache.check_flags()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (16, 0), (64, 64), (65, 4), (100, 70), (200, 1000), (5000, 4), (130, 17)])
def test_windows(kind, hd, window, sinks):
    """Chunks and single tokens; pages that nobody sees are not in the table."""
    n_q, n_kv = 8, 2
    counts, lens = [1, 9, 70, 1, 1, 33, 2], [300, 290, 320, 1, 64, 33, 258]
    cache, table = make(kind, n_kv, hd, len(lens), 5, seed=window)
    kv = fill(cache, table, lens, seed=hd)
    for b, (n, length) in enumerate(zip(counts, lens)):
        low = max(0, length - n + 1 - window)
        for page in range(table.shape[1]):
            if page * 64 >= length or (page * 64 >= sinks and page * 64 + 63 < low):
                table[b, page] = -1 - page
    q = queries(sum(counts), n_q, hd, 2)
    got = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts), window=window, sinks=sinks)
    compare(got, q, kv, counts, lens, n_q, hd, window, sinks)
    one = queries(len(lens), n_q, hd, 3)
    compare(cache.attend(one, i32(lens), table, n_q=n_q, window=window, sinks=sinks), one, kv, [1] * len(lens), lens, n_q, hd, window, sinks)
    cache.check_flags()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("counts,lens,n_q,n_kv,hd,window", [
    ([700], [700], 8, 2, 128, 0), ([300], [2500], 8, 1, 128, 0), ([1], [3000], 4, 4, 64, 0), ([1000, 1, 1, 300], [1300, 1700, 5, 2000], 6, 2, 64, 0),
    ([4] * 40, [100 + 37 * b for b in range(40)], 8, 2, 128, 0), ([300, 257], [2000, 300], 32, 4, 128, 500), ([1] * 150, [70 + b for b in range(150)], 8, 2, 64, 50),
    ([129], [1200], 34, 2, 128, 0), ([130, 5], [800, 700], 12, 4, 128, 300), ([200], [1000], 130, 1, 64, 0)])
def test_longer_ones(kind, counts, lens, n_q, n_kv, hd, window):
    cache, table = make(kind, n_kv, hd, len(lens), -(-max(lens) // 64))
    kv = fill(cache, table, lens, seed=5)
    q = queries(sum(counts), n_q, hd, 2)
    got = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts), window=window, sinks=5 if window else 0)
    compare(got, q, kv, counts, lens, n_q, hd, window, 5 if window else 0)
    again = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts), window=window, sinks=5 if window else 0)
    assert bool((got == again).all())
    cache.check_flags()


@pytest.mark.parametrize("n", [1, 3, 20, 150])
def test_as_many_rows_of_each(n):
    n_q, n_kv, hd, lens = 8, 2, 128, [200, 150, 333]
    cache, table = make("q8_0", n_kv, hd, 3, 6)
    kv = fill(cache, table, lens, seed=1)
    q = queries(3 * n, n_q, hd, 4)
    got = cache.attend_chunk(q, i32(lens), table, n_q=n_q)
    compare(got, q, kv, [n] * 3, lens, n_q, hd)
    told = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts([n] * 3))
    assert bool((got == told).all())


@pytest.mark.parametrize("hd", [128, 256])
def test_one_token_is_the_step_attention(hd):
    import torch

    lens = [1, 700, 64, 0, 333]
    cache, table = make("q8_0", 2, hd, 5, 11)
    fill(cache, table, lens, seed=1)
    q = queries(5, 8, hd, 4)
    a, b = cache.attend(q, i32(lens), table, n_q=8), cache.attend_chunk(q, i32(lens), table, n_q=8)
    assert float((a - b).abs().max()) <= TOL * 6
    assert bool((b[3] == 0).all())
    wide = torch.empty(5, 8 * hd + 64, device="cuda")
    cache.attend(q, i32(lens), table, n_q=8, window=100, sinks=2, out=wide[:, :8 * hd])
    assert bool((wide[:, :8 * hd] == cache.attend(q, i32(lens), table, n_q=8, window=100, sinks=2)).all())


@pytest.mark.parametrize("counts", [[3, 70], [1, 1]])
def test_rows_of_no_sequence_stay(counts):
    import torch

    n_q, n_kv, hd, lens = 8, 2, 128, [150, 200]
    cache, table = make("q8_0", n_kv, hd, 2, 4)
    kv = fill(cache, table, lens, seed=1)
    rows = sum(counts) + 12
    q = queries(rows, n_q, hd, 4)
    first = starts(counts) + 5
    out = torch.full((rows, n_q * hd + 32), 7.0, device="cuda")[:, 16:16 + n_q * hd]
    base = out._base
    cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=first, out=out)
    compare(out, q, kv, counts, lens, n_q, hd, first=5)
    assert bool((out[:5] == 7).all()) and bool((out[5 + sum(counts):] == 7).all()) and bool((base[:, :16] == 7).all()) and bool((base[:, -16:] == 7).all())
    q_wide = torch.full((rows, n_q * hd + 32), float("nan"), device="cuda")
    q_wide[:, :n_q * hd] = q
    again = cache.attend_chunk(q_wide[:, :n_q * hd], i32(lens), table, n_q=n_q, first=first)
    assert bool((again[5:5 + sum(counts)] == out[5:5 + sum(counts)]).all())
    cache.check_flags()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [2, 60])
def test_what_is_not_finite_stays_where_it_is_seen(kind, hd, n):
    """Keys and values of later tokens, outside the window or behind the end may be NaN or infinite."""
    import torch

    n_q, n_kv, length = 8, 2, 200
    cache, table = make(kind, n_kv, hd, 1, 5)
    cache.pages.fill_(0xFF)   # whatever a page held before: NaN scales, NaN halves
    kv = fill(cache, table, [length], seed=1)
    q = queries(n, n_q, hd, 4)
    for window, sinks in ((0, 0), (50, 3)):
        fine = cache.attend_chunk(q, i32([length]), table, n_q=n_q, window=window, sinks=sinks)
        compare(fine, q, kv, [n], [length], n_q, hd, window, sinks)
        saved = cache.pages.clone()
        for at, value in ((length - 1, float("nan")), (length - n, float("inf")), (20, float("nan"))):
            bad = queries(1, 3 * n_kv, hd, 9)
            bad[0, n_kv * hd] = value            # a key of kv head 0
            bad[0, 3 * n_kv * hd - 1] = value    # a value of the last head
            cache.append(bad, i32([at]), table, n_q=n_kv, seq=i32([0]))
            got = cache.attend_chunk(q, i32([length]), table, n_q=n_q, window=window, sinks=sinks).reshape(n, n_q, hd)
            see = torch.tensor([at in sees(length - n + r, window, sinks) for r in range(n)], device="cuda")
            lost = cache.read(i32([at]), table, seq=i32([0]))[1][n_kv - 1, 0].isnan()
            assert bool(got[see][:, :4].isnan().all())
            assert bool((got[see][:, 4:].isnan() == lost).all()) and bool(lost.any())
            ref = fine.reshape(n, n_q, hd)
            assert bool((got[~see] - ref[~see]).abs().max() <= 2 * TOL * 6) if bool((~see).any()) else True
            cache.pages.copy_(saved)
    cache.check_flags()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [0, 90])
def test_far_apart_scores(kind, window):
    """Scores hundreds apart, queries of zero, negative scales."""
    n_q, n_kv, hd, counts, lens = 8, 2, 128, [50, 1, 3], [300, 200, 180]

    def kv(b, k, v):
        k[7].mul_(20.0), k[100].mul_(20.0)

    cache, table = make(kind, n_kv, hd, 3, 5)
    held = fill(cache, table, lens, seed=1, kv=kv)
    q = queries(sum(counts), n_q, hd, 4)
    q[3] = 0.0
    for scale in (0.25, -0.25):
        got = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts), scale=scale, window=window, sinks=8 if window else 0)
        compare(got, q, held, counts, lens, n_q, hd, window, 8 if window else 0, scale, tol=20 * TOL)


def test_what_is_out_of_range():
    import torch

    n_q, n_kv, hd = 8, 2, 128
    counts, lens = [3, 40, 1, 50, 2, 33], [150, 130, 200, 100, 60, 64]
    cache, table = make("q8_0", n_kv, hd, 6, 4)
    kv = fill(cache, table, lens, seed=1)
    q = queries(sum(counts), n_q, hd, 4)
    fine = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts))
    cache.check_flags()
    at = np.concatenate(([0], np.cumsum(counts)))

    def only(which, lens=lens, table=table, first=None):
        got = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=first if first is not None else starts(counts))
        assert int(cache.bad_pos) == 1
        cache.bad_pos.zero_()
        for b in range(6):
            part = slice(at[b], at[b + 1])
            if b in which:
                assert bool(got[part].isnan().all()), b
            else:
                assert bool(((got[part] - fine[part]).abs() <= 2 * TOL * 6).all()), b   # cut up otherwise

    for b in range(6):
        for wrong in (-1, 257, counts[b] - 1):
            if wrong:
                only([b], lens=[wrong if i == b else n for i, n in enumerate(lens)])
        for wrong in (-1, cache.pages.shape[0], 2**31 - 1):
            t = table.clone()
            t[b, 0] = wrong   # seen by all rows
            only([b], table=t)
    out = torch.full_like(fine, 7.0)
    broken = starts(counts)
    broken[2] = int(broken[4]) + 1   # sequence 2 descends; 1 has more rows, the first one of 4 among them
    cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=broken, out=out)
    assert int(cache.bad_pos) == 1
    cache.bad_pos.zero_()
    for part in (slice(0, at[1]), slice(at[4] + 1, at[6])):
        assert bool(((out - fine)[part].abs() <= 2 * TOL * 6).all())
    broken = starts(counts)
    broken[6] = sum(counts) + 1
    out.fill_(7.0)
    cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=broken, out=out)
    assert int(cache.bad_pos) == 1 and bool((out[at[5]:] == 7).all()) and bool(((out - fine)[:at[5]].abs() <= 2 * TOL * 6).all())
    cache.bad_pos.zero_()
    again = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts))
    assert bool((again == fine).all())
    cache.check_flags()


def test_other_streams_and_graphs():
    """Calls on two streams, captured and replayed ones beside eager ones, a scratch of one's own."""
    import torch

    n_q, n_kv, hd, counts, lens = 8, 2, 128, [40, 1, 3, 200], [900, 800, 700, 1000]
    cache, table = make("q8_0", n_kv, hd, 4, 16)
    fill(cache, table, lens, seed=1)
    q, first, n = queries(sum(counts), n_q, hd, 4), starts(counts), i32(lens)
    want = cache.attend_chunk(q, n, table, n_q=n_q, first=first, window=500, sinks=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            outs.append(cache.attend_chunk(q, n, table, n_q=n_q, first=first, window=500, sinks=4))
    torch.cuda.synchronize()
    assert all(bool((o == want).all()) for o in outs)
    scratch = cache.scratch(4, n_q, rows=q.shape[0])
    assert bool((cache.attend_chunk(q, n, table, n_q=n_q, first=first, window=500, sinks=4, scratch=scratch) == want).all())
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(cache.attend_chunk(q, n, table, n_q=n_q, first=first, window=500, sinks=4))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        eager = cache.attend_chunk(q, n, table, n_q=n_q, first=first, window=500, sinks=4)
    torch.cuda.synchronize()
    assert all(bool((r == want).all()) for r in results) and bool((eager == want).all())
    lens2 = [700, 300, 600, 800]
    n.copy_(i32(lens2))
    want = cache.attend_chunk(q, n, table, n_q=n_q, first=first, window=500, sinks=4)
    graphs[0].replay()
    assert bool((results[0] == want).all())
    cache.check_flags()


def test_one_scratch_for_all_calls():
    """Calls of all sizes, both entries, through one scratch: larger and smaller ones in turn."""
    n_q, n_kv, hd = 8, 2, 128
    cache, table = make("q8_0", n_kv, hd, 4, 16)
    fill(cache, table, [1000] * 4, seed=1)
    scratch = cache.scratch(4, n_q, rows=400)
    for counts, lens in (([300, 1, 2, 50], [1000, 900, 50, 400]), ([1, 1, 1, 1], [1000, 3, 900, 20]), ([100] * 4, [100, 1000, 200, 700])) * 2:
        q = queries(sum(counts), n_q, hd, 4)
        got = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts), scratch=scratch)
        assert bool((got == cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts))).all())
        one = queries(4, n_q, hd, 5)
        assert bool((cache.attend(one, i32(lens), table, n_q=n_q, scratch=scratch) == cache.attend(one, i32(lens), table, n_q=n_q)).all())


def test_refusals():
    import torch

    from joshua_b200 import _lib
    from joshua_b200._lib import JoshuaB200Error

    n_q, n_kv, hd = 8, 2, 128
    cache, table = make("q8_0", n_kv, hd, 3, 4)
    fill(cache, table, [100] * 3, seed=1)
    q, lens, first = queries(9, n_q, hd, 4), i32([100] * 3), starts([3, 3, 3])

    def refused(*words, **change):
        args = dict(q=q, lens=lens, table=table, n_q=n_q, first=first)
        args.update(change)
        with pytest.raises(JoshuaB200Error) as e:
            cache.attend_chunk(**args)
        assert e.value.code == _lib.E_INVALID and all(w in str(e.value) for w in words), str(e.value)

    refused("q", q=q.double()), refused("q", q=q[:, :-1]), refused("q", q=q.cpu()), refused("q", q=q.t().contiguous().t())
    refused("lens", lens=lens[:2]), refused("lens", lens=lens.long()), refused("first", first=first[:3]), refused("first", first=first.long())
    refused("table", table=table.long()), refused("out", out=torch.empty(9, n_q * hd + 4, device="cuda"))
    refused("rows of out", out=torch.empty(8, n_q * hd, device="cuda"))
    refused("equal parts", first=None, q=q[:8])
    refused("query heads", n_q=3, q=queries(9, 3, hd, 1))
    for window, sinks in ((-1, 0), (0, 3), (5, -1), (2**31, 0)):
        refused("window", window=window, sinks=sinks)
    refused("scale", scale=float("nan")), refused("scale", scale=float("inf"))
    refused("scratch", scratch=torch.empty(16, device="cuda")), refused("scratch", scratch=cache.scratch(3, n_q, rows=9).cpu())
    with pytest.raises(JoshuaB200Error):
        cache.attend(q[:3], lens, table, n_q=n_q, window=5, shared_pages=1)
    with pytest.raises(JoshuaB200Error):
        cache.attend(q, lens, table, n_q=n_q, window=5)
    with pytest.raises(JoshuaB200Error):
        cache.attend(q[:3], lens, table, n_q=n_q, sinks=5)
    assert cache.attend_chunk(q[:0], lens, table, n_q=n_q, first=first).shape == (0, n_q * hd)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("size", [2.0**8, 2.0**14, 2.0**20, 2.0**26])
def test_scores_far_from_zero(kind, hd, window, size):
    """Scores of up to many millions: what stands out by more than two scores' rounding takes all (products of 22 bits, sums of 23:
    2^-20.4 of the magnitudes added up, which are below 4 times the largest score here: 2^-17.4), and every
    output stays within the values."""
    n_q, n_kv, counts, lens, sinks = 8, 2, [50, 1, 3, 200], [300, 200, 180, 200], 8 if window else 0
    cache, table = make(kind, n_kv, hd, 4, 5)
    held = fill(cache, table, lens, seed=2)
    q = queries(sum(counts), n_q, hd, 5)
    scale = size / np.sqrt(hd)
    got = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts), scale=scale, window=window, sinks=sinks).cpu().numpy()
    got, x, row, clear = got.reshape(-1, n_q, hd), q.cpu().numpy().astype(np.float64).reshape(-1, n_q, hd), 0, 0
    for n, length, (k, v) in zip(counts, lens, held):
        k, v = (np.asarray(t, dtype=np.float64) for t in (k, v))
        for r in range(n):
            t = sees(length - n + r, window, sinks)
            s = np.einsum("hgd,htd->hgt", x[row].reshape(n_kv, -1, hd), k[:, t]) * scale
            for h in range(n_kv):
                vv, out, top = v[h][t], got[row].reshape(n_kv, -1, hd)[h], np.abs(s[h]).max()
                slack = TOL * np.abs(v).max()
                assert np.isfinite(out).all() and (out >= vv.min(0) - slack).all() and (out <= vv.max(0) + slack).all()
                for j in range(out.shape[0]):
                    order = np.argsort(s[h, j])
                    if len(t) == 1 or s[h, j][order[-1]] - s[h, j][order[-2]] > 2.0**-17 * top + 20:   # e^-20 of the rest
                        assert np.abs(out[j] - vv[order[-1]]).max() <= slack, (row, h, j)
                        clear += 1
            row += 1
    assert clear > (0 if size < 2.0**10 else sum(counts) * n_q // 2)


def test_columns_of_one_buffer():
    """Queries and results beside each other in wider rows; in the same place they are refused."""
    import torch

    from joshua_b200._lib import JoshuaB200Error

    n_q, n_kv, hd, counts, lens = 8, 2, 64, [20, 1, 5], [100, 64, 65]
    cache, table = make("q8_0", n_kv, hd, 3, 3)
    fill(cache, table, lens, seed=1)
    q = queries(sum(counts), n_q, hd, 4)
    want = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts))
    for at, to in ((0, 512), (516, 0), (0, 600)):
        wide = torch.full((26, 1112), 7.0, device="cuda")
        wide[:, at:at + 512] = q
        got = wide[:, to:to + 512]
        cache.attend_chunk(wide[:, at:at + 512], i32(lens), table, n_q=n_q, first=starts(counts), out=got)
        assert bool((got == want).all()) and bool((wide[:, at:at + 512] == q).all())
        beside = torch.ones(1112, dtype=torch.bool)
        beside[at:at + 512] = beside[to:to + 512] = False
        assert bool((wide[:, beside.cuda()] == 7.0).all())
        for step in (0, 256, -256):
            if 0 <= at + step <= 600:
                with pytest.raises(JoshuaB200Error):
                    cache.attend_chunk(wide[:, at:at + 512], i32(lens), table, n_q=n_q, first=starts(counts), out=wide[:, at + step:at + step + 512])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n_q,hd", [(160, 64), (256, 128), (129, 128)])
def test_many_heads_on_one(kind, n_q, hd):
    """More query heads on a kv head than a tile has rows; tables that are full to the last position."""
    counts, lens = [3, 40, 1], [130, 320, 320]
    cache, table = make(kind, 1, hd, 3, 5)
    kv = fill(cache, table, lens, seed=3)
    q = queries(sum(counts), n_q, hd, 4)
    for window, sinks in ((0, 0), (70, 3)):
        got = cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts), window=window, sinks=sinks)
        compare(got, q, kv, counts, lens, n_q, hd, window, sinks)
    cache.check_flags()


def test_pages_behind_four_gigabytes():
    import torch

    from joshua_b200.kv_cache import PagedCache

    n_q, n_kv, hd, per, counts, lens = 8, 4, 128, 9, [70, 2, 1], [500, 500, 576]
    n_pages = 2**32 // (n_kv * 2 * 64 * (hd + hd // 16)) + 3 * per
    cache = PagedCache("q8_0", n_kv, hd, n_pages=n_pages, device="cuda")
    assert (n_pages - 3 * per + 1) * cache.page_bytes > 2**32
    table = torch.arange(n_pages - 3 * per, n_pages, device="cuda").int().flip(0).reshape(3, per).contiguous()
    kv = fill(cache, table, lens, seed=5)
    q = queries(sum(counts), n_q, hd, 6)
    for window, sinks in ((0, 0), (100, 4)):
        compare(cache.attend_chunk(q, i32(lens), table, n_q=n_q, first=starts(counts), window=window, sinks=sinks), q, kv, counts, lens, n_q, hd, window,
                sinks)
    cache.check_flags()


def test_wide_rows():
    """Queries and results whose last rows begin behind 2^32 bytes."""
    import torch

    n_q, n_kv, hd, counts, lens = 8, 2, 128, [60, 3, 1], [200, 130, 64]
    cache, table = make("f16", n_kv, hd, 3, 4)
    kv = fill(cache, table, lens, seed=5)
    q = queries(sum(counts), n_q, hd, 6)
    stride = 2**24 + 2**20 + 4
    far = torch.empty(63 * stride + 2 * 1024, device="cuda")
    rows = torch.as_strided(far, (64, 1024), (stride, 1))
    out = torch.as_strided(far, (64, 1024), (stride, 1), 1024)
    rows.copy_(q)
    assert cache.attend_chunk(rows, i32(lens), table, n_q=n_q, first=starts(counts), out=out) is out
    compare(out.contiguous(), q, kv, counts, lens, n_q, hd)
