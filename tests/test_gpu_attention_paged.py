"""Attention over the paged cache against softmax(q K^T) V in 64 bits over the values that the cache reads back.

Tolerance: products of 16-bit terms carry 22 bits of a query or probability and every bit of a code, sums are f32.  A score of
size |s| is off by at most hd 2^-22 of the sum of its products' sizes, in all below 2^-22 * 64 |q| |k| / sqrt(hd); with the scores of these
inputs (below 40) that is below 1.5e-5 of a probability, and rounding the output's sums adds under 1e-6: 2e-5 of the largest
value a row of V holds.
"""
import numpy as np
import pytest

from joshua_b200 import _lib
from joshua_b200._lib import JoshuaB200Error
from tests import serving_ref as ref
from tests.test_gpu_kv_cache import KINDS, i32, make

pytestmark = pytest.mark.gpu
TOL = 2e-5


def fill(cache, table, lens, seed, kv=None, scale=1.0):
    """Rows for positions 0 .. len - 1 of every sequence, through `append`; (keys, values) per sequence as read back."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    n_kv, hd, out = cache.n_kv, cache.head_dim, []
    for b, n in enumerate(lens):
        if n:
            x = torch.randn(n, 3 * n_kv * hd, device="cuda", generator=g) * scale
            if kv is not None:
                kv(b, x[:, n_kv * hd:2 * n_kv * hd], x[:, 2 * n_kv * hd:])
            cache.append(x, i32(range(n)), table, n_q=n_kv, seq=i32([b] * n))
        out.append(tuple(t.cpu().numpy() for t in cache.read(i32(range(n)), table, seq=i32([b] * n))))
    return out


def queries(batch, n_q, hd, seed, scale=1.0):
    import torch

    return torch.randn(batch, n_q * hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * scale


def expect(got, q, kv, n_q, hd, scale=None, tol=TOL):
    got, q = got.cpu().numpy().reshape(-1, n_q, hd), q.cpu().numpy().reshape(-1, n_q, hd)
    for b, (k, v) in enumerate(kv):
        want = ref.attention(q[b], k, v, scale if scale is not None else 1 / np.sqrt(hd))
        top = max(np.abs(v).max(), 1e-30) if v.size else 1.0
        assert np.abs(got[b] - want).max() <= tol * top, (b, k.shape, np.abs(got[b] - want).max() / top)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n_q,n_kv", [(4, 4), (8, 2), (6, 2), (8, 1), (12, 1), (20, 1), (34, 2)])
def test_lengths_and_heads(kind, hd, n_q, n_kv):
    lens = [1, 63, 64, 65, 130, 0, 16, 17, 257]
    cache, table = make(kind, n_kv, hd, len(lens), 5, seed=n_q)
    kv = fill(cache, table, lens, seed=hd)
    q = queries(len(lens), n_q, hd, 1)
    got = cache.attend(q, i32(lens), table, n_q=n_q)
    expect(got, q, kv, n_q, hd)
    assert bool((got[5] == 0).all())
    for _ in range(3):  # the scratch is left as it has to be
        assert np.array_equal(cache.attend(q, i32(lens), table, n_q=n_q).cpu().numpy(), got.cpu().numpy())
    cache.check_flags()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch,length", [(1, 1), (1, 700), (1, 5000), (3, 2000), (200, 70), (40, 129)])
def test_batches(kind, batch, length):
    n_q, n_kv, hd = 8, 2, 128
    lens = [max(0, length - 37 * (b % 5) - b) for b in range(batch)]
    cache, table = make(kind, n_kv, hd, batch, -(-length // 64))
    kv = fill(cache, table, lens, seed=batch)
    q = queries(batch, n_q, hd, 2)
    expect(cache.attend(q, i32(lens), table, n_q=n_q), q, kv, n_q, hd)


def long_prompt(kind, hd, n_q, n_kv, batch, shared, seed=3, kv=None):
    """A common prompt of `shared` pages (seven of them, again and again) and up to three pages of each sequence's own."""
    import torch

    cache, table = make(kind, n_kv, hd, batch, 10, seed=seed)
    fill(cache, table, [640] * batch, seed=seed, kv=kv)
    common = table[0, torch.arange(shared, device="cuda") % 7].expand(batch, shared)
    table = torch.cat([common, table[:, 7:]], 1).contiguous()
    lens = [shared * 64 + (0, 1, 64, 100, 130, 192)[b % 6] for b in range(batch)]
    lens[3] = 0
    return cache, table, lens, queries(batch, n_q, hd, seed + 1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,n_q,n_kv,batch,shared", [
    (128, 32, 8, 32, 20), (128, 8, 2, 33, 100), (64, 24, 2, 40, 75), (64, 8, 8, 40, 33), (128, 16, 1, 32, 150), (128, 9, 3, 60, 41), (64, 64, 8, 129, 5),
    (128, 4, 4, 8, 200), (128, 4, 4, 31, 41), (64, 8, 4, 13, 270), (64, 7, 7, 6, 330), (256, 8, 2, 48, 97), (256, 2, 2, 20, 70), (256, 4, 2, 33, 50)])
def test_long_shared_prompts(kind, hd, n_q, n_kv, batch, shared):
    """Prompts that are worth a pass of their own: the same as each sequence by itself."""
    cache, table, lens, q = long_prompt(kind, hd, n_q, n_kv, batch, shared)
    got = cache.attend(q, i32(lens), table, n_q=n_q, shared_pages=shared)
    for b in sorted({0, 2, 3, batch // 2, batch - 1}):
        kv = tuple(t.cpu().numpy() for t in cache.read(i32(range(lens[b])), table, seq=i32([b] * lens[b])))
        expect(got[b:b + 1], q[b:b + 1], [kv], n_q, hd)
    alone = cache.attend(q, i32(lens), table, n_q=n_q)
    assert float((got - alone).abs().max()) <= 2 * TOL * 6   # values of these inputs are below 6
    assert bool((got == cache.attend(q, i32(lens), table, n_q=n_q, shared_pages=shared)).all())
    cache.check_flags()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,n_q,n_kv,batch,shared", [(128, 32, 8, 32, 20), (64, 24, 2, 40, 75), (128, 4, 4, 8, 200), (256, 2, 2, 20, 70)])
def test_long_shared_prompts_that_go_wrong(kind, hd, n_q, n_kv, batch, shared):
    """Lengths below the prompt, NaN and infinities in it, scores that differ by hundreds, queries of zero, shared pages outside
    the cache."""
    def kv(b, k, v):
        k[7].mul_(20.0)

    cache, table, lens, q = long_prompt(kind, hd, n_q, n_kv, batch, shared, kv=kv)
    q[4] = 0.0
    lens[5], lens[2] = shared * 64 - 1, -3
    got = cache.attend(q, i32(lens), table, n_q=n_q, scale=0.25, shared_pages=shared)
    assert bool(got[[2, 5]].isnan().all()) and bool((got[3] == 0).all()) and int(cache.bad_pos) == 1
    for b in (0, 4, batch - 1):
        held = tuple(t.cpu().numpy() for t in cache.read(i32(range(lens[b])), table, seq=i32([b] * lens[b])))
        expect(got[b:b + 1], q[b:b + 1], [held], n_q, hd, scale=0.25, tol=20 * TOL)
    cache.bad_pos.zero_()
    lens[5], lens[2] = shared * 64 + 1, shared * 64
    bad = queries(1, 3 * n_kv, hd, 9)
    cache.append(bad, i32([70]), table, n_q=n_kv, seq=i32([0]))
    fine = cache.attend(q, i32(lens), table, n_q=n_q, shared_pages=shared)
    bad[0, n_kv * hd] = np.nan                       # a key of kv head 0, a value of the last one
    bad[0, 3 * n_kv * hd - 1] = np.inf
    cache.append(bad, i32([70]), table, n_q=n_kv, seq=i32([0]))
    got = cache.attend(q, i32(lens), table, n_q=n_q, shared_pages=shared).reshape(batch, n_q, hd)
    group = n_q // n_kv
    held = cache.read(i32([70]), table, seq=i32([0]))
    live = [b for b in range(batch) if b != 3]
    assert bool(got[live, :group].isnan().all()) and bool((got[3] == 0).all())
    lost = held[1][n_kv - 1, 0].isnan()
    assert bool((got[live][:, n_q - group:].isnan() == lost).all()) and bool(lost.any())
    if n_kv > 2:
        assert bool((got[:, group:n_q - group] - fine.reshape(batch, n_q, hd)[:, group:n_q - group]).abs().max() <= 2 * TOL * 6)
    assert int(cache.bad_pos) == 0
    for page in (-1, cache.pages.shape[0]):
        table[:, shared // 2] = page
        got = cache.attend(q, i32(lens), table, n_q=n_q, shared_pages=shared)
        assert bool(got[live].isnan().all()) and bool((got[3] == 0).all()) and int(cache.bad_pos) == 1


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,n_q,n_kv,batch,shared", [(128, 8, 2, 5, 1), (128, 32, 8, 32, 3), (64, 8, 2, 33, 4), (256, 8, 2, 9, 2),
                                                      (64, 4, 4, 2, 9), (128, 9, 3, 7, 5), (128, 16, 1, 3, 2), (64, 8, 8, 130, 1), (128, 32, 8, 100, 9),
                                                      (64, 16, 2, 9, 40), (128, 8, 1, 33, 33)])
def test_shared_pages(kind, hd, n_q, n_kv, batch, shared):
    """Sequences behind a common prompt: the same as each by itself, some with nothing of their own, one inactive."""
    import torch

    per = shared + 3
    lens = [shared * 64 + (0, 1, 64, 100, 130)[b % 5] for b in range(batch)]
    if batch > 4:
        lens[3] = 0
    cache, table = make(kind, n_kv, hd, batch, per)
    table[:, :shared] = table[0, :shared]
    kv = fill(cache, table, lens, seed=3)       # the last one to write the common pages wrote for all
    kv = [tuple(t.cpu().numpy() for t in cache.read(i32(range(n)), table, seq=i32([b] * n))) for b, n in enumerate(lens)]
    q = queries(batch, n_q, hd, 4)
    got = cache.attend(q, i32(lens), table, n_q=n_q, shared_pages=shared)
    expect(got, q, kv, n_q, hd)
    expect(cache.attend(q, i32(lens), table, n_q=n_q), q, kv, n_q, hd)
    assert torch.equal(got, cache.attend(q, i32(lens), table, n_q=n_q, shared_pages=shared))
    cache.check_flags()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,n_q,n_kv", [(64, 8, 1), (128, 4, 4), (128, 16, 2), (128, 9, 1), (256, 8, 2), (256, 6, 1)])
def test_sequences_that_span_ctas(kind, hd, n_q, n_kv):
    """Some cut between CTAs, some whole in one, some with nothing; the same answer again from the same scratch."""
    lens = [3001, 1, 0, 1999, 703, 64, 1600]
    cache, table = make(kind, n_kv, hd, len(lens), 47, seed=n_q)
    kv = fill(cache, table, lens, seed=hd)
    q = queries(len(lens), n_q, hd, 3)
    got = cache.attend(q, i32(lens), table, n_q=n_q)
    expect(got, q, kv, n_q, hd)
    for _ in range(3):
        assert bool((got == cache.attend(q, i32(lens), table, n_q=n_q)).all())


@pytest.mark.parametrize("kind", KINDS)
def test_a_long_sequence(kind):
    """Many splits, a batch of very unlike lengths."""
    n_q, n_kv, hd, lens = 8, 2, 64, [30011, 3, 0, 64 * 40, 1]
    cache, table = make(kind, n_kv, hd, len(lens), 470)
    kv = fill(cache, table, lens, seed=11)
    q = queries(len(lens), n_q, hd, 5)
    expect(cache.attend(q, i32(lens), table, n_q=n_q), q, kv, n_q, hd)


@pytest.mark.parametrize("kind", KINDS)
def test_scales_and_sizes(kind):
    """Scores that differ by hundreds, tiny and huge values, a scale of the caller's."""
    n_q, n_kv, hd, lens = 4, 2, 128, [300, 200, 100]
    cache, table = make(kind, n_kv, hd, 3, 5)

    def kv(b, k, v):
        v.mul_((1e-5, 1e4, 1.0)[b])
        k[7].mul_(20.0)

    held = fill(cache, table, lens, seed=21, kv=kv)
    q = queries(3, n_q, hd, 6)
    expect(cache.attend(q, i32(lens), table, n_q=n_q, scale=0.25), q, held, n_q, hd, scale=0.25, tol=20 * TOL)  # scores 20 times as large
    tiny = q * 1e-30
    expect(cache.attend(tiny, i32(lens), table, n_q=n_q), tiny, held, n_q, hd)


@pytest.mark.parametrize("kind", KINDS)
def test_rubbish_behind_the_end(kind):
    """Pages hold NaN and infinities behind the last position (`make` fills them with random bytes; here all of them are NaN):
    nothing of it shows, wherever the sequence ends."""
    n_q, n_kv, hd = 8, 2, 128
    for n in (1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 95):
        cache, table = make(kind, n_kv, hd, 1, 2)
        cache.pages.fill_(0xFF)   # halves, scales: NaN
        kv = fill(cache, table, [n], seed=n)
        q = queries(1, n_q, hd, n)
        expect(cache.attend(q, i32([n]), table, n_q=n_q), q, kv, n_q, hd)


@pytest.mark.parametrize("kind", KINDS)
def test_values_that_are_not_finite_show(kind):
    """A NaN key makes the scores of its kv head NaN; a NaN value the dimensions that hold it; other heads and sequences stay."""
    n_q, n_kv, hd, lens = 4, 2, 64, [90, 90, 90]
    cache, table = make(kind, n_kv, hd, 3, 2)

    def kv(b, k, v):
        if b == 0:
            k[80, 3] = np.nan           # head 0
        if b == 1:
            v[5, hd + 40] = np.inf      # head 1, second block

    held = fill(cache, table, lens, seed=31, kv=kv)
    q = queries(3, n_q, hd, 7)
    got = cache.attend(q, i32(lens), table, n_q=n_q).cpu().numpy().reshape(3, n_q, hd)
    with np.errstate(all="ignore"):
        want = np.stack([ref.attention(q.cpu().numpy().reshape(3, n_q, hd)[b], *held[b], 1 / np.sqrt(hd)) for b in range(3)])
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.nanmax(np.abs(got - want)) <= TOL * 6


@pytest.mark.parametrize("shared", [0, 45])
def test_a_pool_past_32_bits(shared):
    """Pages from 4 GB on: appended, read and attended, by themselves and as a common prompt."""
    import torch

    from joshua_b200.kv_cache import PagedCache

    n_q, n_kv, hd, batch, per = 16, 8, 128, 32, 48
    n_pages = 2**32 // (n_kv * 2 * 64 * (hd + hd // 16)) + batch * per
    cache = PagedCache("q8_0", n_kv, hd, n_pages=n_pages, device="cuda")
    assert (n_pages - batch * per + 1) * cache.page_bytes > 2**32
    table = (n_pages - 1 - torch.randperm(batch * per, device="cuda")).int().reshape(batch, per)
    if shared:
        table[:, :shared] = table[0, :shared].clone()
    lens = [(shared or 40) * 64 + 3 * b for b in range(batch)]
    kv = fill(cache, table, lens, seed=5)
    q = queries(batch, n_q, hd, 6)
    got = cache.attend(q, i32(lens), table, n_q=n_q, shared_pages=shared)
    for b in (0, 7, batch - 1):
        held = tuple(t.cpu().numpy() for t in cache.read(i32(range(lens[b])), table, seq=i32([b] * lens[b])))
        assert shared or all(np.array_equal(x, y) for x, y in zip(held, kv[b]))
        expect(got[b:b + 1], q[b:b + 1], [held], n_q, hd)
    cache.check_flags()


def test_lengths_and_pages_without_a_place():
    import torch

    n_q, n_kv, hd, lens = 4, 2, 64, [100, 100, 100, 100, 100]
    cache, table = make("q8_0", n_kv, hd, 5, 2)
    kv = fill(cache, table, lens, seed=41)
    q = queries(5, n_q, hd, 8)
    table[3, 1] = cache.pages.shape[0]
    table[4, 1] = -7
    got = cache.attend(q, i32([-1, 129, 100, 100, 100]), table, n_q=n_q)
    assert bool(got[[0, 1, 3, 4]].isnan().all())
    expect(got[2:3], q[2:3], kv[2:3], n_q, hd)
    with pytest.raises(JoshuaB200Error):
        cache.check_flags()
    table[3:, 1] = 0
    table[:, 0] = table[0, 0]
    got = cache.attend(q, i32([64, 63, 0, 100, 70]), table, n_q=n_q, shared_pages=1)   # 63: less than the shared page
    assert bool(got[1].isnan().all()) and not bool(got[[0, 3, 4]].isnan().any()) and bool((got[2] == 0).all())
    assert int(cache.bad_pos) == 1
    got = cache.attend(q, i32([64, 64, 0, 100, 70]), table, n_q=n_q, shared_pages=1)   # and the scratch is fine again
    assert not bool(got.isnan().any())
    table[:, 0] = -1   # a shared page outside the cache
    cache.bad_pos.zero_()
    got = cache.attend(q, i32([64, 64, 0, 100, 70]), table, n_q=n_q, shared_pages=1)
    assert bool(got[[0, 1, 3, 4]].isnan().all()) and bool((got[2] == 0).all()) and int(cache.bad_pos) == 1


def test_strided_rows_another_stream_and_a_graph():
    import torch

    n_q, n_kv, hd, lens = 8, 2, 128, [150, 1, 64, 300]
    cache, table = make("q4_0", n_kv, hd, 4, 5)
    fill(cache, table, lens, seed=51)
    q, n = queries(4, n_q, hd, 9), i32(lens)
    want = cache.attend(q, n, table, n_q=n_q)
    wide, into = torch.zeros(4, n_q * hd + 260, device="cuda"), torch.full((4, n_q * hd + 8), 2.0, device="cuda")
    wide[:, 128:128 + n_q * hd] = q
    cache.attend(wide[:, 128:128 + n_q * hd], n, table, n_q=n_q, out=into[:, 4:4 + n_q * hd])
    assert torch.equal(into[:, 4:4 + n_q * hd], want) and bool((into[:, :4] == 2).all()) and bool((into[:, 4 + n_q * hd:] == 2).all())
    torch.cuda.synchronize()
    side, scratch = torch.cuda.Stream(), cache.scratch(4, n_q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(cache.attend(q + 0, n, table, n_q=n_q, scratch=scratch), want)
        side.synchronize()
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
        with torch.cuda.graph(graph, stream=side):
            cache.attend(q, n, table, n_q=n_q, out=out, scratch=scratch)
    q.copy_(queries(4, n_q, hd, 10))
    n.copy_(i32([64, 1, 5, 299]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, cache.attend(q, n, table, n_q=n_q))


def test_refusals():
    import torch

    cache, table = make("q8_0", 2, 64, 2, 2)
    q, n = queries(2, 4, 64, 0), i32([1, 1])
    for bad in (lambda: cache.attend(q, n, table, n_q=3), lambda: cache.attend(q, n, table, n_q=8), lambda: cache.attend(q[:1], n, table, n_q=4),
                lambda: cache.attend(q, n[:1], table, n_q=4), lambda: cache.attend(q, n.long(), table, n_q=4),
                lambda: cache.attend(q, n, table[:1], n_q=4), lambda: cache.attend(q.half(), n, table, n_q=4),
                lambda: cache.attend(q, n, table, n_q=4, shared_pages=3), lambda: cache.attend(q, n, table, n_q=4, scale=float("nan")),
                lambda: cache.attend(q, n, table, n_q=4, out=torch.empty(2, 255, device="cuda"))):
        with pytest.raises(JoshuaB200Error):
            bad()
    assert cache.attend(q[:0], n[:0], table[:0], n_q=4).shape == (0, 256)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,n_q,n_kv,batch,shared", [(128, 32, 8, 32, 20), (64, 24, 2, 40, 75), (128, 4, 4, 8, 200), (256, 2, 2, 20, 70), (64, 8, 2, 3, 1)])
def test_a_negative_scale(kind, hd, n_q, n_kv, batch, shared):
    """On every route, with scores of both signs: |scale| and size of the scores as in the tests above."""
    cache, table, lens, q = long_prompt(kind, hd, n_q, n_kv, max(batch, 4), shared)
    got = cache.attend(q, i32(lens), table, n_q=n_q, scale=-0.2, shared_pages=shared)
    for b in (0, 1, 2, len(lens) - 1):
        held = tuple(t.cpu().numpy() for t in cache.read(i32(range(lens[b])), table, seq=i32([b] * lens[b])))
        expect(got[b:b + 1], q[b:b + 1], [held], n_q, hd, scale=-0.2, tol=4 * TOL)   # up to 3.2 times the scores of scale 1 / sqrt(hd)
    cache.check_flags()


def test_one_scratch_for_calls_of_all_sizes():
    """What one call leaves is what the next one needs, whatever their batches, lengths, heads and shared pages."""
    import torch

    hd, calls = 128, []
    for kind, n_q, n_kv, batch, length, shared in (("q8_0", 32, 8, 1, 3000, 0), ("q8_0", 32, 8, 100, 1700, 0), ("f16", 32, 8, 5, 900, 0), ("q8_0", 8, 2, 40, 300, 0),
                                                   ("q4_0", 32, 8, 32, 1500, 20), ("q8_0", 8, 2, 3, 5000, 0), ("q8_0", 32, 8, 32, 1400, 20)):
        cache, table = make(kind, n_kv, hd, batch, -(-length // 64))
        if shared:
            table[:, :shared] = table[0, :shared].clone()
        lens = [length - b for b in range(batch)]
        fill(cache, table, lens, seed=batch)
        q = queries(batch, n_q, hd, batch)
        n = i32(lens)
        calls.append((cache, q, n, table, n_q, shared, cache.attend(q, n, table, n_q=n_q, shared_pages=shared)))
    big = max((c.scratch(q.shape[0], n_q, shared) for c, q, _, _, n_q, shared, _ in calls), key=lambda s: s.numel())
    for turn in range(3):
        for c, q, n, table, n_q, shared, want in calls[::-1 if turn % 2 else 1]:
            got = torch.full_like(want, 7.0)
            assert torch.equal(c.attend(q, n, table, n_q=n_q, shared_pages=shared, out=got, scratch=big), want)


def test_a_cache_keeps_one_scratch_a_stream():
    import torch

    cache, table = make("q8_0", 8, 128, 32, 24)
    table[:, :20] = table[0, :20].clone()
    lens = i32([1400] * 32)
    fill(cache, table, [1400] * 32, seed=1)
    q = queries(32, 32, 128, 2)
    before = cache.attend(q, lens, table, n_q=32)
    kept = torch.cuda.memory_allocated()
    for shared in range(21):
        for batch in (32, 7, 1):
            cache.attend(q[:batch], lens[:batch], table[:batch], n_q=32, shared_pages=shared, out=torch.empty_like(q[:batch]))
    assert torch.cuda.memory_allocated() - kept <= 4 * cache.scratch(32, 32, 20).numel()
    assert torch.equal(before, cache.attend(q, lens, table, n_q=32))


def test_a_scratch_that_will_not_do():
    import torch

    cache, table = make("q8_0", 8, 128, 32, 24)
    q, n = queries(32, 32, 128, 0), i32([1] * 32)
    fill(cache, table, [1] * 32, seed=1)
    fine = cache.scratch(32, 32, 20)
    small = cache.scratch(32, 32)
    assert small.numel() < fine.numel()
    for bad in (small, fine[:fine.numel() // 2], fine.cpu(), fine[::2], fine[1:], 5, torch.zeros(0, device="cuda")):
        with pytest.raises(JoshuaB200Error, match="scratch"):
            cache.attend(q, n, table, n_q=32, shared_pages=20, scratch=bad)
    whole = torch.zeros(fine.numel() * 4, dtype=torch.uint8, device="cuda")      # of any type
    assert torch.equal(cache.attend(q, n, table, n_q=32, scratch=whole), cache.attend(q, n, table, n_q=32, scratch=small))
