"""Log probabilities, entropy and the likeliest tokens against 64 bits.

Tolerance: l - max is exact or rounded once (2^-24 of it); exp2 of a product with log2(e), rounded once at size |x| <= 150 where it
still counts, is off by 2^-24 * 1.45 * |l - max| plus 2^-22; a thread's sum has at most 512 additions of positive terms and the
joining 12 more, each 2^-24: a sum is off by less than 2^-15 of itself in the worst case and 2^-19 on the average of roundings.  A
logarithm of the sum then is off by at most 3.1e-5 if all roundings went one way, of these inputs by far less; 4e-6 beside the
rounding of the result itself (2^-23 of its size) is asked for.  The entropy's sum has factors |l - max|, so the same times its own size.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
TOL = 4e-6


def plain(l, token, top):
    """One row in 64 bits: (log p, entropy, ids, log p of the ids)."""
    x = np.where(np.isnan(l), -np.inf, np.minimum(l.astype(np.float64), np.finfo(np.float32).max))
    some = np.flatnonzero(x > -np.inf)
    if len(some) == 0:
        lp, entropy = np.full(len(x), -np.inf), 0.0
    else:
        d = x - x.max()
        with np.errstate(all="ignore"):
            e = np.exp(d)
        others = np.delete(e, np.argmax(x)).sum()
        log_s = np.log1p(others)
        lp = d - log_s
        entropy = log_s - (e[some] * d[some]).sum() / (1 + others)
    order = some[np.lexsort((some, -x[some]))][:top]
    ids = np.full(top, -1)
    ids[:len(order)] = order
    best = np.full(top, -np.inf)
    best[:len(order)] = lp[order]
    given = lp[token] if 0 <= token < len(x) else np.nan
    return given, entropy, ids, best


def check(logits, token, top, tol=TOL):
    import torch

    from joshua_b200.sampling import log_probs

    got = log_probs(logits, token, top=top)
    given, entropy, ids, best = (t.cpu().numpy() for t in got)
    for r, l in enumerate(logits.cpu().numpy()):
        want = plain(l, int(token[r]), top)
        with np.errstate(all="ignore"):
            for a, b in ((given[r], want[0]), (best[r], want[3])):
                near = np.abs(a - b) <= tol + 2.0**-23 * np.abs(b)
                assert np.all(near | (a == b) | (np.isnan(a) & np.isnan(b))), (r, a, b)
        assert abs(entropy[r] - want[1]) <= tol * max(1.0, want[1]), (r, entropy[r], want[1])
        assert np.array_equal(ids[r], want[2]), (r, ids[r], want[2])
    again = log_probs(logits, token, top=top)
    assert all(bool(((a == b) | a.isnan()).all()) for a, b in zip(got, again))
    return got


def normal(rows, vocab, seed, scale=2.5):
    import torch

    return torch.randn(rows, vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * scale


def tokens(rows, vocab, seed):
    import torch

    return torch.randint(0, vocab, (rows,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed), dtype=torch.int32)


@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (5, 33), (1, 4095), (2, 4096), (3, 4097), (1, 32000), (40, 32000), (1, 128256), (9, 151936),
                                        (200, 5000), (700, 100)])
def test_sizes(rows, vocab, top):
    check(normal(rows, vocab, vocab), tokens(rows, vocab, rows), top)


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("vocab,stride", [(7, 9), (5003, 5005), (70001, 70002)])
def test_rows_anywhere(offset, vocab, stride):
    """Rows that begin on any float, with others' numbers around them."""
    import torch

    base = torch.full((5 * stride + 8,), 1e30, device="cuda")
    l = base[offset:offset + 5 * stride].view(5, stride)[:, :vocab]
    l.copy_(normal(5, vocab, offset))
    check(l, tokens(5, vocab, 1), 8)


@pytest.mark.parametrize("vocab", [600, 20000, 130000])
def test_orders_and_ties(vocab):
    """Ascending, descending, all equal, few values, a block of large ones: the list is cut back again and again."""
    import torch

    up = torch.arange(vocab, device="cuda", dtype=torch.float32) / vocab * 20
    few = (torch.arange(vocab, device="cuda") * 7919 % 13).float()
    block = torch.zeros(vocab, device="cuda")
    block[vocab // 2:vocab // 2 + 300] = 5 + torch.arange(300, device="cuda") / 100
    zeros = torch.zeros(vocab, device="cuda")
    zeros[::3] = -0.0
    for top in (1, 20, 32):
        check(torch.stack((up, up.flip(0), zeros, few, block, -up * 4)), tokens(6, vocab, 3), top)


@pytest.mark.parametrize("vocab", [50, 9000, 100000])
def test_peaked_rows(vocab):
    """Nearly all of the weight on one token: 1 - p keeps its relative accuracy."""
    import torch

    l = normal(6, vocab, 1, scale=1.0)
    at = torch.tensor([0, 7, vocab - 1, vocab // 2, 33, 1], device="cuda")
    l[torch.arange(6, device="cuda"), at] = torch.tensor([25.0, 30, 40, 60, 200, 20], device="cuda")
    given, entropy, *_ = check(l, at.int(), 4)
    for r in range(6):
        want = plain(l[r].cpu().numpy(), int(at[r]), 1)
        assert abs(float(given[r]) - want[0]) <= 2e-5 * abs(want[0]) + 1e-37 and abs(float(entropy[r]) - want[1]) <= 2e-5 * want[1] + 1e-37


def test_what_is_not_finite():
    import torch

    nan, inf = float("nan"), float("inf")
    l = normal(10, 12000, 2)
    l[0] = -inf
    l[1] = nan
    l[2, 5:] = -inf
    l[3, ::2] = nan
    l[4, 100] = inf
    l[5, 3], l[5, 11000], l[5, 4] = inf, inf, -inf
    l[6, :9000] = -inf
    l[7] = -inf
    l[7, 11999] = -3.0e38
    l[8] = 3.4e38
    l[9, 0], l[9, 1:] = 1e30, -1e30
    token = torch.tensor([3, 3, 6, 3, 7, 4, 5, 11999, 0, 5], device="cuda", dtype=torch.int32)
    for top in (0, 8, 32):
        check(l, token, top, tol=1e-5)
    out = torch.tensor([-1, 12000, 2**31 - 1, 0, 100, 3, 11999, 0, 11999, -2**31], device="cuda", dtype=torch.int32)
    given = check(l, out, 0, tol=1e-5)[0]
    assert bool(given[[0, 1, 2, 9]].isnan().all()) and not bool(given[3:9].isnan().any())


def test_with_the_sampler():
    """A step as a server makes it: a token drawn, its log probability, others beside it; captured too."""
    import torch

    from joshua_b200.sampling import log_probs, sample

    l, u = normal(33, 128256, 5), torch.rand(33, device="cuda")

    def step():
        token, prob = sample(l, u)
        return token, prob, log_probs(l, token, top=5)

    token, prob, scores = step()
    # the sampler rounds weights to 2^-32 of the largest
    assert float((scores[0].exp() - prob).abs().max()) <= 1e-5
    greedy, _ = sample(l, u, temperature=torch.zeros(33, device="cuda"))
    assert bool((scores[2][:, 0] == greedy).all())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for seed in (6, 7):
        l.copy_(normal(33, 128256, seed))
        g.replay()
        eager = step()
        assert bool((captured[0] == eager[0]).all()) and all(bool((a == b).all()) for a, b in zip(captured[2], eager[2]))


def test_refusals():
    import torch

    from joshua_b200 import _lib
    from joshua_b200._lib import JoshuaB200Error
    from joshua_b200.sampling import log_probs

    l, t = normal(3, 100, 1), tokens(3, 100, 1)

    def refused(code, *args, **more):
        with pytest.raises(JoshuaB200Error) as e:
            log_probs(*args, **more)
        assert e.value.code == code

    refused(_lib.E_INVALID, l.double(), t), refused(_lib.E_INVALID, l.cpu(), t), refused(_lib.E_INVALID, l[0], t), refused(_lib.E_INVALID, l.t(), t)
    refused(_lib.E_INVALID, l, t.long()), refused(_lib.E_INVALID, l, t[:2]), refused(_lib.E_INVALID, l, t.cpu()), refused(_lib.E_INVALID, l, t, top=-1)
    refused(_lib.E_TOO_LARGE, l, t, top=33), refused(_lib.E_INVALID, l[:, :0], t)
    out = log_probs(l[:0], t[:0], top=3)
    assert [list(o.shape) for o in out] == [[0], [0], [0, 3], [0, 3]]


@pytest.mark.parametrize("rows,vocab,pad,top", [(1300, 2047, 3, 3), (1201, 2049, 2, 0), (610, 4098, 1, 32), (150, 40001, 5, 20), (75, 9000, 4, 7), (37, 70003, 0, 32)])
def test_rows_in_turn(rows, vocab, pad, top):
    """More rows than are worked on at a time, and rows in several slices, at all distances from a 16-byte boundary."""
    wide = normal(rows, vocab + pad, 7)
    check(wide[:, pad:], tokens(rows, vocab, 8), top)


@pytest.mark.parametrize("rows", [1, 40, 700])
def test_rising_rows(rows):
    """Every value above all before it: each list is cut back again and again."""
    import torch

    l = torch.linspace(-4, 4, 9001, device="cuda").repeat(rows, 1)
    l[::2] = l[::2].flip(1)
    check(l, tokens(rows, 9001, 3), 32)


def test_logits_behind_four_gigabytes():
    """Rows a long way apart, a plain call on a head's width at the end of them."""
    import torch

    from joshua_b200.sampling import log_probs

    rows, vocab, stride = 70, 9001, 2**24 + 1
    far = torch.empty((rows - 1) * stride + vocab, device="cuda")
    l = torch.as_strided(far, (rows, vocab), (stride, 1))
    plain_ones = normal(rows, vocab, 4)
    l.copy_(plain_ones)
    token = tokens(rows, vocab, 5)
    got = log_probs(l, token, top=5)
    check(plain_ones, token, 5)
    for a, b in zip(got, log_probs(plain_ones, token, top=5)):
        assert a.shape == b.shape and bool(((a - b).abs() <= (0 if a.dtype == torch.int32 else 2 * TOL)).all())
