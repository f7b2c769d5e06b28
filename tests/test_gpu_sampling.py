"""Sampling against the rules in 64 bits.

Which tokens are kept and drawn are whole numbers and have to be equal.  The reference's weights are 64-bit exponentials, the
device's f32 ones (a few 2^-24 off each, rounded to 2^-33 of the largest weight): cases where the draw or a rule's border lies
within 1e-5 of the sum of another token are not decided by the rules, and such rows are drawn anew by the test before they are
used.  Probabilities: 1e-5 of themselves.
"""
import numpy as np
import pytest

from joshua_b200 import _lib
from joshua_b200._lib import JoshuaB200Error
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu
NEAR, TOL = 1e-5, 1e-5


def dev(x, dtype):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda", dtype)


def run(l, u, temperature=None, top_k=None, top_p=None, min_p=None, **more):
    import torch

    from joshua_b200.sampling import sample

    f, i = torch.float32, torch.int32
    opt = lambda x, t: None if x is None else dev(np.asarray(x), t)  # noqa: E731
    l = l if isinstance(l, torch.Tensor) else dev(l, f)
    token, prob = sample(l, dev(np.asarray(u), f), opt(temperature, f), opt(top_k, i), opt(top_p, f), opt(min_p, f), **more)
    return token.cpu().numpy(), prob.cpu().numpy()


def decided(l, u, t, k, p, m):
    """Whether neither the draw nor the border of top-p or min-p lies at a token's edge."""
    _, _, edge = ref.sample(l, u, t, k, p, m)
    if edge <= NEAR:
        return False
    order, w = ref.kept(l, t, k, 1.0, 0.0)
    cum = np.cumsum(w[order])
    if p < 1 and np.abs(cum - p * cum[-1]).min() <= NEAR * cum[-1] and len(order) > 1:
        return False
    return not (m > 0 and np.any((np.abs(w[order] - m) <= NEAR * m)))


def rows_of(rng, rows, vocab, kind):
    if kind == "peaked":
        l = rng.randn(rows, vocab) * 2.5
        l[np.arange(rows), rng.randint(0, vocab, rows)] += 8
    elif kind == "flat":
        l = rng.randn(rows, vocab) * 0.1
    else:  # few distinct values: ties everywhere
        l = np.round(rng.randn(rows, vocab) * 4) / 4
    return l.astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 32000, 151936])
@pytest.mark.parametrize("kind", ["peaked", "flat", "ties"])
def test_rules(vocab, kind):
    rng = np.random.RandomState(vocab)
    l, u, t, k, p, m = [], [], [], [], [], []
    for top_k in (0, 1, 7, 50, 5000):
        for top_p in (1.0, 0.9, 0.3):
            for min_p in (0.0, 0.05):
                for _ in range(50):
                    row = rows_of(rng, 1, vocab, kind)[0]
                    draw, temp = np.float32(rng.rand()), np.float32(rng.uniform(0.3, 2.0))
                    if decided(row, draw, temp, top_k, np.float32(top_p), np.float32(min_p)):
                        l.append(row), u.append(draw), t.append(temp), k.append(top_k), p.append(np.float32(top_p)), m.append(np.float32(min_p))
                        break
    assert len(l) >= 15
    token, prob = run(np.stack(l), u, t, k, p, m)
    want = [ref.sample(*a) for a in zip(l, u, t, k, p, m)]
    assert token.tolist() == [w[0] for w in want]
    assert np.all(np.abs(prob - [w[1] for w in want]) <= TOL * np.array([w[1] for w in want]))


@pytest.mark.parametrize("vocab,first,count", [(151936, 100, 1500), (151936, 37000, 1100), (30000, 29000, 1000), (151936, 0, 2500)])
@pytest.mark.parametrize("equal", [False, True])
def test_candidates_close_together(vocab, first, count, equal):
    """The likely tokens are neighbours, so one CTA of a row's has nearly all that the rules look at; all alike, or not."""
    rng = np.random.RandomState(count)
    l, u, k, p = [], [], [], []
    for top_k in (900, 1000, 2000, 0):
        for top_p in (1.0, 0.8):
            for _ in range(50):
                row = (rng.randn(vocab) * 0.5 - 12).astype(np.float32)
                row[first:first + count] = 1.5 if equal else rng.randn(len(row[first:first + count]))
                draw = np.float32(rng.rand())
                if decided(row, draw, 1.0, top_k, np.float32(top_p), 0.0):
                    l.append(row), u.append(draw), k.append(top_k), p.append(np.float32(top_p))
                    break
    assert len(l) >= 4
    token, prob = run(np.stack(l), u, top_k=k, top_p=p)
    want = [ref.sample(a, b, 1.0, c, d) for a, b, c, d in zip(l, u, k, p)]
    assert token.tolist() == [w[0] for w in want]
    assert np.all(np.abs(prob - [w[1] for w in want]) <= TOL * np.array([w[1] for w in want]))


@pytest.mark.parametrize("vocab", [3, 5000, 40000])
def test_each_rule_may_be_absent(vocab):
    rng = np.random.RandomState(1)
    l = rows_of(rng, 4, vocab, "peaked")
    u = np.float32([0.1, 0.35, 0.6, 0.85])
    token, prob = run(l, u)
    want = [ref.sample(a, b) for a, b in zip(l, u)]
    assert token.tolist() == [w[0] for w in want]
    assert np.all(np.abs(prob - [w[1] for w in want]) <= TOL * np.array([w[1] for w in want]))


def test_ties_go_to_the_lower_id():
    l = np.zeros((6, 5000), dtype=np.float32)
    u = np.float32([0.0, 0.5, 0.999999, 0.0, 0.999999, 0.5])
    token, prob = run(l, u, temperature=[1, 1, 1, 1, 1, 0], top_k=[10, 10, 10, 0, 0, 0], top_p=[1, 1, 1, 0.5, 0.5, 1])
    # of equal weights the first ten; half of them; the greedy choice the first
    assert token.tolist() == [0, 5, 9, 0, 2499, 0]
    assert np.allclose(prob, [0.1, 0.1, 0.1, 1 / 2500, 1 / 2500, 1.0], rtol=1e-6)


def test_the_draw_covers_its_ends():
    rng = np.random.RandomState(3)
    l = rows_of(rng, 3, 999, "flat")
    token, _ = run(l, np.float32([0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0]))
    assert token.tolist() == [0, 998, 998]


def test_greedy_rows_beside_sampled_ones():
    rng = np.random.RandomState(4)
    l = rows_of(rng, 8, 33000, "ties")
    t = np.float32([0, 1, 0, -1, 0.5, np.nan, 0, 1])
    u = np.float32(rng.rand(8))
    token, prob = run(l, u, temperature=t)
    for b in range(8):
        if not t[b] > 0:
            assert token[b] == int(l[b].argmax()) and prob[b] == 1.0   # numpy's argmax: the first
        else:
            assert token[b] == ref.sample(l[b], u[b], t[b])[0]


def test_masked_and_unusual_logits():
    low = np.finfo(np.float32).min
    l = np.full((8, 2100), -np.inf, dtype=np.float32)
    l[1, 7] = 0.0                     # one token left
    l[2] = np.nan
    l[3, 5], l[3, 9] = np.nan, -50.0  # a NaN is passed over
    l[4, 3], l[4, 2000] = np.inf, np.inf
    l[4, 100] = 3.0                   # infinities share the draw
    l[5] = low
    l[5, 11] = 1.0                    # masks of the type's lowest value weigh nothing
    l[6] = low                        # everything masked that way: all alike
    l[7, 2099], l[7, 0] = low, -np.inf
    token, prob = run(l, np.float32([0.5, 0.5, 0.5, 0.9, 0.75, 0.99, 0.5, 0.5]), top_p=np.full(8, 0.99, np.float32))
    assert token.tolist() == [-1, 7, -1, 9, 2000, 11, 1040, 2099]
    # 0.99 in 32 bits lies above 2079 / 2100: 2080 tokens are kept of the row whose tokens are all alike
    assert np.allclose(prob, [0, 1, 0, 1, 0.5, 1, 1 / 2080, 1], rtol=1e-6)


def test_rows_do_not_depend_on_their_company():
    """The same row alone, in a batch, with rows further apart than the vocabulary."""
    import torch

    rng = np.random.RandomState(6)
    l = rows_of(rng, 70, 30001, "flat")
    u = np.float32(rng.rand(70))
    t, k, p, m = np.float32(rng.uniform(0.5, 2, 70)), rng.randint(0, 200, 70), np.float32(rng.uniform(0.5, 1.1, 70)), np.float32(rng.uniform(0, 0.1, 70))
    token, prob = run(l, u, t, k, p, m)
    wide = torch.full((70, 30100), 50.0, device="cuda")
    wide[:, 3:30004] = dev(l, torch.float32)
    again = run(wide[:, 3:30004], u, t, k, p, m)
    assert np.array_equal(token, again[0]) and np.array_equal(prob, again[1])
    for b in (0, 13, 69):
        one = run(l[b:b + 1], u[b:b + 1], t[b:b + 1], k[b:b + 1], p[b:b + 1], m[b:b + 1])
        assert one[0][0] == token[b] and one[1][0] == prob[b]


def test_distribution():
    """Evenly spread numbers draw every token as often as its share says (within one draw)."""
    l = np.log(np.float32([[1, 2, 3, 4, 0.5, 5]])).astype(np.float32)
    n = 4000
    u = (np.arange(n, dtype=np.float32) + 0.5) / n
    token, prob = run(np.repeat(l, n, 0), u)
    share = np.exp(l[0].astype(np.float64))
    share /= share.sum()
    assert np.all(np.abs(np.bincount(token, minlength=6) - n * share) <= 1.01)
    assert np.allclose(prob, share[token], rtol=1e-5)


@pytest.mark.parametrize("vocab", [50, 20000])
def test_penalty_window_and_position(vocab):
    import torch

    rng = np.random.RandomState(vocab)
    rows = 5
    l = rows_of(rng, rows, vocab, "flat")
    recent = [list(rng.randint(0, vocab, n)) for n in (0, 3, 63, 64, 64)]
    recent[3][:10] = [7] * 10      # one id ten times
    recent[4][0] = vocab + 5       # an id that the row does not have
    window, state = np.zeros((rows, 64), np.int32), np.zeros((rows, 2), np.int32)
    for b, r in enumerate(recent):
        window[b, :len(r)] = r
        state[b] = len(r), len(r) % 64
    state[4, 1] = 20               # a full ring in the middle
    wd, sd = dev(window, torch.int32), dev(state, torch.int32)
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    logits = dev(l, torch.float32)
    u = np.float32([0.3, 0.5, 0.7, 0.2, 0.9])
    token, prob = run(logits, u, top_k=[0, 5, 0, 0, 40], repetition_penalty=1.3, window=wd, window_state=sd, pos=pos)
    assert np.array_equal(logits.cpu().numpy(), l)   # read only
    for b in range(rows):
        want = ref.sample(ref.penalised(l[b], 1.3, recent[b]), u[b], 1.0, [0, 5, 0, 0, 40][b])
        if want[2] > NEAR:
            assert token[b] == want[0] and abs(prob[b] - want[1]) <= TOL * want[1]
        held, slot = state[b]
        window[b, slot] = token[b]
        state[b] = min(held + 1, 64), (slot + 1) % 64
    assert np.array_equal(wd.cpu().numpy(), window) and np.array_equal(sd.cpu().numpy(), state)
    assert pos.tolist() == [1, 2, 3, 4, 5]


def test_refusals():
    import torch

    from joshua_b200.sampling import sample

    l, u = torch.zeros(2, 100, device="cuda"), torch.zeros(2, device="cuda")
    w = torch.zeros(2, 64, dtype=torch.int32, device="cuda")
    for bad in (lambda: sample(l.half(), u), lambda: sample(l.cpu(), u), lambda: sample(l[0], u), lambda: sample(l, u[:1]),
                lambda: sample(l, u.double()), lambda: sample(l, u, top_k=u), lambda: sample(l, u, temperature=w[:, 0]),
                lambda: sample(l, u, window=w), lambda: sample(l, u, window=w[:, :63], window_state=w[:, :2]),
                lambda: sample(l, u, repetition_penalty=0.0), lambda: sample(l.t(), u), lambda: sample(l[:, :0], u),
                lambda: sample(torch.zeros(1, 393217, device="cuda"), u[:1])):
        with pytest.raises(JoshuaB200Error):
            bad()
    assert sample(l[:0], u[:0])[0].shape == (0,)
    token, _ = sample(torch.zeros(1, 393216, device="cuda"), torch.full((1,), 0.5, device="cuda"))
    assert int(token) == 196608


@pytest.mark.parametrize("vocab", [30, 3000, 151936])
def test_zeros_of_both_signs_are_equal(vocab):
    """-0 and 0 are the same logit: the lower id goes first."""
    l = np.full((5, vocab), -40.0, dtype=np.float32)   # the others weigh nothing
    l[:, 10], l[:, vocab - 10] = -0.0, 0.0
    l[4] = 0.0
    l[4, ::2] = -0.0
    token, _ = run(l, np.float32([0.5, 0.5, 0.5, 0.999, 0.5]), temperature=[0, 1, 1, 1, 1], top_k=[0, 1, 0, 2, 7], top_p=[1, 1, 0.3, 1, 1])
    assert token.tolist() == [10, 10, 10, vocab - 10, 3]
