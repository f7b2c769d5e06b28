"""Rotary positions on the device against the formula in 64 bits.

Tolerances: a table entry is a 64-bit value rounded once (half an ulp, 2^-24 of it; 2^-46 of an angle of up to 2^17 for the
64-bit angle itself is far below).  A rotation is two products and a sum, each rounded once: 3 * 2^-24 (|a| + |b|) m covers it.
"""
import ctypes

import numpy as np
import pytest

from joshua_b200 import _lib
from joshua_b200._lib import JoshuaB200Error
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu
EPS = 2.0**-24


def frequencies(theta, rot):
    return theta ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)


def expect_table(got, f, m=1.0):
    angle = np.arange(got.shape[0], dtype=np.float64)[:, None] * f
    want = np.stack((np.cos(angle), np.sin(angle)), -1) * m
    assert np.abs(got.cpu().numpy() - want).max() <= m * (EPS + got.shape[0] * 2.0**-50)


@pytest.mark.parametrize("theta,rot,n_pos", [(500000.0, 128, 5000), (10000.0, 64, 1), (1e6, 2, 77), (10000.0, 256, 130001)])
def test_table(theta, rot, n_pos):
    from joshua_b200.rope import rope_table

    expect_table(rope_table(theta, rot, n_pos, "cuda"), frequencies(theta, rot))


def test_table_linear_and_factors():
    from joshua_b200.rope import rope_table

    f = frequencies(500000.0, 64)
    expect_table(rope_table(500000.0, 64, 3000, "cuda", scaling="linear", factor=4.0), f / 4)
    factors = 1.0 + np.arange(32) / 4
    expect_table(rope_table(500000.0, 64, 3000, "cuda", freq_factors=factors), f / factors)


@pytest.mark.parametrize("factor,orig,m", [(40.0, 4096, 1.0), (4.0, 32768, 1.1386294), (1.5, 100, 1.0)])
def test_table_yarn(factor, orig, m):
    """Pairs that turn more than beta_fast times in the old context keep their frequency, those below beta_slow are slowed."""
    from joshua_b200.rope import rope_table

    theta, rot = 10000.0, 64
    f = frequencies(theta, rot)

    def pair(turns):
        return rot * np.log(orig / (turns * 2 * np.pi)) / (2 * np.log(theta))

    low, high = max(np.floor(pair(32.0)), 0.0), min(np.ceil(pair(1.0)), rot - 1.0)
    keep = 1 - np.clip((np.arange(rot // 2) - low) / (high - low + (0.001 if low == high else 0.0)), 0, 1)
    expect_table(rope_table(theta, rot, 3000, "cuda", scaling="yarn", factor=factor, orig_ctx=orig, mscale=m),
                 f * keep + f / factor * (1 - keep), float(np.float32(m)))


def test_yarn_agrees_with_the_latent_attention_loader():
    from joshua_b200.deepseek import DeepseekConfig, yarn_table
    from joshua_b200.rope import rope_table

    cfg = DeepseekConfig(yarn_factor=40.0)
    inv, _, _ = yarn_table(cfg)
    t = rope_table(cfg.rope_theta, cfg.qk_rope, 2, "cuda", scaling="yarn", factor=40.0, orig_ctx=cfg.yarn_orig_ctx).cpu().numpy()
    got = np.arctan2(t[1, :, 1].astype(np.float64), t[1, :, 0])  # position 1: the frequencies themselves
    assert np.abs(got - inv).max() <= 1e-6  # the loader's are f32


@pytest.mark.parametrize("hd,rot,heads", [(128, 128, 5), (64, 32, 1), (256, 64, 3), (96, 96, 2), (80, 20, 7), (4, 2, 1), (128, 6, 40)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows", [1, 37])
def test_rotation(hd, rot, heads, interleaved, rows):
    import torch

    from joshua_b200.rope import Rope, rope_table

    rng = np.random.RandomState(hd + rot + rows)
    x = rng.randn(rows, heads * hd).astype(np.float32) * 3
    pos = rng.randint(0, 5000, rows).astype(np.int32)
    table = rope_table(10000.0, rot, 5000, "cuda", mscale=1.25)
    r = Rope(table, interleaved=interleaved)
    xd, pd = torch.from_numpy(x).cuda(), torch.from_numpy(pos).cuda()
    for inverse in (False, True):
        got = r.apply(xd, pd, heads, hd, inverse=inverse).cpu().numpy().reshape(rows, heads, hd)
        want = ref.rope(x.reshape(rows, heads, hd), table.cpu().numpy(), pos, rot, interleaved, inverse)
        other = np.abs(ref.rope(np.abs(x).reshape(rows, heads, hd), np.abs(table.cpu().numpy()), pos, rot, interleaved, False))
        size = np.abs(x).reshape(rows, heads, hd).max(-1, keepdims=True) * 2 * 1.25 + other
        assert np.all(np.abs(got - want) <= 3 * EPS * size)
        assert np.array_equal(got[..., rot:], x.reshape(rows, heads, hd)[..., rot:])


def test_rows_in_place_and_strided():
    import torch

    from joshua_b200.rope import Rope, rope_table

    r = Rope(rope_table(10000.0, 128, 300, "cuda"))
    torch.manual_seed(1)
    x = torch.randn(9, 4 * 128, device="cuda")
    pos = torch.arange(291, 300, dtype=torch.int32, device="cuda")
    want = r.apply(x, pos, 4, 128)
    wide = torch.full((9, 700), 7.0, device="cuda")  # the same rows among other columns, turned where they are
    wide[:, 100:100 + 512] = x
    got = r.apply(wide[:, 100:100 + 512], pos, 4, 128, out=wide[:, 100:100 + 512])
    assert torch.equal(got, want) and bool((wide[:, :100] == 7).all()) and bool((wide[:, 612:] == 7).all())
    back = r.apply(want, pos, 4, 128, inverse=True)
    assert float((back - x).abs().max()) <= 12 * EPS * float(x.abs().max())


def test_gradient():
    """The map is linear, so its gradient is the transposed rotation: against differences of f(x) = <g, turned x>, and against
    the formula."""
    import torch

    from joshua_b200.rope import Rope, rope_table

    for interleaved in (False, True):
        r = Rope(rope_table(10000.0, 16, 50, "cuda"), interleaved=interleaved)
        torch.manual_seed(2)
        x, g = torch.randn(3, 2 * 32, device="cuda"), torch.randn(3, 2 * 32, device="cuda")
        pos = torch.tensor([0, 7, 49], dtype=torch.int32, device="cuda")
        grad = r.apply(g, pos, 2, 32, inverse=True).double()

        def f(t):
            return (g.double() * r.apply(t, pos, 2, 32).double()).sum(-1)

        for d in range(64):
            step = torch.zeros_like(x)
            step[:, d] = 0.5  # the map is linear: a long step differs by rounding only
            diff = f(x + step) - f(x - step)
            # 64 terms of up to |g| |x + step| with 4 roundings each on both sides
            assert float((diff - grad[:, d]).abs().max()) <= 2 * 64 * 4 * EPS * float(g.abs().max()) * (float(x.abs().max()) + 0.5)


def test_positions_outside_the_table():
    import torch

    from joshua_b200.rope import Rope, rope_table

    r = Rope(rope_table(10000.0, 64, 10, "cuda"))
    x = torch.randn(4, 64, device="cuda")
    out = torch.full_like(x, 5.0)
    r.apply(x, torch.tensor([3, -1, 10, 2**31 - 1], dtype=torch.int32, device="cuda"), 1, 64, out=out)
    assert int(r.bad_pos) == 1 and bool((out[1:] == 5).all()) and not bool((out[0] == 5).any())


def test_refusals():
    import torch

    from joshua_b200.rope import Rope, rope_table

    table = rope_table(10000.0, 64, 10, "cuda")
    r, x, p = Rope(table), torch.zeros(2, 128, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: r.apply(x.half(), p, 1, 128), lambda: r.apply(x.cpu(), p, 1, 128), lambda: r.apply(x, p.long(), 1, 128),
                lambda: r.apply(x, p[:1], 1, 128), lambda: r.apply(x, p, 2, 128), lambda: r.apply(x.t().contiguous().t(), p, 1, 128),
                lambda: r.apply(x, p, 4, 32), lambda: r.apply(torch.zeros(2, 130, device="cuda")[:, 1:129], p, 1, 128),
                lambda: r.apply(x, p, 1, 128, out=x[:1]), lambda: Rope(table[:, ::2]), lambda: Rope(table.double()),
                lambda: rope_table(10000.0, 64, 10, "cuda", scaling="other"), lambda: rope_table(0.0, 64, 10, "cuda"),
                lambda: rope_table(10000.0, 63, 10, "cuda"), lambda: rope_table(10000.0, 258, 10, "cuda"),
                lambda: rope_table(10000.0, 64, 10, "cuda", scaling="linear", factor=0.0),
                lambda: rope_table(10000.0, 64, 10, "cuda", scaling="yarn", factor=4.0),
                lambda: rope_table(10000.0, 64, 10, "cuda", freq_factors=[1.0]),
                lambda: rope_table(10000.0, 64, 10, "cuda", freq_factors=[-1.0] * 32)):
        with pytest.raises(JoshuaB200Error):
            bad()
    assert r.apply(x[:0], p[:0], 1, 128).shape == (0, 128)


def test_on_another_stream():
    import torch

    from joshua_b200.rope import Rope, rope_table

    r = Rope(rope_table(10000.0, 128, 300, "cuda"))
    x, pos = torch.randn(64, 1280, device="cuda"), torch.arange(64, dtype=torch.int32, device="cuda")
    want = r.apply(x, pos, 10, 128)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = x + 0  # made on the side stream: an entry that ran on another would read it too early
        got = r.apply(y, pos, 10, 128)
    side.synchronize()
    assert torch.equal(got, want)
