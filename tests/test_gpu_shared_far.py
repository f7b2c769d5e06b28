"""Shared leading pages where scores are far from zero: the attention of a step that takes them once for the batch, on the tensor cores.

What stands out by more than two scores' rounding takes all (tests/test_gpu_attention_chunk.py derives the 2^-17.4 of the largest score;
20 more leave e^-20 to the rest), and every output stays within the values, in sums of 23 bits and products of 22."""
import numpy as np
import pytest

from tests.test_gpu_attention_paged import TOL, fill, queries
from tests.test_gpu_kv_cache import KINDS, i32, make

pytestmark = pytest.mark.gpu
BATCH, N_Q, N_KV, PAGES = 32, 8, 2, 160   # enough of them for a pass of their own with heads of 64 too


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [2.0**8, 2.0**20, 2.0**23, 2.0**26, -2.0**26])
def test_scores_far_from_zero(kind, hd, size):
    import torch

    from joshua_b200 import _lib

    n = PAGES * 64
    cache, own = make(kind, N_KV, hd, 1, PAGES)
    (k, v), = fill(cache, own, [n], seed=2)
    k, v = k.astype(np.float64), v.astype(np.float64)
    table = own.expand(BATCH, -1).contiguous()
    lib = _lib.lib()
    assert lib.jq_attention_paged_scratch_bytes(BATCH, N_Q, N_KV, hd, PAGES) > lib.jq_attention_paged_scratch_bytes(BATCH, N_Q, N_KV, hd, 0)  # it is taken
    q = queries(BATCH, N_Q, hd, 5)
    q[3] *= 2.0**-20    # a row near zero among them
    scale = size / np.sqrt(hd)
    got = cache.attend(q, i32([n] * BATCH), table, n_q=N_Q, scale=scale, shared_pages=PAGES).cpu().numpy().reshape(BATCH, N_KV, -1, hd)
    x = q.cpu().numpy().astype(np.float64).reshape(BATCH, N_KV, -1, hd)
    s = np.einsum("bhgd,htd->bhgt", x, k) * scale
    slack, clear = TOL * np.abs(v).max(), 0
    assert np.isfinite(got).all()
    for h in range(N_KV):
        assert (got[:, h] >= v[h].min(0) - slack).all() and (got[:, h] <= v[h].max(0) + slack).all()
        top = np.abs(s[:, h]).max((-1, -2))
        order = np.argsort(s[:, h], axis=-1)
        best = np.take_along_axis(s[:, h], order[..., -2:], -1)
        alone = best[..., 1] - best[..., 0] > 2.0**-17 * top[:, None] + 20
        err = np.abs(got[:, h] - v[h][order[..., -1]]).max(-1)
        assert (err[alone] <= slack).all()
        clear += int(alone.sum())
    assert clear > BATCH * N_Q // 2 or abs(size) < 2.0**10
    cache.check_flags()
