"""Rows of chunks named by a `first` that goes up and down: sequences may then have more rows together than the call, and the sums that the
kernels cut the work by hold what the host allows a call.  Those calls are refused on the device, whole.  The cases here are far from what
32 bits hold all the same: the page table is wide, the sequences are short."""
import pytest

from tests.test_gpu_attention_chunk import compare, starts
from tests.test_gpu_attention_paged import fill, queries
from tests.test_gpu_kv_cache import i32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128, 256])   # tiles and single rows; heads of 256: single rows alone
@pytest.mark.parametrize("rows", [2, 512])
def test_rows_named_twice(hd, rows):
    import torch

    n_q, n_kv, length = 4, 2, 600
    wide = 2**31 // (4 * rows) - 2           # rows * (4 wide + 8) = 2^31: twice the rows do not fit
    wide = min(wide, 2**20)                  # two rows: they do
    cache, narrow = make("q8_0", n_kv, hd, 4, 10)
    kv = fill(cache, narrow, [length] * 4, seed=hd)
    table = torch.full((4, wide), -1, dtype=torch.int32, device="cuda")
    table[:, :10] = narrow
    lens, q = i32([length] * 4), queries(rows, n_q, hd, 1)
    for up_and_down in ([0, rows, 0, rows, 0], [0, rows, 1, rows, 0], [rows - 1, rows, 0, rows, 0]):
        together = sum(max(b - a, 0) for a, b in zip(up_and_down, up_and_down[1:]))
        out = torch.full((rows, n_q * hd), 7.0, device="cuda")
        cache.attend_chunk(q, lens, table, n_q=n_q, first=i32(up_and_down), out=out)
        assert int(cache.bad_pos) == 1
        cache.bad_pos.zero_()
        if together * (4 * wide + 8) >= 2**32:
            assert bool((out == 7.0).all()), up_and_down
        else:
            assert bool(out.isfinite().all()) and bool((out != 7.0).any())
    assert 2 * rows * (4 * wide + 8) >= 2**32 or rows == 2
    counts = [rows // 2, 0, rows - rows // 2, 0]   # and the rows of an ascending one are as they were
    got = cache.attend_chunk(q, lens, table, n_q=n_q, first=starts(counts))
    compare(got, q, kv, counts, [length] * 4, n_q, hd)
    cache.check_flags()
