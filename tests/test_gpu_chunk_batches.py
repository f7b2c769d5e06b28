"""Chunks of thousands of short sequences: a CTA of the tiles has more pieces of work than it lists at a time (96), batch after batch."""
import pytest

from tests.test_gpu_attention_paged import TOL, queries
from tests.test_gpu_kv_cache import KINDS, i32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [0, 30])
def test_many_pieces_a_cta(kind, window):
    import torch

    seqs, n_kv, hd, new, sinks = 4096, 8, 64, 16, 3 if window else 0
    g = torch.Generator(device="cuda").manual_seed(window)
    cache, table = make(kind, n_kv, hd, seqs, 2, seed=window)
    lens = torch.randint(new, 129, (seqs,), device="cuda", generator=g).int()   # one page or two
    for at in range(0, 128, 32):
        pos = torch.arange(at, at + 32, device="cuda").int().repeat(seqs)
        seq = torch.arange(seqs, device="cuda").int().repeat_interleave(32)
        cache.append(torch.randn(32 * seqs, 3 * n_kv * hd, device="cuda", generator=g), pos, table, n_q=n_kv, seq=seq)
    q = queries(new * seqs, n_kv, hd, 1)
    assert seqs * n_kv // torch.cuda.get_device_properties(0).multi_processor_count > 2 * 96
    got = cache.attend_chunk(q, lens, table, n_q=n_kv, window=window, sinks=sinks)
    first = torch.arange(0, new * seqs + 1, new, device="cuda").int()
    assert bool((cache.attend_chunk(q, lens, table, n_q=n_kv, first=first, window=window, sinks=sinks) == got).all())
    t, some = torch.arange(128, device="cuda"), 256
    for s0 in range(0, seqs, some):   # in 64 bits
        rows = torch.arange(s0, s0 + some, device="cuda").int()
        k, v = cache.read(t.int().repeat(some), table, seq=rows.repeat_interleave(128))
        k, v = (x.view(n_kv, some, 128, hd).transpose(0, 1).double() for x in (k, v))
        x = q[s0 * new:(s0 + some) * new].view(some, new, n_kv, hd).transpose(1, 2).double()
        p = (lens[s0:s0 + some, None] - new + torch.arange(new, device="cuda"))[:, :, None]
        seen = (t <= p) & ((p - t < window) | (t < sinks) if window else True)
        s = (x @ k.transpose(-1, -2) / hd**0.5).masked_fill(~seen[:, None], float("-inf"))
        want = (s.softmax(-1) @ v).transpose(1, 2).reshape(some * new, n_kv * hd)
        assert float((got[s0 * new:(s0 + some) * new] - want).abs().max()) <= TOL * float(v.abs().max())
    cache.check_flags()
