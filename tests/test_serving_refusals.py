"""What the serving entries refuse, at the C boundary and without a device: every fault is named before anything is launched."""
import ctypes

import pytest

from joshua_b200 import _lib
from tests.conftest import ROOT

U32, F32, VP = ctypes.c_uint32, ctypes.c_float, ctypes.c_void_p


class Cache(ctypes.Structure):
    _fields_ = [("type", U32), ("n_kv", U32), ("head_dim", U32), ("n_pages", U32), ("pages", VP)]


class Rope(ctypes.Structure):
    _fields_ = [("table", VP), ("n_pos", U32), ("rot_dim", U32), ("interleaved", ctypes.c_int32)]


class Config(ctypes.Structure):
    _fields_ = [("theta", ctypes.c_double), ("scaling", ctypes.c_int32), ("factor", F32), ("orig_ctx", U32), ("beta_fast", F32),
                ("beta_slow", F32), ("mscale", F32)]


A = 1 << 20   # an aligned address that no refused call may touch


def cache(type_id=8, n_kv=2, hd=128, n_pages=4, pages=A):
    return Cache(type_id, n_kv, hd, n_pages, pages)


def rope(table=A, n_pos=100, rot=128, interleaved=0):
    return Rope(table, n_pos, rot, interleaved)


def refused(rc, *words, code=_lib.E_INVALID):
    assert rc == code
    message = _lib.lib().jq_last_error().decode()
    assert all(w in message for w in words), message


def call(name, args, change):
    """The entry with one argument of a call in order replaced."""
    args = dict(args, **change)
    keep = [v for v in args.values() if isinstance(v, ctypes.Structure)]  # alive during the call
    rc = getattr(_lib.lib(), name)(*[ctypes.addressof(v) if isinstance(v, ctypes.Structure) else v for v in args.values()])
    del keep
    return rc


def test_page_bytes():
    f = _lib.lib().jq_kv_page_bytes
    for type_id, bits, scales in ((1, 16, 0), (8, 8, 1), (2, 4, 1)):
        for hd in (64, 128, 256):
            assert f(type_id, 3, hd) == 3 * 2 * (64 * hd * bits // 8 + scales * 64 * (hd // 32) * 2)
    for bad in ((0, 3, 64), (12, 3, 64), (8, 0, 64), (8, 1025, 64), (8, 3, 96), (8, 3, 0)):
        assert f(*bad) == 0


def test_attention_scratch():
    f = _lib.lib().jq_attention_paged_scratch_bytes
    assert f(0, 8, 2, 128, 0) == f(4097, 8, 2, 128, 0) == f(1, 8, 0, 128, 0) == f(1, 9, 2, 128, 0) == 0
    # results of the leading pages, where they are taken by themselves: not for a few pages of a few sequences
    assert f(32, 32, 8, 128, 64) > f(32, 32, 8, 128, 0) > 0
    assert f(4, 8, 2, 128, 3) == f(4, 8, 2, 128, 0) and f(1, 8, 2, 128, 300) == f(1, 8, 2, 128, 0)


def test_rope_table():
    def args(rot=64, n=10, table=A, factors=None, **cfg):
        c = Config(**{**dict(theta=1e4, scaling=0, factor=1.0, orig_ctx=0, beta_fast=32.0, beta_slow=1.0, mscale=1.0), **cfg})
        return _lib.lib().jq_rope_table_dev(ctypes.byref(c), factors, rot, n, table, None)

    refused(_lib.lib().jq_rope_table_dev(None, None, 64, 10, A, None), "jq_rope_table_dev", "NULL")
    refused(args(table=None), "NULL")
    for rot in (0, 63, 258):
        refused(args(rot=rot), "rot_dim")
    refused(args(table=A + 4), "aligned")
    for theta in (0.0, -1.0, float("nan"), float("inf")):
        refused(args(theta=theta), "theta")
    refused(args(scaling=3), "scaling"), refused(args(scaling=-1), "scaling")
    for factor in (0.0, -2.0, float("nan"), float("inf")):
        refused(args(scaling=1, factor=factor), "factor")
    for more in (dict(orig_ctx=0), dict(orig_ctx=9, beta_slow=0.0), dict(orig_ctx=9, beta_fast=1.0), dict(orig_ctx=9, theta=1.0)):
        refused(args(scaling=2, factor=2.0, **more), "YaRN")
    refused(args(mscale=-1.0), "mscale")
    refused(args(factors=(F32 * 32)(*[0.0] * 32)), "factors")
    assert args(n=0) == _lib.OK


def test_rope():
    ok = dict(rope=rope(), x=A, x_stride=256, pos=A, rows=0, heads=2, head_dim=128, inverse=0, out=A, out_stride=256, bad=None, stream=None)
    assert call("jq_rope_dev", ok, {}) == _lib.OK
    for change, word in ((dict(rope=None), "NULL"), (dict(head_dim=126), "multiple of 4"), (dict(head_dim=2048), "1024"),
                         (dict(rope=rope(table=None)), "table"), (dict(rope=rope(rot=130)), "rot_dim"), (dict(rope=rope(rot=7)), "even"),
                         (dict(rope=rope(interleaved=2)), "interleaved"), (dict(rows=1, x=None), "NULL"), (dict(rows=1, pos=None), "NULL"),
                         (dict(rows=1, out=None), "NULL"), (dict(rows=1, x_stride=255), "rows"), (dict(rows=1, out_stride=258), "rows"),
                         (dict(rows=1, x=A + 4), "boundaries")):
        refused(call("jq_rope_dev", ok, change), "jq_rope_dev", word)


COMMON = [(dict(cache=None), "NULL"), (dict(cache=cache(pages=None)), "NULL"), (dict(table=None), "NULL"), (dict(cache=cache(type_id=12)), "type"),
          (dict(cache=cache(hd=96)), "head_dim"), (dict(cache=cache(n_kv=0)), "kv heads"), (dict(cache=cache(pages=A + 8)), "aligned"),
          (dict(cache=cache(n_pages=0)), "pages"), (dict(n_seq=0), "page table"), (dict(per=0), "page table"), (dict(per=1 << 26), "positions")]


def test_append():
    ok = dict(cache=cache(), rope=rope(), qkv=A, stride=1024, pos=A, seq=None, table=A, n_seq=2, per=3, rows=0, n_q=4, qn=None, kn=None,
              eps=0.0, q_out=A, bad=None, stream=None)
    assert call("jq_kv_append_dev", ok, {}) == _lib.OK and call("jq_kv_append_dev", ok, dict(rope=None)) == _lib.OK
    for change, word in COMMON + [(dict(n_q=0), "query heads"), (dict(n_q=5), "query heads"), (dict(rope=rope(rot=256)), "rot_dim"),
                                  (dict(rows=1, qkv=None), "NULL"), (dict(rows=1, pos=None), "NULL"), (dict(rows=1, q_out=None), "NULL"),
                                  (dict(rows=1, qn=A), "together"), (dict(rows=1, stride=1020), "rows"), (dict(rows=1, stride=1026), "rows"),
                                  (dict(rows=1, qkv=A + 4), "boundaries"), (dict(rows=1, q_out=A + 8), "boundaries"), (dict(rows=1 << 31), "too many")]:
        refused(call("jq_kv_append_dev", ok, change), "jq_kv_append_dev", word)


def test_read():
    ok = dict(cache=cache(), pos=A, seq=None, table=A, n_seq=2, per=3, rows=0, k=A, v=A, row=128, head=1280, bad=None, stream=None)
    assert call("jq_kv_read_dev", ok, {}) == _lib.OK
    for change, word in COMMON + [(dict(rows=1, pos=None), "NULL"), (dict(rows=1, k=None), "NULL"), (dict(rows=1, v=None), "NULL"),
                                  (dict(rows=1, row=127), "strides"), (dict(rows=1, head=64), "strides"), (dict(rows=1, head=1281), "strides"),
                                  (dict(rows=1, v=A + 4), "boundaries")]:
        refused(call("jq_kv_read_dev", ok, change), "jq_kv_read_dev", word)


def test_attention():
    ok = dict(cache=cache(), q=A, q_stride=512, len=A, table=A, n_seq=2, per=3, n_q=4, scale=0.0, shared=0, out=A, out_stride=512, scratch=A,
              bad=None, stream=None)
    assert call("jq_attention_paged_dev", ok, dict(n_seq=0)) == _lib.OK
    for change, word in [c for c in COMMON if "n_seq" not in c[0]] + [
            (dict(n_q=6, cache=cache(n_kv=4)), "query heads"), (dict(q=None), "NULL"), (dict(len=None), "NULL"), (dict(out=None), "NULL"),
            (dict(scratch=None), "NULL"), (dict(shared=4), "shared"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
            (dict(q_stride=511), "rows"), (dict(out_stride=514), "rows"), (dict(q=A + 4), "boundaries"), (dict(scratch=A + 8), "boundaries"),
            (dict(n_seq=4096, per=1 << 20), "2^28")]:
        refused(call("jq_attention_paged_dev", ok, change), "jq_attention_paged_dev", word)
    refused(call("jq_attention_paged_dev", ok, dict(n_seq=4097)), "JQ_ATTENTION_MAX_BATCH", code=_lib.E_TOO_LARGE)


def test_sampling():
    ok = dict(logits=A, stride=100, rows=0, vocab=100, u=A, t=None, k=None, p=None, m=None, penalty=1.0, window=None, state=None, token=A,
              prob=None, pos=None, stream=None)
    assert call("jq_sample_dev", ok, {}) == _lib.OK
    for change, word in ((dict(logits=None), "bad argument"), (dict(u=None), "bad argument"), (dict(token=None), "bad argument"),
                         (dict(vocab=0), "bad argument"), (dict(stride=99), "bad argument"), (dict(rows=65536), "bad argument"),
                         (dict(window=A), "together"), (dict(state=A), "together"), (dict(penalty=0.0), "penalty"),
                         (dict(penalty=float("nan")), "penalty")):
        refused(call("jq_sample_dev", ok, dict(dict(rows=1), **change)), "jq_sample_dev", word)
    refused(call("jq_sample_dev", ok, dict(rows=1, vocab=393217, stride=393217)), "JQ_SAMPLE_MAX_VOCAB", code=_lib.E_TOO_LARGE)


@pytest.mark.parametrize("name", ["attention_lead.cu"])
def test_an_entry_without_a_context_may_have_no_status_flag(name):
    """These kernels take no context: their flag is NULL until one exists on the device, so every store through it is guarded."""
    text = (ROOT / "joshua_b200" / "csrc" / name).read_text()
    stores = [line for line in text.splitlines() if "volatile int*>(error_flag) = 1" in line]
    assert stores and all("&& error_flag)" in line for line in stores)


def test_prompts_on_several_ranks():
    """Refused before a page is taken: the exchange's windows are sized for steps."""
    from joshua_b200.moe_decoder import MoeDecoderConfig
    from joshua_b200.paged import PagedMoeDecoder

    dec = object.__new__(PagedMoeDecoder)
    dec.cfg, dec.world, dec.batch, dec.layers, dec.held = MoeDecoderConfig(), 2, 2, [], [0, 0]
    dec.free, dec.owned = [1, 0], [[], []]
    for call in (lambda: dec.prefill([1, 2, 3]), lambda: dec.share_prompt([1, 2, 3])):
        with pytest.raises(_lib.JoshuaB200Error, match="one GPU"):
            call()
    assert dec.free == [1, 0] and dec.owned == [[], []]
