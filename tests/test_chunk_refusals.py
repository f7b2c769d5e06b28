"""What the entries for chunks, windows and log probabilities refuse, at the C boundary and without a device, and that they launch on their
tensors' device."""
import pytest
import torch

from joshua_b200 import _lib, kv_cache, sampling
from tests import test_serving_devices
from tests.test_serving_devices import a_cache, i32
from tests.test_serving_refusals import A, COMMON, cache, call, refused

current = test_serving_devices.current


B = A + (1 << 20)   # where the results would go: never looked at, as A


def test_chunk_scratch():
    f = _lib.lib().jq_attention_chunk_scratch_bytes
    assert f(0, 8, 8, 2, 128) == f(4097, 8, 8, 2, 128) == f(1, 0, 8, 2, 128) == f(1, 65537, 8, 2, 128) == f(1, 8, 8, 0, 128) == f(1, 8, 9, 2, 128) == 0
    # tiles' parts only where some sequence may have more rows than are taken one by one; heads of 256 have no tiles
    assert f(4, 4, 8, 2, 128) > f(1, 1, 8, 2, 128) > 0 and f(1, 500, 8, 2, 256) == f(1, 1, 8, 2, 256)


def test_chunks():
    ok = dict(cache=cache(), q=A, q_stride=512, first=A, len=A, table=A, n_seq=2, per=3, rows=5, n_q=4, scale=0.0, window=0, sinks=0, out=B,
              out_stride=512, scratch=A, bad=None, stream=None)
    for nothing in (dict(n_seq=0), dict(rows=0)):
        assert call("jq_attention_chunk_dev", ok, nothing) == _lib.OK
    for change, word in [c for c in COMMON if "n_seq" not in c[0]] + [
            (dict(n_q=6, cache=cache(n_kv=4)), "query heads"), (dict(q=None), "NULL"), (dict(len=None), "NULL"), (dict(out=None), "NULL"),
            (dict(scratch=None), "NULL"), (dict(first=None), "equal parts"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
            (dict(q_stride=511), "rows"), (dict(out_stride=514), "rows"), (dict(q=A + 4), "boundaries"), (dict(scratch=A + 8), "boundaries"),
            (dict(n_seq=4096, per=1 << 20), "2^28"), (dict(out=A), "overlap"), (dict(out=A + 4 * 512 * 4), "overlap"), (dict(q=A + 4 * 512 * 5 - 16, out=A), "overlap"),
            (dict(q_stride=1536, out_stride=1536, out=A + 496 * 4), "overlap"), (dict(q_stride=1536, out_stride=1536, out=A + 1040 * 4), "overlap"),
            (dict(q_stride=1536, out_stride=1536, q=A + 1024 * 4, out=A + 528 * 4), "overlap"), (dict(q_stride=1536, out=A + 1024 * 4), "overlap")]:
        refused(call("jq_attention_chunk_dev", ok, change), "jq_attention_chunk_dev", word)
    for change, word in ((dict(n_seq=4097), "JQ_ATTENTION_MAX_BATCH"), (dict(rows=65537), "JQ_ATTENTION_MAX_ROWS"),
                         (dict(rows=65536, n_q=4096, q_stride=1 << 20, out_stride=1 << 20), "too many"), (dict(rows=65536, per=1 << 14), "too many")):
        refused(call("jq_attention_chunk_dev", ok, change), word, code=_lib.E_TOO_LARGE)


def test_log_probs():
    ok = dict(logits=A, stride=100, rows=1, vocab=100, token=A, top=3, given=A, entropy=None, top_token=A, top_given=A, stream=None)
    assert call("jq_log_probs_dev", ok, dict(rows=0)) == _lib.OK
    for change, word in ((dict(logits=None), "NULL"), (dict(token=None), "NULL"), (dict(given=None), "NULL"), (dict(vocab=0), "rows"),
                         (dict(stride=99), "rows"), (dict(vocab=1 << 31, stride=1 << 32), "rows"), (dict(top_token=None), "NULL"), (dict(top_given=None), "NULL")):
        refused(call("jq_log_probs_dev", ok, change), "jq_log_probs_dev", word)
    refused(call("jq_log_probs_dev", ok, dict(top=33)), "JQ_LOG_PROBS_MOST", code=_lib.E_TOO_LARGE)
    refused(call("jq_log_probs_dev", ok, dict(rows=(1 << 24) + 1)), "2^24", code=_lib.E_TOO_LARGE)


@pytest.mark.parametrize("device", [3, -1])
def test_the_tensors_device_is_current(current, monkeypatch, device):
    current["device"] = device
    c = a_cache(current["entry"])
    c._chunk = current["entry"]
    table = i32(0, 1)[:, None]
    c.attend_chunk(torch.zeros(4, 64), i32(2, 2), table, n_q=1, scale=0.5)
    c.attend(torch.zeros(2, 64), i32(1, 1), table, n_q=1, scale=0.5, window=3, sinks=1)
    monkeypatch.setattr(sampling, "device_index", lambda *_: -1)
    monkeypatch.setattr(sampling, "_scores", current["entry"])
    sampling.log_probs(torch.zeros(2, 10), i32(1, 2), top=2)
    assert current["seen"] == [-1] * 3 and current["device"] == device


def test_the_tiles_may_have_no_status_flag():
    from tests.test_serving_refusals import test_an_entry_without_a_context_may_have_no_status_flag as guarded

    guarded("attention_chunk_tiles.cu")


def test_rooms_for_parts():
    """Whether a prompt read in parts fits the pool is worked out before any part is taken: against taking and giving back page by page."""
    from joshua_b200.paged import _Paged

    def decoder(pages, window, sinks, rows, held=0):
        dec = object.__new__(_Paged)
        dec.attention_window, dec.attention_sinks, dec.prompt_rows, dec.max_ctx, dec.pages_per_seq = window, sinks, rows, 5000, 80
        dec.n_pages, dec.free, dec.owned, dec.held, dec.kept_from, dec.holders = pages, list(range(pages)), [[]], [0], [0], [0] * pages
        dec._enter = lambda places, pages: None
        return dec

    def takes(dec, n):
        while n:
            part = min(n, dec.prompt_rows)
            dec._trim([0])
            try:
                dec._reserve({0: dec.held[0] + part})
            except _lib.JoshuaB200Error:
                return False
            dec.held[0] += part
            n -= part
        return True

    for pages in (3, 5, 9):
        for window, sinks in ((64, 0), (100, 4), (30, 130), (1000, 0)):
            for rows in (10, 64, 100, 300):
                for n in (1, 63, 64, 200, 500, 1500):
                    for before in (0, 40, 190):
                        a, b = (decoder(pages, window, sinks, rows) for _ in range(2))
                        if not (takes(a, before) and takes(b, before)):
                            continue
                        state = list(a.free), [list(o) for o in a.owned], list(a.held)
                        try:
                            a._room_for_parts(0, n)
                            fits = True
                        except _lib.JoshuaB200Error:
                            fits = False
                        assert state == (list(a.free), [list(o) for o in a.owned], list(a.held))
                        assert fits == takes(b, n), (pages, window, sinks, rows, n, before)
    with pytest.raises(_lib.JoshuaB200Error):
        decoder(100, 64, 0, 64)._room_for_parts(0, 5001)
