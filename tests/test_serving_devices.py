"""The serving entries take no context, so the library launches on the current device: the calls make the tensors' device current for the
launch and leave the caller's as it was.  Without a GPU: tensors of the host stand for device -1, the entries only say which device is
current."""
import pytest
import torch

from joshua_b200 import kv_cache, rope, sampling


@pytest.fixture
def current(monkeypatch):
    state = {"device": 3, "seen": []}

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state["device"] = state["device"], self.index

        def __exit__(self, *_):
            state["device"] = self.before

    monkeypatch.setattr(torch.cuda, "device", Device)
    for module in (rope, kv_cache, sampling):
        monkeypatch.setattr(module, "_raw_stream", lambda index: 0)
        monkeypatch.setattr(module, "_device", lambda: state["device"], raising=False)
    monkeypatch.setattr(kv_cache, "_capturing", lambda: False)
    state["entry"] = lambda *_: state["seen"].append(state["device"]) or 0
    return state


def a_rope(entry):
    r = object.__new__(rope.Rope)
    r._index, r.device, r.ref, r._entry, r._bad = -1, torch.device("cpu"), 0, entry, 0
    return r


def a_cache(entry):
    c = object.__new__(kv_cache.PagedCache)
    c._index, c.device, c.n_kv, c.head_dim, c._ref, c._bad, c._scratch, c._needs = -1, torch.device("cpu"), 1, 64, 0, 0, {}, {}
    c._append = c._read = c._attend = entry
    return c


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.mark.parametrize("device", [3, -1])
def test_the_tensors_device_is_current(current, monkeypatch, device):
    current["device"] = device
    r, c = a_rope(current["entry"]), a_cache(current["entry"])
    table = i32(0, 1)[:, None]
    r.apply(torch.zeros(2, 64), i32(0, 1), 1, 64)
    c.append(torch.zeros(2, 192), i32(0, 1), table, n_q=1, rope=r)
    c.read(i32(0, 1), table)
    c.attend(torch.zeros(2, 64), i32(1, 1), table, n_q=1, scale=0.5)
    monkeypatch.setattr(sampling, "device_index", lambda *_: -1)
    monkeypatch.setattr(sampling, "_entry", current["entry"])
    sampling.sample(torch.zeros(2, 10), torch.zeros(2))
    assert current["seen"] == [-1] * 5 and current["device"] == device
