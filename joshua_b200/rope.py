"""Rotary positions from a table: half or interleaved pairs, part of the head, scaled for long contexts.

`rope_table` builds the (cosine, sine) table a decoder keeps; `Rope` holds one and turns rows of heads with it, or hands it to
`PagedCache.append`, which turns queries and keys on their way into the cache.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import JoshuaB200Error, check

SCALINGS = {None: 0, "none": 0, "linear": 1, "yarn": 2}

_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None
# the entries launch on the current device, which need not be the tensors'
_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else None
_new, _f32 = torch.empty, torch.float32


def _refuse(t, name, dtype, index, shape):
    got = f"{t.dtype} {list(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
    raise JoshuaB200Error(_lib.E_INVALID, f"{name} must be {shape} of {dtype} on cuda:{index}, not {got}")


def device_index(t, name, dtype) -> int:
    """The GPU that a tensor of `dtype` is on; refuses all else."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != dtype:
        raise JoshuaB200Error(_lib.E_INVALID, f"{name} must be a {dtype} tensor on the GPU")
    return t.get_device()


def rows_arg(t, name, width, index):
    """(pointer, floats between rows, rows) of a two-dimensional f32 tensor with contiguous rows."""
    if isinstance(t, torch.Tensor) and t.dtype is _f32 and t.get_device() == index and t.dim() == 2:
        rows, columns = t.shape
        if columns == width:
            if t.is_contiguous():
                return t.data_ptr(), width, rows
            if width == 1 or t.stride(1) == 1:
                return t.data_ptr(), t.stride(0) if rows > 1 else width, rows
    _refuse(t, name, _f32, index, f"[rows, {width}] with contiguous rows")


def vector_arg(t, name, n, dtype, index):
    """Pointer of a contiguous vector."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != index or t.dim() != 1 or t.numel() != n \
            or not t.is_contiguous():
        _refuse(t, name, dtype, index, f"a contiguous vector of {n}")
    return t.data_ptr()


def block_arg(t, name, shape, dtype, index):
    """Pointer of a contiguous tensor of `shape`."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != index or t.shape != shape or not t.is_contiguous():
        _refuse(t, name, dtype, index, f"contiguous, {list(shape)},")
    return t.data_ptr()


class _Config(ctypes.Structure):
    _fields_ = [("theta", ctypes.c_double), ("scaling", ctypes.c_int32), ("factor", ctypes.c_float), ("orig_ctx", ctypes.c_uint32),
                ("beta_fast", ctypes.c_float), ("beta_slow", ctypes.c_float), ("mscale", ctypes.c_float)]


class _Rope(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("n_pos", ctypes.c_uint32), ("rot_dim", ctypes.c_uint32), ("interleaved", ctypes.c_int32)]


def rope_table(theta: float, rot_dim: int, n_pos: int, device, scaling: str | None = None, factor: float = 1.0, orig_ctx: int = 0,
               beta_fast: float = 32.0, beta_slow: float = 1.0, mscale: float = 1.0, freq_factors=None) -> torch.Tensor:
    """[n_pos, rot_dim / 2, 2] (cosine, sine) of every position and pair.  `scaling`: None, "linear" or "yarn";
    `freq_factors`: divisors of the frequencies (a GGUF file's `rope_freqs.weight`)."""
    if scaling not in SCALINGS:
        raise JoshuaB200Error(_lib.E_INVALID, f"unknown rope scaling {scaling!r}")
    cfg = _Config(theta, SCALINGS[scaling], factor, orig_ctx, beta_fast, beta_slow, mscale)
    factors = None
    if freq_factors is not None:
        if len(freq_factors) != rot_dim // 2:
            raise JoshuaB200Error(_lib.E_INVALID, f"{len(freq_factors)} frequency factors for {rot_dim // 2} pairs")
        factors = (ctypes.c_float * len(freq_factors))(*[float(f) for f in freq_factors])
    device = torch.device(device)
    with torch.cuda.device(device):
        table = _new(max(n_pos, 0), max(rot_dim, 0) // 2, 2, dtype=_f32, device=device)
        check(_lib.lib().jq_rope_table_dev(ctypes.byref(cfg), factors, rot_dim, n_pos, table.data_ptr() or None,
                                           _raw_stream(torch.cuda.current_device())))
    return table


class Rope:
    """A table of `rope_table` and how a head's dimensions pair up."""

    def __init__(self, table: torch.Tensor, interleaved: bool = False):
        self._index = device_index(table, "table", _f32)
        if table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous():
            raise JoshuaB200Error(_lib.E_INVALID, "a rope table is contiguous, [positions, pairs, 2]")
        self.table, self.interleaved, self.device = table, interleaved, table.device
        self._c = _Rope(table.data_ptr(), table.shape[0], 2 * table.shape[1], int(interleaved))
        self.ref = ctypes.addressof(self._c)
        self.bad_pos = torch.zeros(1, dtype=torch.int32, device=table.device)   # a position lay outside the table
        self._entry, self._bad = _lib.lib().jq_rope_dev, self.bad_pos.data_ptr()

    def apply(self, x: torch.Tensor, pos: torch.Tensor, heads: int, head_dim: int, inverse: bool = False,
              out: torch.Tensor | None = None) -> torch.Tensor:
        """Rows [rows, heads * head_dim] turned to their positions (`inverse`: back), into `out` (may be `x`)."""
        index, width = self._index, heads * head_dim
        if index != _device():
            with torch.cuda.device(index):
                return self.apply(x, pos, heads, head_dim, inverse, out)
        at, stride, rows = rows_arg(x, "x", width, index)
        if out is None:
            out = _new(rows, width, dtype=_f32, device=self.device)
            to, out_stride = out.data_ptr(), width
        else:
            to, out_stride, n = rows_arg(out, "out", width, index)
            if n != rows:
                raise JoshuaB200Error(_lib.E_INVALID, f"out has {n} rows for {rows}")
        rc = self._entry(self.ref, at, stride, vector_arg(pos, "pos", rows, torch.int32, index), rows, heads, head_dim, inverse, to,
                         out_stride, self._bad, _raw_stream(index))
        if rc:
            check(rc)
        return out
