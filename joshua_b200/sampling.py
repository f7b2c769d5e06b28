"""Sampling on the device: temperature, top-k, top-p and min-p of every row, drawn with given random numbers."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import JoshuaB200Error, check
from .rope import rows_arg, stream_of, tensor_arg, vector_arg

WINDOW = 64
_entry = None


def sample(logits: torch.Tensor, uniform: torch.Tensor, temperature=None, top_k=None, top_p=None, min_p=None,
           repetition_penalty: float = 1.0, window: torch.Tensor | None = None, window_state: torch.Tensor | None = None,
           pos: torch.Tensor | None = None, token: torch.Tensor | None = None):
    """(token int32 [rows], its probability f32 [rows]) of logits [rows, vocab] and numbers `uniform` [rows] in [0, 1).

    temperature, top_p, min_p (f32) and top_k (int32) are vectors of `rows`, or None: off (temperature 1).  `window` (int32
    [rows, 64]) and `window_state` (int32 [rows, 2]) hold recent ids for `repetition_penalty` and take the new one; `pos` is
    advanced by one.  A row without a token to draw gives -1 and 0."""
    global _entry
    if _entry is None:
        _entry = _lib.lib().jq_sample_dev
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2:
        raise JoshuaB200Error(_lib.E_INVALID, "logits must be [rows, vocab]")
    at, stride, rows = rows_arg(logits, "logits", logits.shape[1])
    dev, f32, i32 = logits.device, torch.float32, torch.int32

    def vec(t, name, dtype):
        return None if t is None else vector_arg(t, name, rows, dtype, dev)

    for t, name, width in ((window, "window", WINDOW), (window_state, "window_state", 2)):
        if t is not None and (tensor_arg(t, name, i32, dev).shape != (rows, width) or not t.is_contiguous()):
            raise JoshuaB200Error(_lib.E_INVALID, f"{name} must be contiguous, [{rows}, {width}]")
    if token is None:
        token = torch.empty(rows, dtype=i32, device=dev)
    prob = torch.empty(rows, dtype=f32, device=dev)
    check(_entry(at, stride, rows, logits.shape[1], vec(uniform, "uniform", f32), vec(temperature, "temperature", f32),
                 vec(top_k, "top_k", i32), vec(top_p, "top_p", f32), vec(min_p, "min_p", f32), repetition_penalty,
                 window.data_ptr() if window is not None else None, window_state.data_ptr() if window_state is not None else None,
                 vec(token, "token", i32), prob.data_ptr(), vec(pos, "pos", i32), stream_of(logits)))
    return token, prob
