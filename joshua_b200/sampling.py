"""Sampling on the device: temperature, top-k, top-p and min-p of every row, drawn with given random numbers."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import JoshuaB200Error, check
from .rope import _device, _new, _raw_stream, block_arg, device_index, rows_arg, vector_arg

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
    f32, i32 = torch.float32, torch.int32
    index = device_index(logits, "logits", f32)
    if index != _device():
        with torch.cuda.device(index):
            return sample(logits, uniform, temperature, top_k, top_p, min_p, repetition_penalty, window, window_state, pos, token)
    if logits.dim() != 2:
        raise JoshuaB200Error(_lib.E_INVALID, "logits must be [rows, vocab]")
    vocab = logits.size(1)
    at, stride, rows = rows_arg(logits, "logits", vocab, index)
    if token is None:
        token = _new(rows, dtype=i32, device=logits.device)
    prob = _new(rows, dtype=f32, device=logits.device)
    rc = _entry(at, stride, rows, vocab, vector_arg(uniform, "uniform", rows, f32, index),
                None if temperature is None else vector_arg(temperature, "temperature", rows, f32, index),
                None if top_k is None else vector_arg(top_k, "top_k", rows, i32, index),
                None if top_p is None else vector_arg(top_p, "top_p", rows, f32, index),
                None if min_p is None else vector_arg(min_p, "min_p", rows, f32, index), repetition_penalty,
                None if window is None else block_arg(window, "window", (rows, WINDOW), i32, index),
                None if window_state is None else block_arg(window_state, "window_state", (rows, 2), i32, index),
                vector_arg(token, "token", rows, i32, index), prob.data_ptr(),
                None if pos is None else vector_arg(pos, "pos", rows, i32, index), _raw_stream(index))
    if rc:
        check(rc)
    return token, prob
