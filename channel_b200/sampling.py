"""Sampling one token per stream from whole logits rows, on torch tensors
(ch_sample_rows of include/channel_cuda.h, where the semantics are stated).

``DeviceSampler`` (engine) draws one stream's token from its 64 top candidates with the
reference's generator and penalties; ``sample_rows`` draws a token for every row of a batch
from the whole vocabulary, each row with its own settings, from random numbers the caller
gives.
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from . import _lib as L
from .paged import _DTYPES, _F32_MAX, _device, _fail, _no_graph, _out_of_range, _run

_ROWS = struct.Struct("@9Pq2Ifi")  # ChSampleRowsArgs of _lib
_F32, _I32 = torch.float32, torch.int32


def _per_row(t: Optional[torch.Tensor], kind, n: int, at: int, name: str) -> int:
    if t is None:
        return 0
    if t.dtype is not kind or t.dim() != 1 or t.shape[0] != n or t.get_device() != at or not t.is_contiguous():
        _fail(f"sample_rows: {name} is a dense {kind} tensor of one value per row on the logits' device")
    return t.data_ptr()


def sample_rows(logits: torch.Tensor, uniform: torch.Tensor, temperature: Optional[torch.Tensor] = None,
                top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                min_p: Optional[torch.Tensor] = None,
                softcap: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """tokens (int32), log-probabilities among the kept tokens (float32) and how many tokens
    were kept (int32), one each per row of logits ``[rows, vocab]`` (f32, f16 or bf16; rows
    may be strided).  uniform: float32 in [0, 1) per row.  Settings are tensors of one value
    per row (top_k int32, the rest float32) or None; temperature <= 0 takes the largest
    logit.  There is no backward pass."""
    shape = logits.shape
    if len(shape) != 2:
        _fail("sample_rows: logits is [rows, vocab]")
    (n, vocab), (row, step) = shape, logits.stride()
    if step != 1 and vocab > 1:
        _fail("sample_rows: logits is dense in its last dimension")
    if uniform is None:
        _fail("sample_rows: uniform is needed")
    if not abs(softcap) <= _F32_MAX:  # packing would make it infinite
        _fail("sample_rows: softcap is out of range")
    if logits.requires_grad:
        _no_graph()
    at = logits.get_device()
    p_uniform, p_temp = _per_row(uniform, _F32, n, at, "uniform"), _per_row(temperature, _F32, n, at, "temperature")
    p_top_p, p_min_p = _per_row(top_p, _F32, n, at, "top_p"), _per_row(min_p, _F32, n, at, "min_p")
    p_top_k = _per_row(top_k, _I32, n, at, "top_k")
    _device(logits)
    out = logits.new_empty(3 * n, dtype=_I32)
    tokens, kept, logprobs = torch.unsafe_split_with_sizes(out, (n, n, n))
    logprobs = logprobs.view(_F32)
    if n:
        p = out.data_ptr()
        try:
            args = _ROWS.pack(logits.data_ptr(), p_uniform, p_temp, p_top_p, p_min_p, p_top_k, p, p + 4 * n, p + 8 * n, row, n,
                              vocab, softcap, _DTYPES.get(logits.dtype, -1))
        except struct.error as e:
            _out_of_range("sample_rows", e)
        _run(L.load().ch_sample_rows, at, args)
    return tokens, logprobs, kept
