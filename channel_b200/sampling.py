"""Sampling one token per stream from whole logits rows, on torch tensors
(ch_sample_rows of include/channel_cuda.h, where the semantics are stated).

``DeviceSampler`` (engine) draws one stream's token from its 64 top candidates with the
reference's generator and penalties; ``sample_rows`` draws a token for every row of a batch
from the whole vocabulary, each row with its own settings, from random numbers the caller
gives.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib as L
from .paged import _DTYPES, _fail, _run


def _per_row(t: Optional[torch.Tensor], kind, n: int, dev, name: str) -> Optional[int]:
    if t is None:
        return None
    if t.dtype is not kind or t.dim() != 1 or t.shape[0] != n or t.device != dev or (n > 1 and t.stride(0) != 1):
        _fail(f"sample_rows: {name} is a dense {kind} tensor of one value per row on {dev}")
    return t.data_ptr()


def sample_rows(logits: torch.Tensor, uniform: torch.Tensor, temperature: Optional[torch.Tensor] = None,
                top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                min_p: Optional[torch.Tensor] = None,
                softcap: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """tokens (int32), log-probabilities among the kept tokens (float32) and how many tokens
    were kept (int32), one each per row of logits ``[rows, vocab]`` (f32, f16 or bf16; rows
    may be strided).  uniform: float32 in [0, 1) per row.  Settings are tensors of one value
    per row (top_k int32, the rest float32) or None; temperature <= 0 takes the largest
    logit."""
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        _fail("sample_rows: logits is [rows, vocab], dense in its last dimension")
    n, vocab = logits.shape
    dev, f32 = logits.device, torch.float32
    out = torch.empty((3, n), dtype=torch.int32, device=dev)
    tokens, kept, logprobs = out.unbind(0)
    logprobs = logprobs.view(f32)
    if n == 0:
        return tokens, logprobs, kept
    at = out.data_ptr()
    if uniform is None:
        _fail("sample_rows: uniform is needed")
    a = L.ChSampleRowsArgs(
        logits.data_ptr(), _per_row(uniform, f32, n, dev, "uniform"), _per_row(temperature, f32, n, dev, "temperature"),
        _per_row(top_p, f32, n, dev, "top_p"), _per_row(min_p, f32, n, dev, "min_p"),
        _per_row(top_k, torch.int32, n, dev, "top_k"), at, at + 4 * n, at + 8 * n, logits.stride(0), n, vocab, softcap,
        _DTYPES.get(logits.dtype, -1))
    _run(L.load().ch_sample_rows, dev, C.byref(a))
    return tokens, logprobs, kept
