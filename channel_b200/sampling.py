"""Whole logits rows on torch tensors: sampling a token per row, scoring given ones, and
accepting drafted ones (ch_sample_rows, ch_score_rows and ch_accept_drafts of
include/channel_cuda.h, where the semantics are stated).

``DeviceSampler`` (engine) draws one stream's token from its 64 top candidates with the
reference's generator and penalties; ``sample_rows`` draws a token for every row of a batch
from the whole vocabulary, each row with its own settings, from random numbers the caller
gives.  ``score_rows`` says how likely given tokens were; ``accept_drafts`` compares the tokens
sampled at the nodes of drafted trees (paged.tree_attention) with what was drafted there.
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib as L
from .paged import _DTYPES, _F32_MAX, _device, _fail, _no_graph, _out_of_range, _run, _status, _vec

_ROWS = struct.Struct("@9Pq2Ifi")  # ChSampleRowsArgs of _lib
_SCORE = struct.Struct("@7Pq3IfiP")  # ChScoreArgs
_ACCEPT = struct.Struct("@7P2IP")    # ChAcceptArgs
_F32, _I32 = torch.float32, torch.int32


class RowScores(NamedTuple):
    logprobs: torch.Tensor      # [rows] float32, of the given tokens
    entropy: torch.Tensor       # [rows] float32
    ranks: torch.Tensor         # [rows] int32, 1 = the most likely token
    top_ids: torch.Tensor       # [rows, top] int32
    top_logprobs: torch.Tensor  # [rows, top] float32


class Accepted(NamedTuple):
    counts: torch.Tensor       # [streams] int32, accepted nodes
    next_tokens: torch.Tensor  # [streams] int32, sampled at the last of them
    kept: torch.Tensor         # [nodes] int32, place among all accepted nodes or -1


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


def score_rows(logits: torch.Tensor, targets: torch.Tensor, top: int = 0, softcap: float = 0.0,
               status: Optional[torch.Tensor] = None) -> RowScores:
    """How likely the token targets[r] (int32) is by row r of logits ``[rows, vocab]`` (f32, f16
    or bf16; rows may be strided): its log-probability and rank, the row's entropy, and its
    ``top`` (at most 64) most likely tokens with their log-probabilities.  A negative target
    gives 0 for the first two.  There is no backward pass."""
    shape = logits.shape
    if len(shape) != 2:
        _fail("score_rows: logits is [rows, vocab]")
    (n, vocab), (row, step) = shape, logits.stride()
    if step != 1 and vocab > 1:
        _fail("score_rows: logits is dense in its last dimension")
    if not abs(softcap) <= _F32_MAX:  # packing would make it infinite
        _fail("score_rows: softcap is out of range")
    if not 0 <= top <= 64:
        _fail("score_rows: top is 0..64")
    if logits.requires_grad:
        _no_graph()
    at = logits.get_device()
    p_targets, p_status = _vec(targets, n, at, "targets"), _status(status, at)
    _device(logits)
    out = logits.new_empty((3 + 2 * top) * n, dtype=_I32)
    logprobs, entropy, ranks, ids, tops = torch.unsafe_split_with_sizes(out, (n, n, n, top * n, top * n))
    if n:
        p = out.data_ptr()
        try:
            args = _SCORE.pack(logits.data_ptr(), p_targets, p, p + 4 * n, p + 8 * n, p + 12 * n, p + (12 + 4 * top) * n, row, n,
                               vocab, top, softcap, _DTYPES.get(logits.dtype, -1), p_status)
        except struct.error as e:
            _out_of_range("score_rows", e)
        _run(L.load().ch_score_rows, at, args)
    return RowScores(logprobs.view(_F32), entropy.view(_F32), ranks, ids.view(n, top), tops.view(_F32).view(n, top))


def accept_drafts(drafted: torch.Tensor, parents: torch.Tensor, starts: torch.Tensor, sampled: torch.Tensor,
                  status: Optional[torch.Tensor] = None) -> Accepted:
    """Which nodes of the streams' drafted trees (rows starts[b] .. starts[b + 1] - 1; a node's
    token, parent in the stream and the token sampled from its logits; all int32) are accepted: the
    stream's node 0, then from each accepted node the first child that is its sampled token.
    ``counts`` are the new tokens of the next ``plan_pages``, and a row's ``kept`` is its place in
    that plan's slots."""
    at = _device(drafted)
    rows = drafted.numel()
    p_drafted, p_parents = _vec(drafted, rows, at, "drafted"), _vec(parents, rows, at, "parents")
    p_starts, p_sampled = _vec(starts, -1, at, "starts"), _vec(sampled, rows, at, "sampled")
    n = starts.shape[0] - 1
    if n < 0:
        _fail("accept_drafts: starts has one number more than there are streams")
    out = drafted.new_empty(2 * n + rows)
    counts, after, kept = torch.unsafe_split_with_sizes(out, (n, n, rows))
    p = out.data_ptr()
    try:
        args = _ACCEPT.pack(p_drafted, p_parents, p_starts, p_sampled, p, p + 4 * n, p + 8 * n, rows, n, _status(status, at))
    except struct.error as e:
        _out_of_range("accept_drafts", e)
    _run(L.load().ch_accept_drafts, at, args)
    return Accepted(counts, after, kept)
