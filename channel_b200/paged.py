"""Streams that share a prompt, on torch tensors: page plans, page writes and attention
over the shared prefix (ch_page_plan, ch_paged_kv_write, ch_prefix_attention of
include/channel_cuda.h, where the semantics are stated).

A layer's K rows lie in a pool ``[n_pages, page_size, n_kv, head_dim]`` and its V rows in a
second one with the same strides.  A decode step of many streams is

    plan = plan_pages(lens, new, table, free, page_size, max_tokens, prefix_len)  # once per step
    kv_write(k, v, plan.slots, k_pool, v_pool)                                    # per layer
    out = prefix_attention(q, k_pool, v_pool, plan.table, plan.lens, prefix_table, prefix_len)
    tokens, _, _ = sampling.sample_rows(logits, uniform, ...)                     # once per step

Every call runs on torch's current stream of the tensors' device and returns without
waiting for it; none has a backward pass, and a tensor that requires a gradient is refused
unless gradients are off.  ``status`` (int32 tensor of one element, optional) collects the bits of
ch_ctx_device_status that the kernels report; ``check_status`` raises on them.
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import torch

from . import _lib as L

_DTYPES = {torch.float32: L.CH_F32, torch.float16: L.CH_F16, torch.bfloat16: L.CH_BF16}
_I32 = torch.int32
_F32_MAX = torch.finfo(torch.float32).max
_NO_PAGES, _BAD = 1 << 5, (1 << 1) | (1 << 2)

# A step makes these calls once per layer, so their host time counts: the argument records
# are packed in one go (the layouts of the ctypes structures of the same name in _lib).
_PLAN = struct.Struct("@10Pq6IP")
_WRITE = struct.Struct("@5P7q5I2iP")
_ATTEND = struct.Struct("@7P8q9IfiP")

try:  # torch's current stream of a device as a cudaStream_t, without building a Stream object
    _stream_of = torch._C._cuda_getCurrentRawStream
except AttributeError:
    def _stream_of(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


class PagePlan(NamedTuple):
    table: torch.Tensor      # [streams, columns], the given table
    lens: torch.Tensor       # [streams] after the step
    starts: torch.Tensor     # [streams + 1]
    slots: torch.Tensor      # [max_tokens]
    positions: torch.Tensor  # [max_tokens]
    rows: torch.Tensor       # [max_tokens]
    counts: torch.Tensor     # [2] packed tokens, pages taken


def _fail(msg: str):
    raise L.ChannelError(L.CH_EINVAL, msg)


def _out_of_range(what: str, why: struct.error):
    _fail(f"{what}: an argument is out of range ({why})")


def _no_graph() -> None:
    """For a tensor that requires a gradient: the operators have no backward pass."""
    if torch.is_grad_enabled():
        _fail("a tensor requires a gradient, and the call has none: detach it or use torch.no_grad()")


def _vec(t: torch.Tensor, n: int, at: int, name: str) -> int:
    """Pointer of a dense int32 vector of n elements (n < 0: any) on device `at`."""
    if t.dtype is not _I32 or t.dim() != 1 or t.get_device() != at or (n >= 0 and t.shape[0] != n) or \
            not t.is_contiguous():
        _fail(f"{name}: a dense int32 vector{f' of {n} elements' if n >= 0 else ''} on the other tensors' device is wanted")
    return t.data_ptr()


def _table(t: torch.Tensor, n: int, at: int, name: str) -> int:
    """Pointer of an int32 table of n rows, dense along a row, on device `at`."""
    if t.dtype is not _I32 or t.dim() != 2 or t.get_device() != at or t.shape[0] != n or \
            (t.stride(1) != 1 and t.shape[1] > 1 and n > 0):
        _fail(f"{name}: an int32 table of {n} rows, dense along a row, on the other tensors' device is wanted")
    return t.data_ptr()


def _status(status: Optional[torch.Tensor], at: int) -> int:
    if status is None:
        return 0
    if status.dtype is not _I32 or status.get_device() != at or status.numel() != 1:
        _fail("status: an int32 tensor of one element on the other tensors' device is wanted")
    return status.data_ptr()


def _run(fn, at: int, *args) -> None:
    """fn(*args, stream) on device `at` and its current torch stream."""
    if at == torch.cuda.current_device():
        rc = fn(*args, _stream_of(at))
    else:
        with torch.cuda.device(at):
            rc = fn(*args, _stream_of(at))
    if rc:
        L.check(rc)


def _device(t: torch.Tensor) -> int:
    at = t.get_device()
    if at < 0:
        _fail("tensors on a CUDA device are wanted")
    return at


def check_status(status: torch.Tensor) -> None:
    """Reads and clears a status word (waits for the stream); raises on a reported error."""
    bits = int(status.item())
    status.zero_()
    if bits & _NO_PAGES:
        raise L.ChannelError(L.CH_ENOMEM, "a page plan ran out of pages, table columns, token rows or slot numbers")
    if bits & _BAD:
        raise L.ChannelError(L.CH_EDEVICE, "a kernel saw a slot or page outside its pool")
    if bits:
        raise L.ChannelError(L.CH_ETIMEOUT, "a bounded device wait gave up")


def plan_pages(lens: torch.Tensor, new_tokens: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor,
               page_size: int, max_tokens: int, prefix_len: int = 0,
               status: Optional[torch.Tensor] = None) -> PagePlan:
    """Block tables (``table``, in place), slot map, positions and row map of a step that
    appends ``new_tokens`` to streams holding ``lens`` tokens; pages come from the front of
    ``free_pages`` (``counts[1]`` of them)."""
    at, n = _device(lens), lens.numel()
    p_lens, p_new = _vec(lens, n, at, "lens"), _vec(new_tokens, n, at, "new_tokens")
    p_free, p_table = _vec(free_pages, -1, at, "free_pages"), _table(table, n, at, "table")
    if not 0 <= max_tokens < 1 << 31 or prefix_len < 0 or page_size < 0:
        _fail("plan_pages: a size is negative or 2^31 or more")
    pad = -max_tokens & 3  # the token arrays start on 16 bytes
    buf = lens.new_empty(3 * (max_tokens + pad) + 2 * n + 3)
    if pad:
        slots, _, positions, _, rows, _, lens_out, starts, counts = buf.split_with_sizes(
            (max_tokens, pad, max_tokens, pad, max_tokens, pad, n, n + 1, 2))
    else:
        slots, positions, rows, lens_out, starts, counts = torch.unsafe_split_with_sizes(
            buf, (max_tokens, max_tokens, max_tokens, n, n + 1, 2))
    p, step = buf.data_ptr(), 4 * (max_tokens + pad)
    try:
        args = _PLAN.pack(p_lens, p_new, p_free, p_table, p + 3 * step, p + 3 * step + 4 * n, p, p + step, p + 2 * step,
                          p + 3 * step + 8 * n + 4, table.stride(0), n, table.shape[1], free_pages.shape[0], page_size,
                          max_tokens, prefix_len, _status(status, at))
    except struct.error as e:
        _out_of_range("plan_pages", e)
    _run(L.load().ch_page_plan, at, args)
    return PagePlan(table, lens_out, starts, slots, positions, rows, counts)


def _pools(k_pool: torch.Tensor, v_pool: torch.Tensor, at: int):
    shape, strides = k_pool.shape, k_pool.stride()
    if len(shape) != 4 or shape != v_pool.shape or strides != v_pool.stride() or k_pool.dtype is not v_pool.dtype or \
            k_pool.get_device() != at or v_pool.get_device() != at or strides[3] != 1:
        _fail("k_pool and v_pool: [n_pages, page_size, n_kv, head_dim] of one type, strides and device")
    return shape, strides


def kv_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
             status: Optional[torch.Tensor] = None) -> None:
    """Rows k[t], v[t] (``[tokens, n_kv, head_dim]``, any token and head strides) into slot
    slots[t] of the pools; negative slots are skipped."""
    at = k.get_device()
    (pages, page, n_kv, dim), (ps, ts, hs, _) = _pools(k_pool, v_pool, at)
    if k.requires_grad or v.requires_grad or k_pool.requires_grad or v_pool.requires_grad:
        _no_graph()
    shape, kind, k_strides, v_strides = k.shape, k.dtype, k.stride(), v.stride()
    if len(shape) != 3 or shape != v.shape or shape[1] != n_kv or shape[2] != dim or kind is not v.dtype or \
            v.get_device() != at or k_strides[2] != 1 or v_strides[2] != 1:
        _fail("kv_write: k and v are [tokens, n_kv, head_dim] of one type, dense in the last dimension")
    _device(k)
    try:
        args = _WRITE.pack(k.data_ptr(), v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
                           _vec(slots, shape[0], at, "slots"), k_strides[0], k_strides[1], v_strides[0], v_strides[1], ps,
                           ts, hs, shape[0], n_kv, dim, page, pages, _DTYPES.get(kind, -1), _DTYPES.get(k_pool.dtype, -1),
                           _status(status, at))
    except struct.error as e:
        _out_of_range("kv_write", e)
    _run(L.load().ch_paged_kv_write, at, args)


def prefix_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, table: torch.Tensor,
                     lens: torch.Tensor, prefix_table: Optional[torch.Tensor] = None, prefix_len: int = 0,
                     window: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one query token per stream (q: ``[streams, n_q, head_dim]``) over the
    prefix_len tokens in the pages of prefix_table and the stream's own lens[b] tokens in
    those of table[b]; window > 0 leaves the last ``window`` positions visible.  scale
    defaults to head_dim ** -0.5."""
    at = q.get_device()
    (pages, page, n_kv, dim), (ps, ts, hs, _) = _pools(k_pool, v_pool, at)
    if q.requires_grad or k_pool.requires_grad or v_pool.requires_grad:
        _no_graph()
    shape, kind = q.shape, q.dtype
    if len(shape) != 3 or shape[2] != dim or kind is not k_pool.dtype or q.stride(2) != 1:
        _fail("prefix_attention: q is [streams, n_q, head_dim] of the pools' type, dense in the last dimension")
    n, n_q, _ = shape
    if prefix_len < 0 or window < 0:
        _fail("prefix_attention: negative size")
    p_prefix = 0 if prefix_table is None else _vec(prefix_table, -1, at, "prefix_table")
    if prefix_len and (prefix_table is None or prefix_table.shape[0] * page < prefix_len):
        _fail("prefix_attention: prefix_table is shorter than prefix_len")
    p_table, p_lens = _table(table, n, at, "table"), _vec(lens, n, at, "lens")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != shape or out.dtype is not kind or out.get_device() != at or out.stride(2) != 1:
        _fail("prefix_attention: out is like q")
    _device(q)
    (qs, qh, _), (os, oh, _) = q.stride(), out.stride()
    if scale is None:
        scale = dim ** -0.5
    elif not abs(scale) <= _F32_MAX:  # packing would make it infinite
        _fail("prefix_attention: scale is out of range")
    try:
        args = _ATTEND.pack(q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr(), p_prefix, p_table, p_lens, qs,
                            qh, os, oh, ps, ts, hs, table.stride(0), n, n_q, n_kv, dim, page, pages, table.shape[1],
                            prefix_len, window, scale, _DTYPES.get(kind, -1), _status(status, at))
    except struct.error as e:
        _out_of_range("prefix_attention", e)
    lib = L.load()
    need = lib.ch_prefix_attention_workspace(args)
    if need:  # torch's caching allocator hands the workspace out in the stream's order
        work = q.new_empty(need, dtype=torch.uint8)
        _run(lib.ch_prefix_attention, at, args, work.data_ptr(), need)
    else:  # sizes the call refuses
        _run(lib.ch_prefix_attention, at, args, None, 0)
    return out
