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
waiting for it.  ``status`` (int32 tensor of one element, optional) collects the bits of
ch_ctx_device_status that the kernels report; ``check_status`` raises on them.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib as L

_DTYPES = {torch.float32: L.CH_F32, torch.float16: L.CH_F16, torch.bfloat16: L.CH_BF16}
_NO_PAGES, _BAD = 1 << 5, (1 << 1) | (1 << 2)


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


def _i32(t: torch.Tensor, dim: int, dev, name: str) -> int:
    """Pointer of a dense int32 tensor (the last dimension; a table's rows may be strided)."""
    if t.dtype is not torch.int32 or t.dim() != dim or t.device != dev or (t.stride(-1) != 1 and t.numel() > 1):
        _fail(f"{name}: a {dim}-dimensional int32 tensor on {dev}, dense in its last dimension, is wanted")
    return t.data_ptr()


def _status(status: Optional[torch.Tensor], dev) -> Optional[int]:
    if status is None:
        return None
    if status.dtype is not torch.int32 or status.device != dev or status.numel() != 1:
        _fail("status: an int32 tensor of one element on the other tensors' device is wanted")
    return status.data_ptr()


def _run(fn, dev, *args) -> None:
    """fn(*args, stream) on dev's current torch stream."""
    if dev.type != "cuda":
        _fail("tensors on a CUDA device are wanted")
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    if rc != L.CH_OK:
        L.check(rc)


def check_status(status: torch.Tensor) -> None:
    """Reads and clears a status word (waits for the stream); raises on a reported error."""
    bits = int(status.item())
    status.zero_()
    if bits & _NO_PAGES:
        raise L.ChannelError(L.CH_ENOMEM, "a page plan ran out of pages, table columns or token rows")
    if bits & _BAD:
        raise L.ChannelError(L.CH_EDEVICE, "a kernel saw a slot or page outside its pool")


def plan_pages(lens: torch.Tensor, new_tokens: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor,
               page_size: int, max_tokens: int, prefix_len: int = 0,
               status: Optional[torch.Tensor] = None) -> PagePlan:
    """Block tables (``table``, in place), slot map, positions and row map of a step that
    appends ``new_tokens`` to streams holding ``lens`` tokens; pages come from the front of
    ``free_pages`` (``counts[1]`` of them)."""
    dev, n = lens.device, lens.shape[0]
    pad = (max_tokens + 3) & ~3  # the token arrays start on 16 bytes
    buf = torch.empty(3 * pad + 2 * n + 3, dtype=torch.int32, device=dev)
    slots, positions, rows, lens_out, starts, counts = buf.split_with_sizes((pad, pad, pad, n, n + 1, 2))
    a = L.ChPagePlanArgs(
        _i32(lens, 1, dev, "lens"), _i32(new_tokens, 1, dev, "new_tokens"), _i32(free_pages, 1, dev, "free_pages"),
        _i32(table, 2, dev, "table"), lens_out.data_ptr(), starts.data_ptr(), slots.data_ptr(), positions.data_ptr(),
        rows.data_ptr(), counts.data_ptr(), table.stride(0), n, table.shape[1], free_pages.shape[0], page_size,
        max_tokens, prefix_len, _status(status, dev))
    if new_tokens.shape[0] != n or table.shape[0] != n:
        _fail("plan_pages: lens, new_tokens and table differ in their number of streams")
    _run(L.load().ch_page_plan, dev, C.byref(a))
    if pad != max_tokens:
        slots, positions, rows = slots[:max_tokens], positions[:max_tokens], rows[:max_tokens]
    return PagePlan(table, lens_out, starts, slots, positions, rows, counts)


def _pools(k_pool: torch.Tensor, v_pool: torch.Tensor, dev):
    if k_pool.dim() != 4 or k_pool.shape != v_pool.shape or k_pool.stride() != v_pool.stride() or \
            k_pool.dtype is not v_pool.dtype or k_pool.device != dev or v_pool.device != dev or k_pool.stride(3) != 1:
        _fail("k_pool and v_pool: [n_pages, page_size, n_kv, head_dim] of one type, strides and device")
    return k_pool.shape, k_pool.stride()


def kv_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
             status: Optional[torch.Tensor] = None) -> None:
    """Rows k[t], v[t] (``[tokens, n_kv, head_dim]``, any token and head strides) into slot
    slots[t] of the pools; negative slots are skipped."""
    dev = k.device
    (pages, page, n_kv, dim), (ps, ts, hs, _) = _pools(k_pool, v_pool, dev)
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (n_kv, dim) or k.dtype is not v.dtype or \
            v.device != dev or k.stride(2) != 1 or v.stride(2) != 1 or slots.shape[0] != k.shape[0]:
        _fail("kv_write: k and v are [tokens, n_kv, head_dim] of one type, with one slot per token")
    a = L.ChKvWriteArgs(k.data_ptr(), v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), _i32(slots, 1, dev, "slots"),
                        k.stride(0), k.stride(1), v.stride(0), v.stride(1), ps, ts, hs, k.shape[0], n_kv, dim, page,
                        pages, _DTYPES.get(k.dtype, -1), _DTYPES.get(k_pool.dtype, -1), _status(status, dev))
    _run(L.load().ch_paged_kv_write, dev, C.byref(a))


def prefix_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, table: torch.Tensor,
                     lens: torch.Tensor, prefix_table: Optional[torch.Tensor] = None, prefix_len: int = 0,
                     window: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one query token per stream (q: ``[streams, n_q, head_dim]``) over the
    prefix_len tokens in the pages of prefix_table and the stream's own lens[b] tokens in
    those of table[b]; window > 0 leaves the last ``window`` positions visible.  scale
    defaults to head_dim ** -0.5."""
    dev = q.device
    (pages, page, n_kv, dim), (ps, ts, hs, _) = _pools(k_pool, v_pool, dev)
    if q.dim() != 3 or q.shape[2] != dim or q.dtype is not k_pool.dtype or q.stride(2) != 1 or \
            lens.shape[0] != q.shape[0] or table.shape[0] != q.shape[0]:
        _fail("prefix_attention: q is [streams, n_q, head_dim] of the pools' type, with lens and table rows per stream")
    n, n_q, _ = q.shape
    if out is None:
        out = torch.empty((n, n_q, dim), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype is not q.dtype or out.device != dev or out.stride(2) != 1:
        _fail("prefix_attention: out is like q")
    if prefix_len and (prefix_table is None or prefix_table.shape[0] * page < prefix_len):
        _fail("prefix_attention: prefix_table is shorter than prefix_len")
    a = L.ChPrefixAttnArgs(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr(),
        None if prefix_table is None else _i32(prefix_table, 1, dev, "prefix_table"), _i32(table, 2, dev, "table"),
        _i32(lens, 1, dev, "lens"), q.stride(0), q.stride(1), out.stride(0), out.stride(1), ps, ts, hs,
        table.stride(0), n, n_q, n_kv, dim, page, pages, table.shape[1], prefix_len, window,
        dim ** -0.5 if scale is None else scale, _DTYPES.get(q.dtype, -1), _status(status, dev))
    lib, ref = L.load(), C.byref(a)
    if dev.type != "cuda":
        _fail("tensors on a CUDA device are wanted")
    need = lib.ch_prefix_attention_workspace(ref)
    # torch's caching allocator hands the workspace out in the stream's order
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _run(lib.ch_prefix_attention, dev, ref, work.data_ptr() if need else None, need)
    return out
