"""Streams that continue one prompt, end to end: page plan, page writes, attention over the
shared pages and row sampling around the Q4 projections of the op-level interface.

``SharedPromptDecoder`` holds a decoder of seeded synthetic Q4 weights in the reference's
layer order (input norm, q|k|v, per-head RoPE at the token's position, attention, o,
residual, pre-FFN norm, GELU gate * up, down, residual; src/model/forward.zig:49-230) whose
K/V caches are pages.  The prompt is decoded once, into the pages of a first stream; those
pages then become the shared prefix of a batch of streams, each of which owns only the pages
of its own tokens.  All work runs on the context's stream; a step called from another torch
stream is ordered after that stream's work, and what follows there after the step.

    python -m channel_b200.shared_prompt [--streams N] [--prompt N] [--tokens N]
"""
from __future__ import annotations

import argparse
import math
import time
from dataclasses import dataclass

import torch

from . import _lib as L
from .engine import GpuContext
from .paged import PagePlan, _fail, check_status, kv_write, plan_pages, prefix_attention
from .sampling import sample_rows


@dataclass
class DecoderShape:
    vocab: int = 4096
    hidden: int = 512
    intermediate: int = 1024
    layers: int = 3
    n_q: int = 4
    n_kv: int = 2
    head_dim: int = 256
    rope_theta: float = 10000.0
    eps: float = 1e-6


class SharedPromptDecoder:
    def __init__(self, ctx: GpuContext, shape: DecoderShape, n_pages: int, page_size: int = 16, seed: int = 7):
        self.ctx, self.shape, self.page_size = ctx, shape, page_size
        self.lib = L.load()
        self.device = torch.device("cuda", ctx.device)
        self.stream = torch.cuda.ExternalStream(ctx.stream, device=self.device)
        s = shape
        with torch.cuda.stream(self.stream):
            g = torch.Generator(self.device).manual_seed(seed)
            self.embed = 0.5 * torch.randn(s.vocab, s.hidden, generator=g, device=self.device)
            self.layers = []
            for layer in range(s.layers):
                make = lambda t, rows, cols: self._weight(self.lib.ch_tensor_seed(seed, layer, t), rows, cols)  # noqa: E731
                self.layers.append(dict(
                    qkv=make(0, (s.n_q + 2 * s.n_kv) * s.head_dim, s.hidden), o=make(1, s.hidden, s.n_q * s.head_dim),
                    mlp=self._gate_up(seed, layer), down=make(4, s.hidden, s.intermediate)))
            self.head = self._weight(self.lib.ch_tensor_seed(seed, s.layers, 5), s.vocab, s.hidden)
            self.ones = torch.ones(max(s.hidden, s.n_q * s.head_dim), device=self.device)
            pool = (s.layers, n_pages, page_size, s.n_kv, s.head_dim)
            self.k_pool = torch.zeros(pool, dtype=torch.float16, device=self.device)
            self.v_pool = torch.zeros(pool, dtype=torch.float16, device=self.device)
            self.free = torch.arange(n_pages, dtype=torch.int32, device=self.device)
            self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.max_pages = n_pages

    # ---- Q4 weights and the op-level calls ----

    def _blocks(self, seed: int, rows: int, cols: int) -> torch.Tensor:
        blocks = torch.empty(rows * (cols // 32) * 5, dtype=torch.int32, device=self.device)
        L.check(self.lib.ch_gen_q4_blocks(self.ctx.handle, blocks.data_ptr(), rows, cols, seed, 0.3 / math.sqrt(cols)))
        return blocks

    def _weight(self, seed: int, rows: int, cols: int):
        tiles = torch.empty(self.lib.ch_q4_tile_bytes(rows, cols), dtype=torch.uint8, device=self.device)
        L.check(self.lib.ch_q4_pack(self.ctx.handle, self._blocks(seed, rows, cols).data_ptr(), rows, cols, tiles.data_ptr()))
        self.ctx.synchronize()  # the blocks are freed here
        return tiles, rows, cols

    def _gate_up(self, seed: int, layer: int):
        s = self.shape
        gate, up = (self._blocks(self.lib.ch_tensor_seed(seed, layer, t), s.intermediate, s.hidden) for t in (2, 3))
        tiles = torch.empty(self.lib.ch_q4_tile_bytes(2 * s.intermediate, s.hidden), dtype=torch.uint8, device=self.device)
        L.check(self.lib.ch_q4_pack_gateup(self.ctx.handle, gate.data_ptr(), up.data_ptr(), s.intermediate, s.hidden,
                                           tiles.data_ptr()))
        self.ctx.synchronize()
        return tiles, s.intermediate, s.hidden

    def _gemm(self, weight, x: torch.Tensor, fn: str = "ch_batch_gemm_q4") -> torch.Tensor:
        tiles, rows, cols = weight
        y = torch.empty(x.shape[0], rows, device=self.device)
        L.check(getattr(self.lib, fn)(self.ctx.handle, tiles.data_ptr(), rows, cols, x.data_ptr(), x.shape[0], y.data_ptr()))
        return y

    def _norm(self, x: torch.Tensor) -> torch.Tensor:
        y = torch.empty_like(x)
        L.check(self.lib.ch_rmsnorm(self.ctx.handle, x.data_ptr(), self.ones.data_ptr(), y.data_ptr(), x.numel() // x.shape[-1],
                                    x.shape[-1], self.shape.eps))
        return y

    def _rope(self, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        half = x.shape[-1] // 2
        rate = self.shape.rope_theta ** (-torch.arange(half, device=self.device, dtype=torch.float64) / half)
        angle = (positions.double()[:, None] * rate).float()[:, None]
        cos, sin = angle.cos(), angle.sin()
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    # ---- one token per stream ----

    def step(self, tokens: torch.Tensor, plan: PagePlan, prefix_table=None, prefix_len: int = 0) -> torch.Tensor:
        """Logits ``[streams, vocab]`` of one token per stream, placed by plan (made for one
        new token per stream)."""
        caller = torch.cuda.current_stream(self.device)
        if caller == self.stream:
            return self._step(tokens, plan, prefix_table, prefix_len)
        self.stream.wait_stream(caller)
        with torch.cuda.stream(self.stream):
            logits = self._step(tokens, plan, prefix_table, prefix_len)
        caller.wait_stream(self.stream)
        logits.record_stream(caller)
        return logits

    def _step(self, tokens: torch.Tensor, plan: PagePlan, prefix_table, prefix_len: int) -> torch.Tensor:
        s, n = self.shape, tokens.shape[0]
        x = self.embed[tokens.long()] * math.sqrt(s.hidden)
        for layer, w in enumerate(self.layers):
            qkv = self._gemm(w["qkv"], self._norm(x)).view(n, s.n_q + 2 * s.n_kv, s.head_dim)
            q = self._rope(self._norm(qkv[:, :s.n_q].contiguous()), plan.positions)
            k = self._rope(self._norm(qkv[:, s.n_q:s.n_q + s.n_kv].contiguous()), plan.positions)
            kv_write(k, qkv[:, s.n_q + s.n_kv:].contiguous(), plan.slots, self.k_pool[layer], self.v_pool[layer], self.status)
            a = prefix_attention((2.0 * q).half(), self.k_pool[layer], self.v_pool[layer], plan.table, plan.lens, prefix_table,
                                 prefix_len, status=self.status)
            x = x + self._gemm(w["o"], a.float().view(n, -1))
            x = x + self._gemm(w["down"], self._gemm(w["mlp"], self._norm(x), "ch_batch_fused_mlp_q4"))
        return self._gemm(self.head, self._norm(x))

    def _plan(self, lens, table, prefix_len: int) -> PagePlan:
        plan = plan_pages(lens, torch.ones_like(lens), table, self.free, self.page_size, lens.shape[0], prefix_len,
                          status=self.status)
        self.free = self.free[int(plan.counts[1]):]
        return plan

    def decode(self, prompt, streams: int, n_tokens: int, temperature: float = 0.0, share: bool = True, seed: int = 1,
               **filters) -> torch.Tensor:
        """n_tokens tokens for each of `streams` continuations of one prompt (a list of token
        ids), ``[streams, n_tokens]``.  share: the prompt is decoded once and its pages are
        shared; otherwise every stream holds a copy of its own."""
        prompt = [int(t) for t in prompt]
        if streams < 1 or n_tokens < 1 or not prompt:
            _fail("decode: a stream, a token of the prompt and a token to decode are wanted at least")
        if min(prompt) < 0 or max(prompt) >= self.shape.vocab:  # an index past the table is a fault on the device
            _fail(f"decode: token ids are 0..{self.shape.vocab - 1}")
        with torch.cuda.stream(self.stream), torch.no_grad():
            g = torch.Generator(self.device).manual_seed(seed)
            self.free = torch.arange(self.max_pages, dtype=torch.int32, device=self.device)
            first = 1 if share else streams
            cols = -(-(len(prompt) + n_tokens) // self.page_size)
            lens = torch.zeros(first, dtype=torch.int32, device=self.device)
            table = torch.full((first, cols), -1, dtype=torch.int32, device=self.device)
            for token in prompt:
                plan = self._plan(lens, table, 0)
                logits = self.step(torch.full((first,), token, device=self.device), plan)
                lens = plan.lens
            prefix_table, prefix_len = None, 0
            if share:  # the first stream's pages become the prefix of all
                prefix_table, prefix_len = table[0, :-(-len(prompt) // self.page_size)].contiguous(), len(prompt)
                logits = logits.expand(streams, -1)
                lens = torch.zeros(streams, dtype=torch.int32, device=self.device)
                table = torch.full((streams, -(-n_tokens // self.page_size)), -1, dtype=torch.int32, device=self.device)
            heat = torch.full((streams,), temperature, device=self.device)
            filters = {k: torch.full((streams,), v, device=self.device, dtype=torch.int32 if k == "top_k" else torch.float32)
                       for k, v in filters.items()}
            out = []
            while True:
                tokens, _, _ = sample_rows(logits, torch.rand(streams, generator=g, device=self.device), temperature=heat,
                                           softcap=30.0, **filters)
                out.append(tokens)
                if len(out) == n_tokens:
                    break
                plan = self._plan(lens, table, prefix_len)
                logits = self.step(tokens, plan, prefix_table, prefix_len)
                lens = plan.lens
            result = torch.stack(out, 1)
            check_status(self.status)
            if int(result.min()) < 0:  # and what followed took another token's embedding
                raise L.ChannelError(L.CH_EDEVICE, "decode: a row of logits had nothing to choose from (NaN or -inf throughout)")
        self.stream.synchronize()
        return result


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--streams", type=int, default=32)
    p.add_argument("--prompt", type=int, default=200)
    p.add_argument("--tokens", type=int, default=32)
    a = p.parse_args()
    ctx = GpuContext.init(0)
    pages = a.streams * (-(-(a.prompt + a.tokens) // 16) + 1)
    d = SharedPromptDecoder(ctx, DecoderShape(), pages)
    prompt = [(37 * i + 11) % d.shape.vocab for i in range(a.prompt)]
    for timed in (False, True):  # first both once, untimed: the first calls load kernels
        for share in (True, False):
            t = time.perf_counter()
            tokens = d.decode(prompt, a.streams, a.tokens, temperature=1.0, share=share, top_k=64, top_p=0.95, min_p=0.02)
            t = time.perf_counter() - t
            if timed:
                print(f"{'shared prompt' if share else 'own copies   '}: {a.streams} streams x {tokens.shape[1]} tokens in "
                      f"{t:.3f} s, first stream {tokens[0, :8].tolist()} ...")
    ctx.deinit()


if __name__ == "__main__":
    main()
