"""Streams that continue one prompt, end to end: page plan, page writes, attention over the
shared pages and row sampling around the Q4 projections of the op-level interface.

``SharedPromptDecoder`` holds a decoder of seeded synthetic Q4 weights in the reference's
layer order (input norm, q|k|v, per-head RoPE at the token's position, attention, o,
residual, pre-FFN norm, GELU gate * up, down, residual; src/model/forward.zig:49-230) whose
K/V caches are pages.  The prompt is decoded once, into the pages of a first stream (token by
token, or in chunks); those pages then become the shared prefix of a batch of streams, each of
which owns only the pages of its own tokens.  ``decode_drafted`` takes several tokens a step, drafted
by looking the last one up in the stream's own text; ``score`` says how likely texts are.  All work runs on the context's stream; a step called from another torch
stream is ordered after that stream's work, and what follows there after the step.

    python -m channel_b200.shared_prompt [--streams N] [--prompt N] [--tokens N] [--chunk N] [--drafts N]
"""
from __future__ import annotations

import argparse
import math
import time
from dataclasses import dataclass

import torch

from . import _lib as L
from .engine import GpuContext
from .paged import TREE_NODES, PagePlan, _fail, check_status, kv_write, plan_pages, prefix_attention, prompt_attention, tree_attention
from .sampling import RowScores, accept_drafts, sample_rows, score_rows


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
        return self._ordered(self._step, tokens, plan, prefix_table, prefix_len)

    def extend(self, tokens: torch.Tensor, plan: PagePlan, lens: torch.Tensor, prefix_table=None,
               prefix_len: int = 0) -> torch.Tensor:
        """Logits ``[tokens, vocab]`` of several tokens per stream, packed and placed by plan; lens
        is what the streams held before it (the plan's own first argument)."""
        return self._ordered(self._extend, tokens, plan, lens, prefix_table, prefix_len)

    def _ordered(self, fn, *args) -> torch.Tensor:
        """fn(*args) on the context's stream, behind the caller's and ahead of what follows there"""
        caller = torch.cuda.current_stream(self.device)
        if caller == self.stream:
            return fn(*args)
        self.stream.wait_stream(caller)
        with torch.cuda.stream(self.stream):
            logits = fn(*args)
        caller.wait_stream(self.stream)
        logits.record_stream(caller)
        return logits

    def _handed_over(self, result: torch.Tensor) -> torch.Tensor:
        """A result of the context's stream whose memory waits for what the caller queues on its own"""
        caller = torch.cuda.current_stream(self.device)
        if caller != self.stream:
            result.record_stream(caller)
        return result

    def _forward(self, tokens: torch.Tensor, positions: torch.Tensor, attend) -> torch.Tensor:
        """Logits of tokens at positions; attend(layer, q, k, v) gives a layer's attention of f16 q
        over the cache and f32 k, v."""
        s, n = self.shape, tokens.shape[0]
        x = self.embed[tokens.long()] * math.sqrt(s.hidden)
        for layer, w in enumerate(self.layers):
            qkv = self._gemm(w["qkv"], self._norm(x)).view(n, s.n_q + 2 * s.n_kv, s.head_dim)
            q = self._rope(self._norm(qkv[:, :s.n_q].contiguous()), positions)
            k = self._rope(self._norm(qkv[:, s.n_q:s.n_q + s.n_kv].contiguous()), positions)
            a = attend(layer, (2.0 * q).half(), k, qkv[:, s.n_q + s.n_kv:].contiguous())
            x = x + self._gemm(w["o"], a.float().view(n, -1))
            x = x + self._gemm(w["down"], self._gemm(w["mlp"], self._norm(x), "ch_batch_fused_mlp_q4"))
        return self._gemm(self.head, self._norm(x))

    def _step(self, tokens: torch.Tensor, plan: PagePlan, prefix_table, prefix_len: int) -> torch.Tensor:
        def attend(layer, q, k, v):
            kv_write(k, v, plan.slots, self.k_pool[layer], self.v_pool[layer], self.status)
            return prefix_attention(q, self.k_pool[layer], self.v_pool[layer], plan.table, plan.lens, prefix_table, prefix_len,
                                    status=self.status)
        return self._forward(tokens, plan.positions, attend)

    def _extend(self, tokens: torch.Tensor, plan: PagePlan, lens: torch.Tensor, prefix_table, prefix_len: int) -> torch.Tensor:
        def attend(layer, q, k, v):
            kv_write(k, v, plan.slots, self.k_pool[layer], self.v_pool[layer], self.status)
            return prompt_attention(q, k.half(), v.half(), plan.starts, self.k_pool[layer], self.v_pool[layer], plan.table, lens,
                                    prefix_table, prefix_len, status=self.status)
        return self._forward(tokens, plan.positions, attend)

    def _plan(self, lens, table, prefix_len: int, new=None, total: int = 0) -> PagePlan:
        """One token per stream, or new[b] of them, total in all."""
        if new is None:
            new, total = torch.ones_like(lens), lens.shape[0]
        plan = plan_pages(lens, new, table, self.free, self.page_size, total, prefix_len, status=self.status)
        self.free = self.free[int(plan.counts[1]):]
        return plan

    def _ids(self, name: str, tokens) -> list:
        tokens = [int(t) for t in tokens]
        if tokens and (min(tokens) < 0 or max(tokens) >= self.shape.vocab):  # an index past the table is a fault on the device
            _fail(f"{name}: token ids are 0..{self.shape.vocab - 1}")
        return tokens

    def _prompt(self, prompt: list, streams: int, chunk: int):
        """The prompt into the pages of `streams` new streams: logits of its last token, lens, the table."""
        lens = torch.zeros(streams, dtype=torch.int32, device=self.device)
        table = torch.full((streams, -(-len(prompt) // self.page_size)), -1, dtype=torch.int32, device=self.device)
        for at in range(0, len(prompt), chunk):
            part = torch.tensor(prompt[at:at + chunk], device=self.device)
            plan = self._plan(lens, table, 0, torch.full_like(lens, len(part)), streams * len(part))
            logits = self._extend(part.repeat(streams), plan, lens, None, 0)[len(part) - 1::len(part)]
            lens = plan.lens
        return logits, lens, table

    def score(self, texts, top: int = 0, chunk: int = 256) -> list:
        """How likely each text (a list of at least two token ids) is: a ``RowScores`` per text with
        a row for every token but its first.  The texts go through the decoder together, chunk tokens
        of each at a time."""
        texts = [self._ids("score", x) for x in texts]
        if not texts or min(len(x) for x in texts) < 2 or chunk < 1:
            _fail("score: a text of two tokens is wanted at least")
        with torch.cuda.stream(self.stream), torch.no_grad():
            self.free = torch.arange(self.max_pages, dtype=torch.int32, device=self.device)
            lens = torch.zeros(len(texts), dtype=torch.int32, device=self.device)
            cols = -(-max(len(x) for x in texts) // self.page_size)
            table = torch.full((len(texts), cols), -1, dtype=torch.int32, device=self.device)
            found = [[] for _ in texts]
            for at in range(0, max(len(x) for x in texts) - 1, chunk):
                parts = [x[at:min(at + chunk, len(x) - 1)] for x in texts]
                sizes = [len(x) for x in parts]
                plan = self._plan(lens, table, 0, torch.tensor(sizes, dtype=torch.int32, device=self.device), sum(sizes))
                logits = self._extend(torch.tensor(sum(parts, []), device=self.device), plan, lens, None, 0)
                after = torch.tensor(sum((x[at + 1:at + 1 + n] for x, n in zip(texts, sizes)), []), dtype=torch.int32,
                                     device=self.device)
                scores = score_rows(logits, after, top=top, softcap=30.0, status=self.status)
                for b, rows in enumerate(zip(*(x.split(sizes) for x in scores))):
                    found[b].append(rows)
                lens = plan.lens
            check_status(self.status)
            scores = [RowScores(*(torch.cat(x) for x in zip(*rows))) for rows in found]
        self.stream.synchronize()
        return [RowScores(*map(self._handed_over, x)) for x in scores]

    def decode_drafted(self, prompt, streams: int, n_tokens: int, temperature: float = 0.0, seed: int = 1, depth: int = 4,
                       branches: int = 2, chunk: int = 256, **filters) -> list:
        """As ``decode``, with several tokens a step: after a stream's newest token come, as branches
        of a tree, up to `branches` continuations of `depth` tokens that followed the same token
        earlier in its text; the tokens sampled along them are kept as far as they were drafted.
        n_tokens token ids for each stream."""
        prompt = self._ids("decode_drafted", prompt)
        if streams < 1 or n_tokens < 1 or not prompt or depth < 0 or branches < 0 or chunk < 1:
            _fail("decode_drafted: a stream, a token of the prompt and a token to decode are wanted at least")
        with torch.cuda.stream(self.stream), torch.no_grad():
            g = torch.Generator(self.device).manual_seed(seed)
            self.free = torch.arange(self.max_pages, dtype=torch.int32, device=self.device)
            logits, _, prefix_table = self._prompt(prompt, 1, chunk)
            prefix_table, prefix_len = prefix_table[0].contiguous(), len(prompt)

            def sample(rows):
                n = rows.shape[0]
                given = {k: torch.full((n,), v, device=self.device, dtype=torch.int32 if k == "top_k" else torch.float32)
                         for k, v in filters.items()}
                return sample_rows(rows, torch.rand(n, generator=g, device=self.device), softcap=30.0,
                                   temperature=torch.full((n,), temperature, device=self.device), **given)[0]

            texts = [prompt + [t] for t in sample(logits.expand(streams, -1)).tolist()]
            # a step keeps up to depth + 1 tokens more than are wanted in the end
            cols = -(-(n_tokens + depth + 1) // self.page_size)
            table = torch.full((streams, cols), -1, dtype=torch.int32, device=self.device)
            lens = torch.zeros(streams, dtype=torch.int32, device=self.device)
            end = len(prompt) + n_tokens
            while min(len(x) for x in texts) < end:
                if min(x[-1] for x in texts) < 0:
                    check_status(self.status)
                    raise L.ChannelError(L.CH_EDEVICE, "decode_drafted: a row of logits had nothing to choose from")
                trees = [self._draft(x, depth, branches) if len(x) < end else ([], [], []) for x in texts]
                tokens, parents, depths, starts = [], [], [], [0]
                for (ids, up, below), held in zip(trees, lens.tolist()):
                    tokens += ids
                    parents += up
                    depths += [prefix_len + held + d for d in below]
                    starts.append(len(tokens))
                tokens, parents, positions, starts = (torch.tensor(x, dtype=torch.int32, device=self.device)
                                                      for x in (tokens, parents, depths, starts))
                fresh = []

                def attend(layer, q, k, v):
                    fresh.append((k, v))
                    return tree_attention(q, k.half(), v.half(), starts, parents, self.k_pool[layer], self.v_pool[layer], table,
                                          lens, prefix_table, prefix_len, status=self.status)
                sampled = sample(self._forward(tokens, positions, attend))
                accepted = accept_drafts(tokens, parents, starts, sampled, status=self.status)
                # the accepted nodes' keys and values into the pages
                plan = self._plan(lens, table, prefix_len, accepted.counts, tokens.shape[0])
                slots = torch.where(accepted.kept >= 0, plan.slots[accepted.kept.clamp(min=0).long()], -1)
                for layer, (k, v) in enumerate(fresh):
                    kv_write(k, v, slots, self.k_pool[layer], self.v_pool[layer], self.status)
                lens = plan.lens
                kept, ids, after, first = (x.tolist() for x in (accepted.kept, tokens, accepted.next_tokens, starts))
                for b, text in enumerate(texts):
                    if first[b] < first[b + 1]:
                        text += [ids[t] for t in range(first[b] + 1, first[b + 1]) if kept[t] >= 0] + [after[b]]
            check_status(self.status)
            if min(min(x) for x in texts) < 0:
                raise L.ChannelError(L.CH_EDEVICE, "decode_drafted: a row of logits had nothing to choose from")
        self.stream.synchronize()
        return [x[len(prompt):end] for x in texts]

    @staticmethod
    def _draft(text: list, depth: int, branches: int):
        """Tokens, parents and depths of a tree after the text's last token, its root: what followed
        that token earlier, latest first, paths that begin alike shared; no more than a tree may have."""
        tokens, parents, depths = [text[-1]], [-1], [0]
        found = 0
        for i in range(len(text) - 2, -1, -1):
            if found == branches:
                break
            if text[i] != text[-1]:
                continue
            found += 1
            at = 0
            for token in text[i + 1:i + 1 + depth]:
                known = [j for j in range(at + 1, len(tokens)) if parents[j] == at and tokens[j] == token]
                if known:
                    at = known[0]
                    continue
                if len(tokens) == TREE_NODES:
                    return tokens, parents, depths
                tokens.append(token)
                parents.append(at)
                depths.append(depths[at] + 1)
                at = len(tokens) - 1
        return tokens, parents, depths

    def decode(self, prompt, streams: int, n_tokens: int, temperature: float = 0.0, share: bool = True, seed: int = 1,
               chunk: int = 0, **filters) -> torch.Tensor:
        """n_tokens tokens for each of `streams` continuations of one prompt (a list of token
        ids), ``[streams, n_tokens]``.  share: the prompt is decoded once and its pages are
        shared; otherwise every stream holds a copy of its own.  chunk: tokens of the prompt that
        go through the decoder at a time (0: one, as in the steps that follow)."""
        prompt = [int(t) for t in prompt]
        if streams < 1 or n_tokens < 1 or not prompt or chunk < 0:
            _fail("decode: a stream, a token of the prompt and a token to decode are wanted at least")
        self._ids("decode", prompt)
        with torch.cuda.stream(self.stream), torch.no_grad():
            g = torch.Generator(self.device).manual_seed(seed)
            self.free = torch.arange(self.max_pages, dtype=torch.int32, device=self.device)
            first = 1 if share else streams
            cols = -(-(len(prompt) + n_tokens) // self.page_size)
            lens = torch.zeros(first, dtype=torch.int32, device=self.device)
            table = torch.full((first, cols), -1, dtype=torch.int32, device=self.device)
            if chunk:
                logits, lens, pages = self._prompt(prompt, first, chunk)
                table[:, :pages.shape[1]] = pages
            else:
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
        return self._handed_over(result)


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--streams", type=int, default=32)
    p.add_argument("--prompt", type=int, default=200)
    p.add_argument("--tokens", type=int, default=32)
    p.add_argument("--chunk", type=int, default=0, help="tokens of the prompt at a time (0: one)")
    p.add_argument("--drafts", type=int, default=0, help="drafted tokens on a path (0: none)")
    a = p.parse_args()
    ctx = GpuContext.init(0)
    pages = a.streams * (-(-(a.prompt + a.tokens + a.drafts) // 16) + 2)
    d = SharedPromptDecoder(ctx, DecoderShape(), pages)
    prompt = [(37 * i + 11) % d.shape.vocab for i in range(a.prompt)]
    for timed in (False, True):  # first both once, untimed: the first calls load kernels
        for share in (True, False):
            t = time.perf_counter()
            tokens = d.decode(prompt, a.streams, a.tokens, temperature=1.0, share=share, chunk=a.chunk, top_k=64, top_p=0.95,
                              min_p=0.02)
            t = time.perf_counter() - t
            if timed:
                print(f"{'shared prompt' if share else 'own copies   '}: {a.streams} streams x {tokens.shape[1]} tokens in "
                      f"{t:.3f} s, first stream {tokens[0, :8].tolist()} ...")
        if a.drafts:
            t = time.perf_counter()
            drafted = d.decode_drafted(prompt, a.streams, a.tokens, temperature=1.0, depth=a.drafts, chunk=a.chunk or 256, top_k=64,
                                       top_p=0.95, min_p=0.02)
            t = time.perf_counter() - t
            if timed:
                print(f"drafted      : {a.streams} streams x {len(drafted[0])} tokens in {t:.3f} s, first stream {drafted[0][:8]} ...")
    ctx.deinit()


if __name__ == "__main__":
    main()
