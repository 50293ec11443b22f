"""channel_b200.shared_prompt: what decode refuses, and its logits against a plain decoder."""
import copy
import math

import numpy as np
import pytest
import torch

from channel_b200 import _lib as L
from channel_b200.paged import plan_pages
from channel_b200.shared_prompt import DecoderShape, SharedPromptDecoder
from tests.gpu_util import rel_err


@pytest.mark.parametrize("prompt,streams,n", [([], 2, 3), ([1, 2], 0, 3), ([1, 2], 2, 0), ([1, 2], 2, -1), ([1, -1], 2, 3),
                                              ([4096], 2, 3), ([5, 1 << 40], 2, 3)])
def test_decode_refuses(prompt, streams, n):
    decoder = SharedPromptDecoder.__new__(SharedPromptDecoder)  # the checks come before any work
    decoder.shape = DecoderShape()
    with pytest.raises(L.ChannelError):
        decoder.decode(prompt, streams, n)


@pytest.fixture(scope="module")
def decoder(ctx):
    return SharedPromptDecoder(ctx, DecoderShape(), 64)


def start(streams, columns=2):
    """no tokens yet, and free pages"""
    return (torch.zeros(streams, dtype=torch.int32, device="cuda"),
            torch.full((streams, columns), -1, dtype=torch.int32, device="cuda"),
            torch.arange(20, 60, dtype=torch.int32, device="cuda"))


@pytest.mark.gpu
def test_a_step_from_another_stream(decoder):
    """tokens and plan come from work on the caller's stream that takes a while, and the logits are
    read there"""
    lens, table, free = start(5)
    ids = torch.tensor([3, 9, 27, 81, 243], device="cuda")
    big = torch.randn(8192, 8192, device="cuda")

    def one():
        late = (big @ big @ big).abs().sum().clamp(max=0).long()  # 0
        plan = plan_pages(lens, torch.ones_like(lens) + late.int(), table, free, 16, 5)
        logits = decoder.step(ids + late, plan)
        return logits.clone()
    with torch.cuda.stream(decoder.stream):
        ref = one()
    decoder.stream.synchronize()
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream()):
        decoder.k_pool.zero_(), decoder.v_pool.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            got = one()
        stream.synchronize()
        assert torch.equal(got, ref)
    assert torch.isfinite(ref).all() and int(decoder.status.item()) == 0


@pytest.mark.gpu
def test_rows_of_nan_are_not_tokens(decoder):
    """an activation that is not a number ends in an error, not in token -1"""
    with torch.cuda.stream(decoder.stream):
        row = decoder.embed[7].clone()
        decoder.embed[7] = float("nan")
    try:
        for share in (True, False):
            with pytest.raises(L.ChannelError, match="nothing to choose"):
                decoder.decode([1, 7], 3, 2, share=share)
    finally:
        with torch.cuda.stream(decoder.stream):
            decoder.embed[7] = row
    assert int(decoder.decode([1, 8], 3, 2).min()) >= 0


class PlainDecoder:
    """One stream, token by token, in 64 bits around the oracle's Q4 products; k, v and q are
    rounded to f16 where the caches and the attention hold them."""

    def __init__(self, oracle, shape, embed, seed=7):
        s, std = shape, lambda cols: 0.3 / math.sqrt(cols)
        seed_of = oracle.tensor_seed
        self.oracle, self.s, self.embed = oracle, s, embed
        d = s.head_dim
        self.shapes = dict(qkv=((s.n_q + 2 * s.n_kv) * d, s.hidden), o=(s.hidden, s.n_q * d), gate=(s.intermediate, s.hidden),
                           up=(s.intermediate, s.hidden), down=(s.hidden, s.intermediate))
        ids = dict(qkv=0, o=1, gate=2, up=3, down=4)
        self.w = [{k: oracle.gen_q4(m, n, seed_of(seed, layer, ids[k]), std(n)) for k, (m, n) in self.shapes.items()}
                  for layer in range(s.layers)]
        self.head = oracle.gen_q4(s.vocab, s.hidden, seed_of(seed, s.layers, 5), std(s.hidden))
        self.k, self.v = ([[] for _ in range(s.layers)] for _ in range(2))

    def fork(self):
        other = copy.copy(self)
        other.k, other.v = ([list(x) for x in c] for c in (self.k, self.v))
        return other

    def norm(self, x):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.s.eps)

    def rope(self, x, pos):
        half = x.shape[-1] // 2
        angle = pos * self.s.rope_theta ** (-np.arange(half) / half)
        a, b = x[..., :half], x[..., half:]
        return np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], -1)

    def product(self, layer, name, x):
        return self.oracle.gemv_q4(self.w[layer][name], x.astype(np.float32), *self.shapes[name]).astype(np.float64)

    def step(self, token):
        s, group, d, pos = self.s, self.s.n_q // self.s.n_kv, self.s.head_dim, len(self.k[0])
        x = self.embed[token].astype(np.float64) * math.sqrt(s.hidden)
        for layer in range(s.layers):
            qkv = self.product(layer, "qkv", self.norm(x)).reshape(-1, d)
            q = (2 * self.rope(self.norm(qkv[:s.n_q]), pos)).astype(np.float16).astype(np.float64)
            self.k[layer].append(self.rope(self.norm(qkv[s.n_q:s.n_q + s.n_kv]), pos).astype(np.float16).astype(np.float64))
            self.v[layer].append(qkv[s.n_q + s.n_kv:].astype(np.float16).astype(np.float64))
            k, v = np.stack(self.k[layer]), np.stack(self.v[layer])
            out = []
            for h in range(s.n_q):
                z = k[:, h // group] @ q[h] / math.sqrt(d)
                p = np.exp(z - z.max())
                out.append(p @ v[:, h // group] / p.sum())
            x = x + self.product(layer, "o", np.concatenate(out))
            n = self.norm(x).astype(np.float32)
            y = self.oracle.fused_mlp_q4(self.w[layer]["gate"], self.w[layer]["up"], n, s.intermediate, s.hidden)
            x = x + self.product(layer, "down", y)
        return self.oracle.gemv_q4(self.head, self.norm(x).astype(np.float32), s.vocab, s.hidden)


@pytest.mark.gpu
def test_steps_against_a_plain_decoder(decoder, oracle):
    """Logits of a prompt's steps and of streams behind its pages.  Weights of the attention and its
    output are rounded to f16, 2^-11 of sum p|v| each, some two times |out|: 2e-3 of the attention's
    share of each of the 3 layers' sums, below 1e-2 of the logits; a position, page, head or layer out
    of place is off by the logits' own size."""
    s, prompt, columns = decoder.shape, [(37 * i + 11) % 4096 for i in range(21)], 3
    with torch.cuda.stream(decoder.stream):
        plain = PlainDecoder(oracle, s, decoder.embed.cpu().numpy())
        lens, table, free = start(1, columns)
        for token in prompt:
            plan = plan_pages(lens, torch.ones_like(lens), table, free, 16, 1)
            free, lens = free[int(plan.counts[1]):], plan.lens
            logits = decoder.step(torch.tensor([token], device="cuda"), plan)
            assert rel_err(logits[0].cpu().numpy(), plain.step(token)) < 1e-2
        streams = [plain.fork() for _ in range(4)]
        shared = table[0, :2].contiguous()
        lens, table, _ = start(4, columns)
        for i in range(4):
            tokens = [(911 * b + 77 * i + 5) % 4096 for b in range(4)]
            plan = plan_pages(lens, torch.ones_like(lens), table, free, 16, 4, len(prompt))
            free, lens = free[int(plan.counts[1]):], plan.lens
            logits = decoder.step(torch.tensor(tokens, device="cuda"), plan, shared, len(prompt)).cpu().numpy()
            for b in range(4):
                assert rel_err(logits[b], streams[b].step(tokens[b])) < 1e-2
    assert int(decoder.status.item()) == 0
