"""ch_score_rows (sampling.score_rows) against the formulas in 64 bits."""
import math

import pytest
import torch

from channel_b200 import ChannelError
from channel_b200.paged import check_status
from channel_b200.sampling import score_rows

pytestmark = pytest.mark.gpu
LOWEST = {t: torch.finfo(t).min for t in (torch.float32, torch.float16, torch.bfloat16)}


def reference(logits, targets, top, cap):
    raw = logits.double()
    raw = torch.where(raw.isnan() | (raw <= LOWEST[logits.dtype]), -math.inf, raw)
    n, vocab = raw.shape
    order = torch.sort(raw, dim=1, descending=True, stable=True).indices
    place = torch.empty_like(order).scatter_(1, order, torch.arange(vocab, device=raw.device).expand(n, -1).contiguous())
    x = torch.where(raw == -math.inf, raw, cap * torch.tanh(raw / cap)) if cap else raw
    none = (x == -math.inf).all(1, keepdim=True)
    infinite = (x == math.inf).any(1, keepdim=True)
    x = torch.where(infinite, torch.where(x == math.inf, 0.0, -math.inf), x)
    logp = torch.where(none, -math.inf, torch.log_softmax(torch.where(none, 0.0, x), 1))
    entropy = -torch.where(logp == -math.inf, 0.0, logp.exp() * logp).sum(1)
    asked = (targets >= 0) & (targets < vocab)
    at = torch.where(asked, targets, 0).long()[:, None]
    ids = order[:, :top]
    return (torch.where(asked, logp.gather(1, at)[:, 0], 0.0), torch.where(none[:, 0], 0.0, entropy),
            torch.where(asked, place.gather(1, at)[:, 0] + 1, 0), ids, logp.gather(1, ids))


def check(logits, targets, top, cap):
    r = score_rows(logits, targets, top=top, softcap=cap)
    logprobs, entropy, ranks, ids, tops = reference(logits, targets, top, cap)
    assert torch.equal(r.ranks.long(), ranks.long())
    assert torch.equal(r.top_ids.long(), ids)
    # A log-probability is (x - m) - log S rounded once: half a step, 2^-24, of the result.  x and m
    # carry tanh's error, a few steps of 2^-24, times the cap (32 at most here); S's terms have a
    # relative error of some steps (exponential, argument up to 88: 88 * 2^-24 * 2) and its log as much.
    room = 2.0 ** -24
    for got, want in ((r.logprobs, logprobs), (r.top_logprobs, tops)):
        same = torch.isinf(want) & (got.double() == want)
        off = torch.where(same, 0.0, (got.double() - torch.where(torch.isinf(want), 0.0, want)).abs())
        assert bool((off <= room * (want.abs().nan_to_num(posinf=0) + 12 * cap + 200)).all()), off.max()
    off = (r.entropy.double() - entropy).abs()
    assert bool((off <= room * (entropy.abs() + 12 * cap + 400)).all()), off.max()
    return r


def rows_of(n, vocab, dtype, seed=0, pad=0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = 2.5 * torch.randn(n, vocab + pad, generator=g, device="cuda")
    hot = torch.randint(0, vocab, (n, min(vocab, 20)), generator=g, device="cuda")
    x.scatter_add_(1, hot, 8 + 8 * torch.rand(hot.shape, generator=g, device="cuda"))
    targets = torch.where(torch.arange(n, device="cuda") % 2 == 0, hot[:, 0], torch.randint(0, vocab, (n,), generator=g, device="cuda"))
    return x.to(dtype)[:, :vocab], targets.int()


@pytest.mark.parametrize("dtype", list(LOWEST))
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 255, 256, 257, 1000, 4096, 12345])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_sizes_and_types(vocab, dtype, cap):
    for pad in (0, 1, 8):
        x, t = rows_of(5, vocab, dtype, seed=vocab + pad, pad=pad)
        check(x, t, min(20, vocab), cap)


@pytest.mark.parametrize("rows", [1, 2, 3, 20, 149, 300, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_vocabularies(rows, dtype):
    x, t = rows_of(rows, 100003 if rows > 100 else 262144, dtype, seed=rows)
    check(x, t, 20, 30.0)


@pytest.mark.parametrize("top", [0, 1, 2, 31, 32, 33, 64])
def test_counts_of_alternatives(top):
    x, t = rows_of(6, 5000, torch.float32, seed=top)
    check(x, t, top, 0.0)
    x, t = rows_of(3, 64, torch.float16, seed=top)
    check(x, t, top, 0.0)


def test_ties_go_to_the_lowest_index():
    x = torch.zeros(4, 3000, device="cuda")
    x[1, 1500:] = -0.0
    x[2, 2999], x[2, 17], x[2, 1234] = 5.0, 5.0, 5.0
    x[3] = torch.arange(3000, device="cuda") // 100
    check(x, torch.tensor([2999, 1500, 17, 50], dtype=torch.int32, device="cuda"), 64, 0.0)
    coarse = (4 * torch.randn(8, 20000, device="cuda")).round()
    check(coarse, torch.randint(0, 20000, (8,), device="cuda").int(), 64, 30.0)


@pytest.mark.parametrize("ordering", ["rising", "falling"])
def test_sorted_rows(ordering):
    x = torch.linspace(-20, 20, 50000, device="cuda").expand(3, -1).contiguous()
    check(x if ordering == "rising" else x.flip(1).contiguous(), torch.tensor([0, 49999, 777], dtype=torch.int32, device="cuda"), 33, 0.0)


@pytest.mark.parametrize("dtype", list(LOWEST))
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_masked_infinite_and_nan_logits(dtype, cap):
    x, t = rows_of(8, 700, dtype, seed=4)
    x = x.clone()
    x[0, ::2], x[1, ::3], x[2, 5:] = -math.inf, LOWEST[dtype], math.nan
    x[3], x[4], x[5] = -math.inf, LOWEST[dtype], math.nan
    x[6, 100], x[6, 300] = math.inf, math.inf
    x[7, 3] = math.inf
    t[:] = torch.tensor([0, 4, 699, 3, 3, 3, 300, 4])
    check(x, t, 10, cap)
    t[:] = torch.tensor([2, 3, 1, 699, 0, 0, 7, 3])
    check(x, t, 64, cap)


def test_one_likely_token():
    x = torch.full((2, 5000), -50.0, device="cuda")
    x[:, 3] = 60.0
    x[1, 4999] = 58.0
    check(x, torch.tensor([3, 4999], dtype=torch.int32, device="cuda"), 3, 0.0)


def test_large_and_small_logits():
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(4, 3000, generator=g, device="cuda") * torch.tensor([[1e-6], [1.0], [1e3], [1e30]], device="cuda")
    check(x, torch.zeros(4, dtype=torch.int32, device="cuda"), 5, 30.0)
    check(x[:2].contiguous(), torch.zeros(2, dtype=torch.int32, device="cuda"), 5, 0.0)
    # without a cap: one token has all the weight, and the others' log-probabilities are differences of logits
    for big in (1e6, 1e30, 3e38):
        y = torch.zeros(1, 3000, device="cuda")
        y[0, 7], y[0, 9], y[0, 11] = big, big / 2, -big / 8
        r = score_rows(y, torch.tensor([9], dtype=torch.int32, device="cuda"), top=3)
        assert r.top_ids.tolist() == [[7, 9, 0]] and r.entropy.item() == 0 and r.ranks.item() == 2
        want = torch.tensor([0.0, big / 2 - big, -big])
        assert torch.allclose(r.top_logprobs[0].cpu(), want, rtol=2.0 ** -22) and abs(r.logprobs.item() - want[1]) <= 2.0 ** -22 * big


def test_targets_outside():
    x, t = rows_of(3, 100, torch.float32)
    t[:] = torch.tensor([-1, -100, 5])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    r = score_rows(x, t, status=status)
    check_status(status)
    assert r.logprobs[:2].tolist() == [0, 0] and r.ranks[:2].tolist() == [0, 0] and r.ranks[2] > 0
    t[1] = 100
    check(x, t, 3, 0.0)
    score_rows(x, t, status=status)
    with pytest.raises(ChannelError):
        check_status(status)


def test_strided_and_broadcast_rows():
    x, t = rows_of(6, 1000, torch.float32, pad=3)
    check(x[::2], t[::2].contiguous(), 5, 0.0)
    check(x[:1].expand(6, -1), t, 5, 30.0)
    check(x[:, 1:], (t - 1).clamp(min=0), 5, 0.0)


def test_no_rows_and_grad():
    r = score_rows(torch.zeros(0, 10, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), top=3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)
    with pytest.raises(ChannelError):
        score_rows(torch.zeros(1, 10, device="cuda", requires_grad=True), torch.zeros(1, dtype=torch.int32, device="cuda"))


def test_captured_and_other_stream():
    x, t = rows_of(20, 5000, torch.bfloat16, seed=7)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        score_rows(x, t, top=7)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        r = score_rows(x, t, top=7)
    y, u = rows_of(20, 5000, torch.bfloat16, seed=8)
    x.copy_(y), t.copy_(u)
    graph.replay()
    torch.cuda.synchronize()
    want = check(y, u, 7, 0.0)
    assert all(torch.equal(a, b) for a, b in zip(r, want))
