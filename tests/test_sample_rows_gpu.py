"""ch_sample_rows against a plain implementation in 64 bits, and exactly where the answer
follows from the definition (ties, uniform weights, masked rows)."""
import ctypes as C

import numpy as np
import pytest
import torch

from channel_b200 import _lib as L
from channel_b200 import sampling

gpu = pytest.mark.gpu


def settings(n, temperature=None, top_k=None, top_p=None, min_p=None):
    def row(v, kind):
        if v is None:
            return None
        return torch.as_tensor(np.broadcast_to(np.asarray(v), (n,)).copy()).to(kind).cuda()
    return dict(temperature=row(temperature, torch.float32), top_k=row(top_k, torch.int32),
                top_p=row(top_p, torch.float32), min_p=row(min_p, torch.float32))


def draw(logits, uniform, softcap=0.0, **kw):
    n = logits.shape[0]
    u = torch.as_tensor(np.broadcast_to(np.asarray(uniform, np.float32), (n,)).copy()).cuda()
    t, lp, k = sampling.sample_rows(logits.cuda() if not logits.is_cuda else logits, u, softcap=softcap, **settings(n, **kw))
    return t.cpu().numpy(), lp.cpu().numpy(), k.cpu().numpy()


# How far f32 weights can be from real ones: (x - m) / T is off by 2^-23 |x - m| / T at most
# (two roundings; |x - m| / T <= 31 where the weight is not 0), the soft cap by 3 ulp of 30
# (2^-18) over T >= 0.5, exp by 2 ulp.  Together below 2^-16; sums of weights likewise, and
# the 2^-44 rounding of 2^18 weights adds 2^-26.  Twice that is the slack.
SLACK = 2.0 ** -15


def check_row(x, token, logprob, kept, u, softcap, temperature, top_k, top_p, min_p):
    """the row's answer lies between what the definition gives with weights off by SLACK"""
    x = x.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if softcap:
        x = softcap * np.tanh(x / softcap)
    if temperature <= 0:
        assert (token, logprob, kept) == (int(np.argmax(x)), 0.0, 1)
        return
    p = np.exp((x - x.max()) / temperature)

    def kept_range(sign):
        s = 1 + sign * SLACK
        order = np.argsort(-p, kind="stable")
        down = p[order]
        count = int((down >= 2.0 ** -44 / s).sum())
        if min_p > 0:
            count = min(count, max(1, int((down >= min_p / s).sum())))
        if top_k > 0:
            count = min(count, top_k)
        if top_p < 1:
            mass = np.cumsum(down[:count])
            count = min(count, int((mass - down[:count] < top_p * s * mass[-1]).sum()))
        return count, order

    (lo, order), (hi, _) = kept_range(-1), kept_range(+1)
    assert lo <= kept <= hi, (lo, kept, hi)
    keep = np.zeros(len(p), bool)
    keep[order[:hi]] = True
    # tokens within SLACK of the last one kept may be in or out
    edge = p[order[hi - 1]]
    assert p[token] >= edge * (1 - SLACK)
    stay = np.zeros(len(p))
    stay[order[:kept]] = p[order[:kept]]
    total = stay.sum()
    below, upto = stay[:token].sum() / total, (stay[:token].sum() + p[token]) / total
    assert below - 2 * SLACK <= u <= upto + 2 * SLACK, (below, u, upto)
    assert abs(logprob - np.log(p[token] / total)) <= 4 * SLACK


def plain(logits, u, softcap, temperature, top_k, top_p, min_p):
    """the definition's integer arithmetic with torch's f32 exp and tanh, on the same device"""
    x = logits.float()
    x = torch.where(x.isnan(), -torch.inf, x)
    if softcap:
        x = torch.tanh(x / torch.full_like(x[:, :1], softcap)) * softcap
    n, v = x.shape
    top = x.amax(1, keepdim=True)
    best = (x == top).long().argmax(1)
    cold = ~(temperature > 0)
    t = torch.where(cold, 1.0, temperature)[:, None]
    e = torch.exp(torch.where(x == top, 0.0, (x - top) / t))
    w = (e * 2.0 ** 44).long()
    e, order = torch.sort(e, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    keep = (ws > 0) & ((e >= min_p[:, None]) | (e == 1))
    keep &= torch.arange(v, device=x.device) < torch.where(top_k > 0, top_k, v)[:, None]
    wk = torch.where(keep, ws, 0)
    mass = wk.cumsum(1)
    need = torch.ceil(top_p.double()[:, None] * mass[:, -1:].double()).long().clamp(min=1)
    keep &= (mass - wk < need) | (top_p >= 1)[:, None]
    run = torch.where(torch.zeros_like(keep).scatter(1, order, keep), w, 0).cumsum(1)
    total = run[:, -1]
    goal = torch.minimum((u.double() * total.double()).long(), total - 1)
    token = torch.where(cold, best, (run <= goal[:, None]).sum(1).clamp(max=v - 1))
    lp = torch.log(w.gather(1, token[:, None])[:, 0].double() / total.double())
    return token, torch.where(cold, 0.0, lp).float(), torch.where(cold, 1, keep.sum(1))


def lm_logits(n, v, seed, dtype=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    x = 2.0 * torch.randn(n, v, generator=g, device="cuda")
    top = torch.randint(0, v, (n, 40), generator=g, device="cuda")
    x.scatter_add_(1, top, 12.0 * torch.rand(n, 40, generator=g, device="cuda"))
    return x.to(dtype)


def random_settings(n, rng):
    return dict(temperature=rng.choice([0.0, 0.5, 0.8, 1.0, 1.7], n), top_k=rng.choice([0, 1, 5, 64, 1000, 5000], n),
                top_p=rng.choice([0.3, 0.9, 0.95, 0.999, 1.0], n), min_p=rng.choice([0.0, 0.0, 0.02, 0.3, 1.0], n))


@gpu
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 2, 100, 4097, 16385, 100003, 262144])
def test_against_64_bits(v, dtype, softcap):
    rng = np.random.default_rng(v)
    n = 12
    x = lm_logits(n, v, v, dtype)
    kw, u = random_settings(n, rng), rng.random(n).astype(np.float32)
    token, lp, kept = draw(x, u, softcap, **kw)
    xs = x.float().cpu().numpy()
    for r in range(n):
        check_row(xs[r], int(token[r]), float(lp[r]), int(kept[r]), float(u[r]), softcap,
                  *(np.float32(kw[k][r]).item() if k != "top_k" else int(kw[k][r]) for k in ("temperature", "top_k", "top_p", "min_p")))


@gpu
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v,pad", [(7, 0), (1000, 1), (2049, 0), (16384, 3), (40001, 2), (262144, 0), (262143, 5)])
def test_equals_the_integer_arithmetic(v, pad, dtype, softcap):
    """token for token, count for count, on rows of any alignment"""
    for seed in range(3):
        rng = np.random.default_rng(100 * seed + v)
        n = 17
        x = lm_logits(n, v + pad, seed + v, dtype)[:, :v]
        kw, u = random_settings(n, rng), rng.random(n).astype(np.float32)
        token, lp, kept = draw(x, u, softcap, **kw)
        s = settings(n, **kw)
        rt, rl, rk = plain(x, torch.from_numpy(u).cuda(), softcap, **s)
        assert np.array_equal(token, rt.cpu().numpy())
        assert np.array_equal(kept, rk.cpu().numpy())
        # log in 64 bits, rounded once
        assert np.allclose(lp, rl.cpu().numpy(), rtol=2.0 ** -22, atol=0)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,pad", [(40, 262144, 0), (67, 100003, 2), (300, 9001, 1), (600, 300, 3)])
def test_many_rows(n, v, pad, dtype):
    """batches of more rows than are taken at once, of every kind: greedy, few candidates, many,
    ties at the cuts, rows of masks, of +inf"""
    for seed, softcap in ((1, 0.0), (2, 30.0)):
        rng = np.random.default_rng(seed)
        x = lm_logits(n, v + pad, seed, dtype)[:, :v]
        x[3], x[4, 5:], x[5, v // 2] = -torch.inf, -torch.inf, torch.inf
        x[6], x[7] = 1.5, torch.finfo(dtype).min
        x[8:12] = (x[8:12] * 2).round() / 2
        kw, u = random_settings(n, rng), rng.random(n).astype(np.float32)
        for k in ("temperature", "top_k", "top_p", "min_p"):  # a setting left out, too
            given = {i: j for i, j in kw.items() if i != k}
            token, lp, kept = draw(x, u, softcap, **given)
            s = settings(n, **{**kw, k: np.full(n, dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)[k])})
            seen = torch.arange(n, device="cuda") != 3
            if softcap:
                seen &= (torch.arange(n, device="cuda") != 4) & (torch.arange(n, device="cuda") != 7)
            rt, rl, rk = plain(x[seen], torch.from_numpy(u).cuda()[seen], softcap, **{i: j[seen] for i, j in s.items()})
            at = seen.cpu().numpy()
            assert np.array_equal(token[at], rt.cpu().numpy()) and np.array_equal(kept[at], rk.cpu().numpy())
            assert token[3] == -1 and kept[3] == 0 and token[4] < 5


@gpu
def test_wide_nucleus():
    """flat rows: the kept part is most of the vocabulary, cut inside runs of near-equal weights"""
    n, v = 6, 262144
    g = torch.Generator("cuda").manual_seed(3)
    x = 0.01 * torch.randn(n, v, generator=g, device="cuda")
    kw = dict(temperature=np.full(n, 1.0), top_k=np.array([0, 0, 200000, 100000, 0, 131072]),
              top_p=np.array([0.5, 0.999, 1.0, 0.7, 1.0, 0.01]), min_p=np.zeros(n))
    u = np.linspace(0.01, 0.99, n).astype(np.float32)
    token, lp, kept = draw(x, u, **kw)
    rt, rl, rk = plain(x, torch.from_numpy(u).cuda(), 0.0, **settings(n, **kw))
    assert np.array_equal(token, rt.cpu().numpy()) and np.array_equal(kept, rk.cpu().numpy())
    assert kept[2] == 200000


@gpu
@pytest.mark.parametrize("v", [1, 33, 1000, 50000, 262144])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits(v, dtype):
    """every weight is 2^44: the draw is floor(u n), cuts keep the lowest indices"""
    x = torch.full((5, v), -3.0, dtype=dtype)
    k = max(1, v // 3)
    u = np.float32(0.7)
    token, lp, kept = draw(x, u, temperature=0.5, top_k=[0, k, 0, k, 1], top_p=[1, 1, 0.5, 0.25, 1])
    n = [v, k, int(np.ceil(np.float64(v) * 0.5)), int(np.ceil(0.25 * k)), 1]
    assert kept.tolist() == n
    assert token.tolist() == [min(int(np.float64(u) * c), c - 1) for c in n]
    assert np.allclose(lp, -np.log(n), rtol=1e-6, atol=1e-7)


@gpu
def test_masked_rows():
    """rows of -inf, the type's lowest value, NaN, +inf"""
    v = 5000
    x = torch.zeros(8, v)
    x[0] = -torch.inf
    x[1] = float("nan")
    x[2] = -torch.inf
    x[2, 77] = 1.0
    x[3] = torch.finfo(torch.float32).min
    x[3, [4, 9]] = 2.0
    x[4, 100] = torch.inf
    x[5, :4000] = float("nan")
    x[6] = torch.finfo(torch.float32).min
    x[7] = -torch.inf
    x[7, 4999] = torch.finfo(torch.float32).min
    token, lp, kept = draw(x, 0.9, temperature=1.0, top_k=50, top_p=0.9)
    assert token[0] == token[1] == -1 and kept[0] == kept[1] == 0 and np.isneginf(lp[:2]).all()
    assert (token[2], kept[2], lp[2]) == (77, 1, 0.0)
    assert (token[3], kept[3]) == (9, 2)
    assert (token[4], kept[4], lp[4]) == (100, 1, 0.0)
    assert (token[5], kept[5]) == (4000 + int(np.float32(0.9).astype(float) * 45), 45)
    assert (token[6], kept[6]) == (int(np.float32(0.9).astype(float) * 45), 45)
    assert (token[7], kept[7]) == (4999, 1)
    token, lp, kept = draw(x, 0.9, temperature=0.0)
    assert token.tolist() == [-1, -1, 77, 4, 100, 4000, 0, 4999] and kept.tolist() == [0, 0] + [1] * 6
    token, _, _ = draw(x.to(torch.float16)[2:5], 0.9, 30.0, temperature=1.0)
    assert token[0] == 77 and token[1] == 9


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v", [600, 70000])
def test_masks_stay_masked_under_the_cap(v, dtype):
    """tokens masked with -inf or the type's lowest value are not drawn, however warm; a row
    of nothing but masks of the lowest value is even"""
    x = torch.randn(64, v)
    x[:, 10:] = torch.finfo(dtype).min
    x[:, 100:] = -torch.inf
    x[1:3] = torch.finfo(dtype).min
    for kw in (dict(), dict(top_p=0.99999), dict(top_k=300), dict(min_p=1e-6), dict(top_k=1)):
        token, lp, kept = draw(x.to(dtype), (np.arange(64) + 0.5) / 64, 30.0, temperature=50.0, **kw)
        assert (token[[0, *range(3, 64)]] < 10).all() and (kept[[0, *range(3, 64)]] <= 10).all()
        if not kw:
            assert kept[1] == kept[2] == v and token[1] == int(1.5 / 64 * v)


@gpu
def test_saturated_cap_ties():
    """logits far past the cap are equal: cuts and greedy take the lowest indices"""
    x = torch.full((4, 50000), 1.0)
    x[:, 7::5000] = 400.0 + torch.arange(10.0)
    x[2] = 400.0 + torch.rand(50000)
    x[3] = 400.0 + torch.rand(50000)
    token, _, kept = draw(x, 0.999, 30.0, temperature=[0.0, 1.0, 0.0, 1.0], top_k=[0, 4, 0, 100])
    assert token.tolist() == [7, 15007, 0, 99] and kept.tolist() == [1, 4, 1, 100]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(min_p=1e-5, top_p=0.95), dict(top_k=5000, top_p=0.8)])
def test_more_rows_with_many_candidates_than_run_at_once(kw, dtype):
    n = 150
    x = lm_logits(n, 50001, 11, dtype)
    u = np.linspace(0, 0.999, n).astype(np.float32)
    full = dict(temperature=1.2, top_k=0, top_p=1.0, min_p=0.0)
    full.update(kw)
    token, _, kept = draw(x, u, **full)
    rt, _, rk = plain(x, torch.from_numpy(u).cuda(), 0.0, **settings(n, **full))
    assert np.array_equal(token, rt.cpu().numpy()) and np.array_equal(kept, rk.cpu().numpy())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("step", [0.0, 1e-6, 2e-3, 0.7])
def test_cuts_among_thousands_of_near_weights(step, dtype):
    """six values, so that thousands of tokens share a weight or differ in its last bits"""
    v, p = 100003, [0.05, 0.37, 0.8, 0.999]
    g = torch.Generator("cuda").manual_seed(3)
    x = (step * torch.randint(0, 6, (8, v), generator=g, device="cuda")).to(dtype)
    x[:, 77] += 0.5
    u = np.linspace(0, 0.99, 8).astype(np.float32)
    full = dict(temperature=0.9, top_k=[0] * 4 + [1, 3000, 50000, 99999], top_p=p + p[::-1], min_p=0.0)
    token, _, kept = draw(x, u, **full)
    rt, _, rk = plain(x, torch.from_numpy(u).cuda(), 0.0, **settings(8, **full))
    assert np.array_equal(token, rt.cpu().numpy()) and np.array_equal(kept, rk.cpu().numpy())


@gpu
@pytest.mark.parametrize("temperature", [1e-3, 0.37, 3.0, 1e4, 1e30])
@pytest.mark.parametrize("scale", [1e-4, 1.0, 1e4])
def test_scales(scale, temperature):
    """logits of any scale, temperatures from near 0 to where all weights are equal"""
    n = 9
    x = lm_logits(n, 70001, 4) * scale
    u = np.linspace(0, 0.999, n).astype(np.float32)
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=900, top_p=0.99)):
        full = dict(temperature=temperature, top_k=0, top_p=1.0, min_p=0.0)
        full.update(kw)
        token, lp, kept = draw(x, u, **full)
        rt, rl, rk = plain(x, torch.from_numpy(u).cuda(), 0.0, **settings(n, **full))
        assert np.array_equal(token, rt.cpu().numpy()) and np.array_equal(kept, rk.cpu().numpy())


@gpu
def test_greedy_takes_the_lowest_index():
    x = torch.randn(4, 262144)
    x[0, [200000, 5, 70000]] = 9.0
    x[1, 262143] = 9.0
    x[2, 0] = 9.0
    token, _, _ = draw(x, 0.5, temperature=[0.0, -1.0, 0.0, 0.0])
    assert token[:3].tolist() == [5, 262143, 0] and token[3] == int(x[3].argmax())


@gpu
def test_ends_of_the_uniform_range():
    x = torch.tensor([[0.0, -torch.inf, 1.0, 0.5, -torch.inf]]).repeat(5, 1)
    token, _, _ = draw(x, [0.0, 1 - 2.0 ** -24, 1.0, -0.5, float("nan")])
    assert token.tolist() == [0, 3, 3, 0, 0]


@gpu
def test_frequencies():
    """draws over an even grid of numbers hit each token in proportion to its weight"""
    n, v = 4096, 9
    x = torch.log(torch.arange(1.0, v + 1)).repeat(n, 1)
    token, _, kept = draw(x, (np.arange(n) + 0.5) / n, top_k=7)
    share = np.bincount(token, minlength=v) / n
    want = np.where(np.arange(v) >= 2, np.arange(1, v + 1), 0) / 42.0
    assert np.abs(share - want).max() <= 1.0 / n + 1e-6 and (kept == 7).all()


@gpu
def test_on_another_stream_and_in_a_graph():
    x = lm_logits(8, 50000, 1)
    u = torch.rand(8, device="cuda")
    ref = sampling.sample_rows(x, u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sampling.sample_rows(x, u)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sampling.sample_rows(x, u)
    u.copy_(1 - u)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, sampling.sample_rows(x, u)))


@gpu
def test_one_row_for_all():
    """logits broadcast over the rows (stride 0): as many draws from one row"""
    x = lm_logits(1, 30000, 9)
    u = torch.linspace(0, 0.999, 50, device="cuda")
    many = sampling.sample_rows(x.expand(50, -1), u)
    assert all(torch.equal(a, b) for a, b in zip(many, sampling.sample_rows(x.repeat(50, 1), u)))


@gpu
def test_no_rows():
    t, lp, k = sampling.sample_rows(torch.zeros(0, 100, device="cuda"), torch.zeros(0, device="cuda"))
    assert t.shape == lp.shape == k.shape == (0,)


@gpu
def test_row_offsets_past_32_bits():
    rows, stride = 9, 1 << 28
    buf = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda")
    x = buf.view(rows, stride)[:, :1000]
    x.copy_(lm_logits(rows, 1000, 5, torch.bfloat16))
    u = torch.rand(rows, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(sampling.sample_rows(x, u), sampling.sample_rows(x.contiguous(), u)))


# ---- refusals (no GPU needed) --------------------------------------------------------------


@pytest.mark.parametrize("bad,why", [
    (dict(vocab=0), "vocab"), (dict(vocab=262145, row_stride=300000), "vocab"),
    (dict(logits=None), "NULL"), (dict(uniform=None), "NULL"), (dict(tokens=None), "NULL"), (dict(dtype=7), "dtype"),
    (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"), (dict(softcap=float("inf")), "softcap"),
    (dict(logits=4098), "aligned"), (dict(n_rows=(1 << 20) + 1), "rows")])
def test_refuses(bad, why):
    lib = L.load()
    base = dict(logits=4096, uniform=4096, tokens=4096, row_stride=100, n_rows=2, vocab=100, softcap=0.0, dtype=L.CH_F32)
    base.update(bad)
    assert lib.ch_sample_rows(C.byref(L.ChSampleRowsArgs(**base)), None) == L.CH_EINVAL
    assert why in lib.ch_last_error().decode()
    assert lib.ch_sample_rows(None, None) == L.CH_EINVAL


def test_wrapper_refuses():
    x, u = torch.zeros(3, 50), torch.zeros(3)
    for args, kw in [((x[0], u), {}), ((x.t(), u), {}), ((x, u[:2]), {}), ((x, u.double()), {}), ((x, None), {}),
                     ((x.int(), u), {}), ((x, u), dict(temperature=torch.zeros(2))), ((x, u), dict(top_k=torch.zeros(3))),
                     ((x, u), dict(top_p=torch.zeros(3, 1))), ((x, u), {})]:  # the last: tensors on the CPU
        with pytest.raises(L.ChannelError):
            sampling.sample_rows(*args, **kw)
