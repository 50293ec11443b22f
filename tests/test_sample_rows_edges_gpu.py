"""ch_sample_rows: batches, launches and values at the ends of what it takes."""
import numpy as np
import pytest
import torch

from channel_b200 import sampling
from tests.test_sample_rows_gpu import draw, lm_logits, plain, random_settings, settings

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("n,v", [(310, 16391), (310, 32768), (160, 40001), (310, 500)])
def test_batches_of_small_clusters(n, v, dtype):
    """more rows than run at once where a row takes two CTAs, four, or one"""
    for seed, softcap in ((3, 0.0), (4, 30.0)):
        rng = np.random.default_rng(seed)
        x = lm_logits(n, v, seed, dtype)
        kw, u = random_settings(n, rng), rng.random(n).astype(np.float32)
        token, _, kept = draw(x, u, softcap, **kw)
        rt, _, rk = plain(x, torch.from_numpy(u).cuda(), softcap, **settings(n, **kw))
        assert np.array_equal(token, rt.cpu().numpy()) and np.array_equal(kept, rk.cpu().numpy())


@gpu
@pytest.mark.parametrize("n", [200, 400])
def test_clusters_without_a_row(n):
    """batches in which no row has many candidates, or every one has"""
    x = lm_logits(n, 20000, 5)
    u = np.linspace(0, 0.999, n).astype(np.float32)
    for kw in (dict(top_k=20), dict(temperature=0.0), dict(top_p=0.9)):
        full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
        full.update(kw)
        token, _, kept = draw(x, u, **full)
        rt, _, rk = plain(x, torch.from_numpy(u).cuda(), 0.0, **settings(n, **full))
        assert np.array_equal(token, rt.cpu().numpy()) and np.array_equal(kept, rk.cpu().numpy())


@gpu
def test_many_rows_in_a_graph():
    """the launches of a batch of many rows, replayed with other logits and settings that the work
    just in front of them writes"""
    n, v = 64, 262144
    rng = np.random.default_rng(9)
    kw = random_settings(n, rng)
    kw["temperature"][:] = np.where(kw["temperature"] == 0, 0, 1.0)
    s = settings(n, **kw)
    source = [lm_logits(n, v, seed) for seed in (1, 2, 3)]
    heat = [s["temperature"] * f for f in (0.7, 1.0, 1.3)]
    x, u = torch.empty_like(source[0]), torch.rand(n, device="cuda")
    x.copy_(source[0])
    sampling.sample_rows(x, u, **s)
    torch.cuda.synchronize()
    graph, new_x, new_t = torch.cuda.CUDAGraph(), source[0].clone(), heat[0].clone()
    with torch.cuda.graph(graph):
        x.copy_(new_x)
        s["temperature"].copy_(new_t)
        got = sampling.sample_rows(x, u, **s)
    for i in (0, 1, 2, 1):
        new_x.copy_(source[i])
        new_t.copy_(heat[i])
        graph.replay()
        rt, _, rk = plain(source[i], u, 0.0, **{**s, "temperature": heat[i]})
        assert torch.equal(got[0].long(), rt) and torch.equal(got[2].long(), rk)
        # and without the graph, right behind the copies
        x.copy_(source[(i + 1) % 3])
        s["temperature"].copy_(heat[i])
        now = sampling.sample_rows(x, u, **s)
        rt, _, rk = plain(source[(i + 1) % 3], u, 0.0, **{**s, "temperature": heat[i]})
        assert torch.equal(now[0].long(), rt) and torch.equal(now[2].long(), rk)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("n", [4, 400])
def test_zeros_of_either_sign_are_equal(n, softcap, dtype):
    """-0.0 at a lower index than +0.0 as a row's largest logit, greedy and with one kept"""
    v = 20000
    x = torch.full((n, v), -1.0)
    x[:, 17], x[:, 16000] = -0.0, 0.0
    x[1::2, 17], x[1::2, 16000] = 0.0, -0.0
    x[2::4, 3:9000] = -0.0
    want = np.full(n, 17)
    want[2::4] = 3
    for kw in (dict(temperature=0.0), dict(top_k=1)):
        token, _, kept = draw(x.to(dtype), 0.5, softcap, **kw)
        assert np.array_equal(token, want) and (kept == 1).all()
