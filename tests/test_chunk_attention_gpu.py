"""ch_chunk_attention (paged.prompt_attention, paged.tree_attention) against a plain form in 64
bits: every head layout, type and page size, lengths from none to several tiles, windows, what
lies behind the last token, streams, graphs and devices."""
import math

import pytest
import torch

from channel_b200 import ChannelError
from channel_b200.paged import check_status, prompt_attention, tree_attention
from tests.chunk_util import attend64, check_close, make, random_parents

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def both(s, parents=None, what="", **kw):
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    given = kw.setdefault("status", word)
    out = tree_attention(parents=parents, **s, **kw) if parents is not None else prompt_attention(**s, **kw)
    if given is word:
        check_status(word)
    kw.pop("out", None), kw.pop("status", None)
    check_close(out, *attend64(**s, parents=parents, **kw), what)
    return out


HEADS = [(4, 2, 256, F16), (2, 1, 256, BF16), (4, 1, 128, BF16), (3, 3, 128, F16), (6, 2, 64, F16), (5, 1, 64, BF16),
         (16, 1, 64, F16), (9, 1, 256, BF16)]


@pytest.mark.parametrize("n_q,n_kv,dim,dtype", HEADS)
def test_prompts_without_a_cache(n_q, n_kv, dim, dtype):
    both(make([1, 0, 7, 64, 130, 33], n_q=n_q, n_kv=n_kv, dim=dim, dtype=dtype, seed=1))


@pytest.mark.parametrize("n_q,n_kv,dim,dtype", HEADS)
def test_chunks_behind_caches(n_q, n_kv, dim, dtype):
    both(make([5, 1, 40, 0, 129], [0, 33, 127, 16, 250], prefix=70, n_q=n_q, n_kv=n_kv, dim=dim, dtype=dtype, page=16, seed=2))


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_page_sizes(page, dim):
    both(make([3, 20], [300, 129], prefix=131, dim=dim, page=page, seed=page), what=f"page {page}")


@pytest.mark.parametrize("new", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_lengths_around_a_tile(new):
    both(make([new], n_q=2, n_kv=1, dim=128, seed=new), what=str(new))


@pytest.mark.parametrize("old", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 256, 257, 511])
def test_cached_lengths_around_a_tile(old):
    both(make([2, 1], [old, 3], n_q=4, n_kv=2, dim=256, seed=old), what=str(old))


@pytest.mark.parametrize("window", [1, 2, 16, 60, 64, 100, 128, 129, 200, 1000])
def test_windows(window):
    both(make([150, 1, 20], [40, 300, 0], prefix=90, n_q=4, n_kv=2, dim=128, seed=window), window=window, what=str(window))


@pytest.mark.parametrize("n_q,n_kv,dim,dtype", HEADS)
def test_trees(n_q, n_kv, dim, dtype):
    new = [16, 1, 0, 61, 8]
    both(make(new, [100, 0, 5, 257, 64], prefix=33, n_q=n_q, n_kv=n_kv, dim=dim, dtype=dtype, seed=3),
         random_parents(new, 3, roots=0.1))


@pytest.mark.parametrize("new", [[300], [129, 2, 140]])
def test_trees_of_several_tiles(new):
    both(make(new, [10] * len(new), n_q=2, n_kv=1, dim=64, seed=4), random_parents(new, 4, back=3))


def test_tree_without_a_cache():
    both(make([20, 3], n_q=4, n_kv=4, dim=128, seed=5), random_parents([20, 3], 5))


@pytest.mark.parametrize("window", [1, 2, 4, 50, 130])
def test_tree_windows(window):
    new = [40, 7, 150]
    both(make(new, [60, 0, 33], prefix=20, dim=64, seed=6), random_parents(new, 6, back=2), window=window)


def test_a_chain_is_a_prompt():
    s = make([70, 5], [20, 0], dim=128, seed=7)
    parents = torch.cat([torch.arange(n) - 1 for n in (70, 5)]).int().cuda()
    ref = attend64(**s)
    check_close(tree_attention(parents=parents, **s), *ref)
    check_close(prompt_attention(**s), *ref)


def test_parents_that_are_not_earlier_nodes_are_roots():
    s = make([6], [9], dim=64, seed=8)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    odd = torch.tensor([3, 0, 2, 1, 700, -5], dtype=torch.int32, device="cuda")
    good = torch.tensor([-1, 0, -1, 1, -1, -1], dtype=torch.int32, device="cuda")
    out = tree_attention(parents=odd, status=status, **s)
    assert torch.equal(out, tree_attention(parents=good, **s))
    with pytest.raises(ChannelError):
        check_status(status)
    tree_attention(parents=good, status=status, **s)
    check_status(status)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 0.01])
def test_scales(scale):
    both(make([33, 2], [40, 1], dim=64, seed=9, spread=1.0), scale=scale)


@pytest.mark.parametrize("stale", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_what_no_token_owns_is_not_seen(stale, dim):
    new = [5, 1, 40]
    s = make(new, [30, 17, 0], prefix=21, dim=dim, pad=70, seed=10, stale=stale)
    both(s)
    both(s, torch.cat([random_parents(new, 10), torch.zeros(70, dtype=torch.int32, device="cuda")]))
    both(s, random_parents(new, 10))  # (no parents for the padding)


@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_later_tokens_and_other_branches_are_not_seen(what, value):
    """A NaN or an infinity in a key or value reaches the rows that see it, and no others."""
    s = make([100, 30], [20, 3], n_q=2, n_kv=1, dim=128, seed=11)
    s[what] = s[what].clone()
    s[what][60] = value
    out = prompt_attention(**s)
    ref = attend64(**s)
    clean = list(range(60)) + list(range(100, 130))
    check_close(out[clean], *(r[clean] for r in ref))
    if math.isnan(value):
        assert bool(out[60:100].isnan().all())
    new = [100, 30]
    parents = random_parents(new, 11)
    sees = []
    for i in range(100):
        j = i
        while j > 60:
            j = int(parents[j])
        sees.append(j == 60)
    out = tree_attention(parents=parents, **s)
    ref = attend64(**s, parents=parents)
    clean = [i for i in range(100) if not sees[i]] + list(range(100, 130))
    check_close(out[clean], *(r[clean] for r in ref))


def test_every_value_nan_ends():
    s = make([700], [64], n_q=2, n_kv=1, dim=64, seed=12)
    s["v"] = torch.full_like(s["v"], math.nan)
    assert bool(prompt_attention(**s).isnan().all())


def test_rows_of_no_stream_stay():
    s = make([5, 40], [3, 8], dim=64, pad=9, seed=13)
    out = torch.full_like(s["q"], 7.0).contiguous()
    s["starts"] = torch.tensor([2, 5, 45], dtype=torch.int32, device="cuda")
    both(s, out=out)
    assert bool((out[:2] == 7).all()) and bool((out[45:] == 7).all())


def test_starts_past_the_rows_or_falling_are_reported():
    s = make([20, 20], dim=64, seed=14)
    for starts in ([0, 30, 55], [0, 25, 10], [-4, 10, 40]):
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        both(s, status=status)
        with pytest.raises(ChannelError):
            check_status(status)


def test_bad_pages_are_left_out_and_reported():
    s = make([10, 3], [100, 40], prefix=50, dim=128, seed=15)
    s["table"][0, 2], s["table"][1, 1], s["prefix_table"][1] = -1, s["k_pool"].shape[0], -7
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    both(s, status=status)
    with pytest.raises(ChannelError):
        check_status(status)


def test_lengths_past_the_table_and_negative():
    s = make([10, 3], [100, 40], dim=64, seed=16)
    s["lens"] = torch.tensor([1000, -3], dtype=torch.int32, device="cuda")
    both(s)
    both(s, window=950)


def test_lowest_scores():
    """Scores at the far end of f32, and rows where one key has nearly all the weight."""
    s = make([40], [30], dim=64, seed=17, spread=60.0)
    both(s)


def test_strides_and_broadcast():
    s = make([30, 10], [20, 5], n_q=4, n_kv=2, dim=64, seed=18)
    wide = torch.zeros(40, 4, 128, dtype=F16, device="cuda")
    out = wide[..., :64]
    assert both(s, out=out) is out
    assert bool((wide[..., 64:] == 0).all())
    turned = dict(s, q=s["q"].transpose(0, 1).contiguous().transpose(0, 1), k=s["k"].transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(prompt_attention(**turned), prompt_attention(**s))
    one = dict(s, k=s["k"][:, :1].expand(-1, 2, -1), v=s["v"][:, :1].expand(-1, 2, -1))
    both(one)
    pools = dict(s, k_pool=s["k_pool"].transpose(1, 2).contiguous().transpose(1, 2),
                 v_pool=s["v_pool"].transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(prompt_attention(**pools), prompt_attention(**s))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_stream(dim):
    """Many tiles for a row, against the same formula in 64 bits for some rows."""
    s = make([5000, 3], [0, 0], n_q=2, n_kv=1, dim=dim, dtype=BF16, seed=19)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = prompt_attention(status=status, **s)
    check_status(status)
    q, k, v = (s[x].double() for x in "qkv")
    for i in list(range(0, 5000, 97)) + [127, 128, 2047, 4095, 4999]:
        z = torch.einsum("hd,kd->hk", q[i], k[:i + 1, 0]) * dim ** -0.5
        p = torch.softmax(z, 1)
        ref, mass = p @ v[:i + 1, 0], p @ v[:i + 1, 0].abs()
        drift = mass * (torch.einsum("hd,kd->hk", q[i].abs(), k[:i + 1, 0].abs()).amax(1, keepdim=True) * dim ** -0.5)
        check_close(out[i], ref, mass, drift, str(i))


def test_repeated_calls_give_the_same_bits():
    s = make([300, 1, 77, 40], [100, 2000, 0, 33], prefix=64, dim=128, seed=20)
    first = prompt_attention(**s)
    for _ in range(5):
        assert torch.equal(prompt_attention(**s), first)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 200])
def test_many_units_give_the_same_bits(dim, window):
    """More units than pairs of SMs, whole ones and cut ones, again and again: no wait gives up."""
    s = make([16 + 37 * i % 700 for i in range(40)], [53 * i % 300 for i in range(40)], n_q=8, n_kv=4, dim=dim, dtype=BF16, seed=21)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    first = prompt_attention(status=status, window=window, **s)
    check_status(status)
    for _ in range(30):
        assert torch.equal(prompt_attention(status=status, window=window, **s), first)
    check_status(status)
    rows = torch.arange(0, s["q"].shape[0], 61, device="cuda")
    starts = s["starts"].tolist()
    for r in rows.tolist():  # each as the last token of a shorter prompt
        b = max(i for i in range(40) if starts[i] <= r)
        one = {x: s[x][starts[b]:r + 1] for x in "qkv"}
        one.update(starts=torch.tensor([0, r + 1 - starts[b]], dtype=torch.int32, device="cuda"), k_pool=s["k_pool"],
                   v_pool=s["v_pool"], table=s["table"][b:b + 1], lens=s["lens"][b:b + 1])
        alone = prompt_attention(window=window, **one)[-1].double()
        assert (alone - first[r].double()).norm() <= 4 * torch.finfo(BF16).eps * alone.norm()


def test_another_stream_and_two_at_once():
    a, b = make([200, 9], [50, 700], dim=128, seed=21), make([64, 64, 64], dim=128, seed=22)
    want = prompt_attention(**a), prompt_attention(**b)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        got = []
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(prompt_attention(**x))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_captured_and_replayed():
    s = make([60, 3], [100, 20], prefix=40, dim=128, seed=23)
    parents = random_parents([60, 3], 23)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        prompt_attention(**s)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        a = prompt_attention(**s)
        b = tree_attention(parents=parents, **s)
    for seed in (24, 25):
        other = make([60, 3], [100, 20], prefix=40, dim=128, seed=seed)
        for x in ("q", "k", "v", "k_pool", "v_pool", "table", "prefix_table"):
            s[x].copy_(other[x])
        s["lens"].copy_(torch.tensor([70 + seed, 11], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check_close(a, *attend64(**s))
        check_close(b, *attend64(**s, parents=parents))


def test_no_streams_and_no_tokens():
    s = make([5], dim=64, seed=26)
    out = torch.full_like(s["q"], 3.0).contiguous()
    prompt_attention(**dict(s, starts=torch.zeros(1, dtype=torch.int32, device="cuda")), out=out)
    assert bool((out == 3).all())
    none = {x: s[x][:0] for x in "qkv"}
    assert prompt_attention(**none, starts=torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)


def test_requires_grad_is_refused():
    s = make([5], dim=64, seed=27)
    s["q"] = s["q"].clone().requires_grad_()
    with pytest.raises(ChannelError):
        prompt_attention(**s)
    with torch.no_grad():
        prompt_attention(**s)


def test_many_streams():
    new = [(7 * i) % 5 for i in range(300)]
    both(make(new, [(11 * i) % 40 for i in range(300)], n_q=4, n_kv=1, dim=64, seed=28))


@pytest.mark.parametrize("streams", [1, 2, 12, 13])
@pytest.mark.parametrize("n_q,n_kv,dim", [(16, 1, 64), (8, 2, 128)])
def test_runs_that_start_far_into_a_stream(streams, n_q, n_kv, dim):
    """Streams of many units, more of them than a warp has lanes: each pair finds its own first one."""
    new = [(1100, 7, 640, 0, 333)[i % 5] for i in range(streams)]
    both(make(new, [(0, 290, 31)[i % 3] for i in range(streams)], prefix=40, n_q=n_q, n_kv=n_kv, dim=dim, dtype=BF16, seed=29))
    both(make(new, n_q=n_q, n_kv=n_kv, dim=dim, dtype=BF16, seed=30), window=150)


def test_the_largest_tree_and_a_larger_one():
    s = make([4096, 5], n_q=1, n_kv=1, dim=64, seed=31)
    chain = torch.cat([torch.arange(-1, 4095), torch.arange(-1, 4)]).int().cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a, b = tree_attention(parents=chain, status=status, **s).double(), prompt_attention(**s).double()
    check_status(status)
    assert (a - b).norm() <= 4 * torch.finfo(F16).eps * b.norm()
    s = make([4097, 5], n_q=1, n_kv=1, dim=64, seed=32)
    chain = torch.cat([torch.arange(-1, 4096), torch.arange(-1, 4)]).int().cuda()
    out = torch.full_like(s["q"], 7.0)
    tree_attention(parents=chain, status=status, out=out, **s)
    with pytest.raises(ChannelError):
        check_status(status)
    b = prompt_attention(**s).double()
    assert (out[:4097] == 7.0).all() and (out[4097:].double() - b[4097:]).norm() <= 4 * torch.finfo(F16).eps * b[4097:].norm()
