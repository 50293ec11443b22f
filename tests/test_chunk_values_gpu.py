"""Values that are not finite, and scores at the end of f32's range, through ch_chunk_attention:
which rows they reach, in units that one pair computes and in cut ones."""
import math

import pytest
import torch

from channel_b200.paged import check_status, prompt_attention, tree_attention
from tests.chunk_util import attend64, check_close, make, random_parents

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def call(s, parents=None, **kw):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = tree_attention(parents=parents, status=status, **s, **kw) if parents is not None else \
        prompt_attention(status=status, **s, **kw)
    check_status(status)
    return out


@pytest.mark.parametrize("tiles", range(98, 104))
@pytest.mark.parametrize("dim", [64, 256])
def test_a_nan_ahead_of_a_tile_that_a_row_does_not_see(tiles, dim):
    """One unit of 256 rows, cut into parts of two tiles (74 pairs): the first 128 rows see
    nothing of the last tile, which lies in one part with the NaN or does not."""
    s = make([256], [tiles * 128], n_q=1, n_kv=1, dim=dim, seed=1)
    s["k"] = s["k"].clone()
    s["k"][0] = math.nan
    assert bool(call(s).isnan().all())


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_nan_beside_far_larger_scores(dim):
    """A NaN among keys whose scores lie 200 and more below those of the other parts."""
    s = make([3], [150 * 128], n_q=1, n_kv=1, dim=dim, seed=2)
    s["q"] = torch.ones_like(s["q"])
    pages = s["table"][0].long()
    level = torch.where(torch.arange(len(pages), device="cuda") < 40 * 8, -400.0, 400.0) / dim
    s["k_pool"][pages] = level[:, None, None, None].to(F16)
    assert bool(call(s, scale=1.0).isfinite().all())
    s["k_pool"][pages[1], 5] = math.nan  # (with tiles of finite scores behind it in its part)
    assert bool(call(s, scale=1.0).isnan().all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scale", [1e38, 2.3e38, 2.4e38, 3.4e38])
def test_scales_near_the_end_of_f32(scale, dtype):
    """Scores of -2^-10 scale, 0 and -2^-8 scale: the largest has all the weight."""
    s = make([3], n_q=1, n_kv=1, dim=64, dtype=dtype, seed=3)
    s["q"] = torch.zeros_like(s["q"])
    s["k"] = torch.zeros_like(s["k"])
    s["q"][..., 0] = 2.0 ** -5
    s["k"][:, 0, 0] = torch.tensor([-2.0 ** -5, 0.0, -2.0 ** -3])
    out = call(s, scale=scale)
    assert torch.equal(out, s["v"][[0, 1, 1]])


def check_values(out, ref, mass, drift, what=""):
    """As check_close where the result is finite; the same infinity, or NaN, elsewhere."""
    rows = ref.isfinite()
    got = out.double()
    same = (got == ref) | (got.isnan() & ref.isnan())
    assert bool(same[~rows].all()), f"{what}: {int((~same & ~rows).sum())} of {int((~rows).sum())} values"
    check_close(out[rows][:, None], ref[rows][:, None], mass[rows][:, None], drift[rows][:, None], what)


def poison(s, where, at, value, dim=3):
    """value in one dim of the value of a new token, or of a cached one of stream 0."""
    s = dict(s)
    if where == "new":
        s["v"] = s["v"].clone()
        s["v"][at, 0, dim] = value
    else:
        page = s["k_pool"].shape[1]
        s["v_pool"] = s["v_pool"].clone()
        s["v_pool"][int(s["table"][0, at // page]), at % page, 0, dim] = value
    return s


VALUES = [math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("where,at", [("new", 0), ("new", 60), ("new", 129), ("old", 0), ("old", 140)])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (256, F16)])
def test_values_reach_the_rows_that_see_them(value, where, at, dim, dtype):
    s = poison(make([150, 30], [200, 3], n_q=4, n_kv=2, dim=dim, dtype=dtype, seed=4), where, at, value)
    check_values(call(s), *attend64(**s))
    check_values(call(s, window=100), *attend64(**s, window=100), "window")
    parents = random_parents([150, 30], 4)
    check_values(call(s, parents), *attend64(**s, parents=parents), "tree")


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("dim", [64, 256])
def test_values_in_units_that_are_not_cut(value, dim):
    """More units than pairs: a pair's run holds whole ones, of several streams and heads."""
    new = [(23 * i) % 40 for i in range(150)]
    s = make(new, [(7 * i) % 60 for i in range(150)], n_q=8, n_kv=4, dim=dim, seed=5)
    s["v"] = s["v"].clone()
    for at in (0, 700, 1500, 1501, 2222):
        s["v"][at, at % 4, 5] = value
    check_values(call(s), *attend64(**s))
    parents = random_parents(new, 5)
    check_values(call(s, parents), *attend64(**s, parents=parents), "tree")


def test_infinities_of_both_signs():
    s = make([120], [40], n_q=2, n_kv=1, dim=128, seed=6)
    s = poison(poison(s, "new", 30, math.inf), "new", 50, -math.inf)
    out = call(s)
    check_values(out, *attend64(**s))
    assert bool((out[30:50, :, 3] == math.inf).all()) and bool(out[50:, :, 3].isnan().all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("below", [10.0, 25.0, 60.0, 150.0])
def test_an_infinity_with_a_small_weight(below, dtype):
    """A key `below` under the others' scores holds an infinity: that is the result, whatever its weight."""
    s = make([70], [40], n_q=2, n_kv=1, dim=64, dtype=dtype, seed=7)
    for x in "qk":
        s[x] = torch.zeros_like(s[x])
    s["k_pool"] = torch.zeros_like(s["k_pool"])
    s["q"][..., 0] = 1.0
    s["k"][20, 0, 0] = -below
    s = poison(s, "new", 20, -math.inf)
    out = call(s, scale=1.0)
    check_values(out, *attend64(**s, scale=1.0))
    assert bool((out[20:, :, 3] == -math.inf).all())


@pytest.mark.parametrize("form", ["prompt", "tree"])
def test_infinite_scores(form):
    """A key with an infinity gives scores of +inf (NaN) and -inf (as if it were not there)."""
    s = make([100, 30], [20, 3], n_q=4, n_kv=2, dim=128, seed=8)
    parents = random_parents([100, 30], 8) if form == "tree" else None
    s["q"], s["k"] = s["q"].clone(), s["k"].clone()
    s["q"][..., 0] = torch.where(torch.arange(130, device="cuda") % 3 == 0, 1.0, -1.0)[:, None]
    s["k"][60, 0, 0] = 60000.0  # 5,300 below the others, where q is negative
    ref, mass, drift = attend64(**s, parents=parents)
    with_key = attend64(**dict(s, v=torch.where(torch.arange(130, device="cuda")[:, None, None] == 60, math.nan, s["v"])),
                        parents=parents)[0]
    up = with_key[:, :2].isnan().all(2) & (torch.arange(130, device="cuda") % 3 == 0)[:, None]  # the rows that see it, from above
    clean = attend64(**dict(s, k=torch.where(s["k"] > 1000, 0, s["k"])), parents=parents)[2]
    drift[:, :2] = clean[:, :2]
    ref[:, :2][up] = math.nan
    s["k"][60, 0, 0] = math.inf
    check_values(call(s, parents), ref, mass, drift)


@pytest.mark.parametrize("scale", [1.0, 1.3, 1.5, 1.9])
def test_scores_near_the_end_of_f32(scale):
    """2^127 scale: a number of f32, times log2(e) none."""
    s = make([40, 150], n_q=2, n_kv=1, dim=64, dtype=BF16, seed=9)
    s["q"], s["k"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"])
    s["q"][..., 0] = 2.0 ** 63
    s["k"][3, 0, 0], s["k"][60, 0, 0], s["k"][70, 0, 0] = 2.0 ** 64, 2.0 ** 63, 2.0 ** 64
    out = call(s, scale=scale)
    for rows, key in ((range(3, 40), 3), (range(60, 70), 60), (range(70, 190), 70)):
        assert torch.equal(out[list(rows)], s["v"][key].expand(len(rows), 2, 64)), key
    check_close(out[:3], *(r[:3] for r in attend64(**s, scale=scale)))


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("at", ["first", "own"])
def test_a_bad_value_behind_a_long_cache(value, at):
    """A value that is not finite at the first of 150,000 cached positions, which all rows see, or at a
    new token: the other roles of the kernel must not wait for what is looked at again."""
    g = torch.Generator("cuda").manual_seed(10)
    s = make([200], n_q=2, n_kv=1, dim=128, seed=10)
    pools = [torch.randn(1200, 128, 1, 128, generator=g, device="cuda").half() for _ in range(2)]
    prefix = torch.randperm(1200, generator=g, device="cuda").int()
    s.update(k_pool=pools[0], v_pool=pools[1], prefix_table=prefix, prefix_len=150000)
    k, v = (torch.cat([p[prefix.long()].view(-1, 128)[:150000], s[x][:, 0]]).double() for p, x in zip(pools, "kv"))
    q = s["q"].double()
    z = torch.einsum("thd,kd->thk", q, k) * 128 ** -0.5
    z.masked_fill_(torch.arange(150200, device="cuda") > 150000 + torch.arange(200, device="cuda")[:, None, None], -math.inf)
    p = torch.softmax(z, 2)
    ref, mass = p @ v, p @ v.abs()
    drift = mass * torch.einsum("thd,kd->thk", q.abs(), k.abs()).amax(2, keepdim=True) * 128 ** -0.5
    # 150,000 weights added one by one, sqrt(150,000) roundings of 2^-24 (six standard deviations): 2^-12.8
    drift += mass * 2.0 ** -12.8 / (2 * 128 * 2.0 ** -24)
    if at == "first":
        s["v_pool"][int(prefix[0]), 0, 0, 3] = value
        ref[..., 3] = value
    else:
        s = poison(s, "new", 150, value)
        ref[150:, :, 3] = value
    check_values(call(s), ref, mass, drift)


@pytest.mark.parametrize("form", ["prompt", "tree"])
@pytest.mark.parametrize("n_q,n_kv,dim", [(2, 1, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("score", [math.nan, math.inf])
@pytest.mark.parametrize("streams", [1, 90])
def test_scores_and_values_that_are_not_finite_together(form, n_q, n_kv, dim, score, streams):
    """Rows that see a score that is not finite are NaN throughout, whatever the values of other keys."""
    new = [110] * streams if streams == 1 else [41 + i % 7 for i in range(streams)]
    s = make(new, [30] * streams, n_q=n_q, n_kv=n_kv, dim=dim, seed=13)
    starts = s["starts"].tolist()
    s["k"], s["v"] = s["k"].clone(), s["v"].clone()
    s["q"] = s["q"].clone()
    s["q"][..., 1] = 0.5  # (the infinity alone decides the score)
    for at in starts[:-1:max(1, streams // 6)]:
        s["k"][at + 20, :, 1] = score
        s["v"][at + 10, :, 3] = math.inf
        s["v"][at + 20, :, 4:] = -math.inf
        s["v"][at + 35, :, :] = math.inf
    parents = random_parents(new, 13) if form == "tree" else None
    nan = dict(s, k=torch.where(s["k"].isinf(), math.nan, s["k"]))
    check_values(call(s, parents), *attend64(**nan, parents=parents))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("below", [25.0, 150.0, 600.0])
@pytest.mark.parametrize("scale", [1.0, -1.0])
def test_a_token_of_infinities_with_a_small_weight(below, scale, dtype):
    """All of a key's values are infinite, of alternating sign: so is the result."""
    s = make([70, 9], [40, 3], n_q=2, n_kv=1, dim=64, dtype=dtype, seed=14)
    for x in "qk":
        s[x] = torch.zeros_like(s[x])
    s["k_pool"] = torch.zeros_like(s["k_pool"])
    s["q"][..., 0] = 1.0
    s["k"][20, 0, 0] = -below * scale
    s["v"] = s["v"].clone()
    s["v"][20, 0, 0::2], s["v"][20, 0, 1::2] = math.inf, -math.inf
    s["v"][73, 0, :] = math.inf
    out = call(s, scale=scale)
    check_values(out, *attend64(**s, scale=scale))
    assert bool((out[20:70, :, 0::2] == math.inf).all()) and bool((out[20:70, :, 1::2] == -math.inf).all())


@pytest.mark.parametrize("dtype,most", [(F16, 65504.0), (BF16, torch.finfo(BF16).max)])
@pytest.mark.parametrize("scale", [None, -0.1])
@pytest.mark.parametrize("dim", [64, 256])
def test_values_at_the_end_of_the_type(dtype, most, scale, dim):
    """Values of the type's largest magnitude: a mean of them is no larger, neither by the rounding of
    the weights nor because a sum of weighted values leaves f32."""
    s = make([200, 31], [300, 5], n_q=4, n_kv=2, dim=dim, dtype=dtype, seed=15)
    for x in ("v", "v_pool"):
        s[x] = torch.full_like(s[x], most)
        s[x][..., 1::2] = -most
        s[x][..., 4] = 0.5
    out = call(s, scale=scale)
    ref = s["v"][:, :1].expand_as(out)
    assert bool(((out.double() - ref.double()).abs() <= 2.5 * torch.finfo(dtype).eps * ref.double().abs()).all())
    assert bool(out.isfinite().all())


def test_a_large_value_with_a_large_weight():
    """bf16 values whose sum of weights times values would leave f32, under scores that grow."""
    s = make([60], [200], n_q=2, n_kv=1, dim=128, dtype=BF16, seed=16)
    s["v"] = (s["v"].float() * 1e36).to(BF16)
    s["v_pool"] = (s["v_pool"].float() * 1e36).to(BF16)
    check_values(call(s), *attend64(**s))
    s["v"], s["v_pool"] = (x.float().clamp(-3e36, 3e36).mul(1e2).to(BF16) for x in (s["v"], s["v_pool"]))
    check_values(call(s), *attend64(**s))
