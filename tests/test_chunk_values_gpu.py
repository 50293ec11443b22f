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
