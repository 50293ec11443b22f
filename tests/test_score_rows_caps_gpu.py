"""score_rows: caps over their whole range, and log-probabilities that are never above 0."""
import pytest
import torch

from channel_b200.sampling import score_rows
from tests.test_score_rows_gpu import LOWEST, check, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(LOWEST))
@pytest.mark.parametrize("cap", [1e-30, 1e-5, 9e-5, 1.1e-4, 0.5, 50.0, 9e3, 1.1e4, 1e6, 1e30])
def test_caps(cap, dtype):
    """Logits around the cap, and of an ordinary size."""
    for size in (1.0, cap):
        x, t = rows_of(7, 5000, torch.float32, seed=3)
        x = (x * size).clamp(-6e4, 6e4).to(dtype)
        r = check(x, t, 20, cap)
        assert bool((r.logprobs <= 0).all()) and bool((r.top_logprobs <= 0).all())


@pytest.mark.parametrize("dtype", list(LOWEST))
@pytest.mark.parametrize("cap", [0.0, 0.5, 30.0, 50.0, 1000.0, 2e4])
def test_one_likely_token(cap, dtype):
    """Its log-probability is 0 or the little that the others take, not more, wherever it lies."""
    g = torch.Generator("cuda").manual_seed(4)
    n = 2000
    size = cap or 30.0
    x = torch.full((n, 700), -20 * size, device="cuda")
    at = torch.randint(0, 700, (n,), generator=g, device="cuda")
    x[torch.arange(n, device="cuda"), at] = size * (0.05 + 2.5 * torch.rand(n, generator=g, device="cuda"))
    x[:, 5::7] = float("-inf")  # (blocks with something masked take another way)
    x[n // 2:, 5::7] = -20 * size
    x[torch.arange(n, device="cuda"), at] = x[torch.arange(n, device="cuda"), at].clamp(min=0.05 * size)
    r = score_rows(x.to(dtype), at.int(), top=1, softcap=cap)
    assert bool((r.ranks == 1).all()) and bool((r.logprobs <= 0).all()) and bool((r.top_logprobs <= 0).all())
    assert torch.equal(r.logprobs, r.top_logprobs[:, 0]) and bool((r.entropy >= 0).all())
