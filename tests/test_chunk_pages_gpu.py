"""Which pages ch_chunk_attention looks up: those that a row sees something of."""
import pytest
import torch

from channel_b200 import ChannelError
from channel_b200.paged import check_status, prompt_attention, tree_attention
from tests.chunk_util import attend64, check_close, make, random_parents

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [8, 16, 64, 128, 256])
@pytest.mark.parametrize("window", [1, 20, 57, 130, 200, 313])
@pytest.mark.parametrize("form", ["prompt", "tree"])
def test_pages_ahead_of_the_window_may_be_gone(page, window, form):
    new, old, prefix = [3, 40], [300, 129], 150
    s = make(new, old, prefix=prefix, n_q=4, n_kv=2, dim=64, page=page, seed=window)
    parents = random_parents(new, 1) if form == "tree" else None
    first = [max(0, prefix + n + 1 - window) for n in old]  # position that a stream's first token sees first
    s["prefix_table"] = s["prefix_table"].clone()
    s["prefix_table"][:min(first) // page] = -1
    for b, at in enumerate(first):
        s["table"][b, :max(0, at - prefix) // page] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def out():
        if parents is None:
            return prompt_attention(window=window, status=status, **s)
        return tree_attention(parents=parents, window=window, status=status, **s)

    ref = attend64(**s, parents=parents, window=window)
    check_close(out(), *ref)
    check_status(status)
    # the first one that is seen is reported when it is not there
    for b, at in enumerate(first):
        if at >= prefix + old[b]:
            continue
        table, col = (s["prefix_table"], at // page) if at < prefix else (s["table"][b], (at - prefix) // page)
        kept = int(table[col])
        table[col] = s["k_pool"].shape[0]
        check_close(out(), *attend64(**s, parents=parents, window=window))
        with pytest.raises(ChannelError):
            check_status(status)
        table[col] = kept


@pytest.mark.parametrize("dim,n_q", [(64, 4), (128, 4), (256, 2)])
@pytest.mark.parametrize("window", [0, 77])
def test_stale_rows_change_no_bit(dim, n_q, window):
    """What no token owns, and positions ahead of the window, hold zeros, infinities or NaN: the
    tensor cores see zeros there, in both CTAs of a pair, so that the results are the same bits."""
    new, old, prefix = [3, 40, 131, 9] * 10, [300, 129, 7, 601] * 10, 150
    outs = []
    for stale in (0.0, float("inf"), float("nan")):
        s = make(new, old, prefix=prefix, n_q=n_q, n_kv=2, dim=dim, pad=70, seed=11, stale=stale)
        first = [max(0, prefix + n + 1 - window) if window else 0 for n in old]
        for b, at in enumerate(first):
            j = torch.arange(max(0, at - prefix), device="cuda")
            for p in (s["k_pool"], s["v_pool"]):
                p[s["table"][b, j // 16].long(), j % 16] = stale
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        outs += [prompt_attention(window=window, status=status, **s)[:sum(new)] for _ in range(5)]
        check_status(status)
    assert bool(outs[0].isfinite().all()) and all(torch.equal(x, outs[0]) for x in outs)


@pytest.mark.parametrize("window", [0, 25, 60])
def test_lengths_count_without_columns(window):
    """A table without columns holds no cached token, but the new ones keep their positions."""
    s = make([10, 3], [0, 0], prefix=50, dim=64, seed=12)
    s["table"] = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    s["lens"] = torch.tensor([30, 7], dtype=torch.int32, device="cuda")
    check_close(prompt_attention(window=window, **s), *attend64(**s, window=window))
    parents = random_parents([10, 3], 12)
    check_close(tree_attention(parents=parents, window=window, **s), *attend64(**s, parents=parents, window=window))
