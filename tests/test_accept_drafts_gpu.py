"""ch_accept_drafts (sampling.accept_drafts) against a walk on the host."""
import pytest
import torch

from channel_b200 import ChannelError
from channel_b200.paged import check_status
from channel_b200.sampling import accept_drafts

pytestmark = pytest.mark.gpu


def walk(drafted, parents, starts, sampled):
    counts, after, kept, place = [], [], [-1] * len(drafted), 0
    for b in range(len(starts) - 1):
        lo = min(max(starts[b], 0), len(drafted))
        n = max(0, min(max(starts[b + 1], 0), len(drafted)) - lo)
        at, path = 0, [0] if n else []
        while n:
            want = sampled[lo + at]
            children = [j for j in range(at + 1, n) if parents[lo + j] == at and drafted[lo + j] == want and want >= 0]
            if not children:
                break
            at = children[0]
            path.append(at)
        for j in path:
            kept[lo + j] = place
            place += 1
        counts.append(len(path))
        after.append(sampled[lo + at] if n else -1)
    return counts, after, kept


def run(drafted, parents, starts, sampled, **kw):
    r = accept_drafts(*(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (drafted, parents, starts, sampled)), **kw)
    want = walk(drafted, parents, starts, sampled)
    assert r.counts.tolist() == want[0] and r.next_tokens.tolist() == want[1] and r.kept.tolist() == want[2]
    return r


def random_case(new, seed, tokens=3, back=6, pad=0):
    g = torch.Generator().manual_seed(seed)
    parents = [max(-1, int(i - torch.randint(1, back, (1,), generator=g))) for n in new for i in range(n)]
    starts = [0] + torch.tensor(new).cumsum(0).tolist()
    total = starts[-1] + pad
    draw = lambda: torch.randint(0, tokens, (total,), generator=g).tolist()  # noqa: E731
    return draw(), parents + [0] * pad, starts, draw()


@pytest.mark.parametrize("new", [[1], [0], [5], [31, 32, 33], [0, 1, 0, 200, 64, 65], [7] * 9, [300, 2]])
@pytest.mark.parametrize("tokens", [1, 2, 4])
def test_trees(new, tokens):
    for seed in range(3):
        run(*random_case(new, seed, tokens, pad=seed))


def test_many_streams():
    run(*random_case([(7 * i) % 19 for i in range(1000)], 1, 2))
    run(*random_case([1] * 8192, 2, 2))


def test_chain_accepted_whole():
    n = 500
    tokens = [(i * 7) % 11 for i in range(n)]
    r = run(tokens, list(range(-1, n - 1)), [0, n], tokens[1:] + [5])
    assert int(r.counts) == n


def test_first_of_equal_siblings():
    run([9, 4, 4, 4], [-1, 0, 0, 1], [0, 4], [4, 8, 4, 3])


def test_negative_samples_and_bad_parents():
    run([9, -1, 4], [-1, 0, 0], [0, 3], [-1, 2, 2])
    run([1, 1, 1, 1], [-1, 1, 5, 2], [0, 4], [1, 1, 1, 1])


def test_rows_of_no_stream_and_bad_starts():
    run([1] * 9, [-1, 0, 1, -1, 0, 1, 0, 1, 2], [3, 6], [1] * 9)
    for starts in ([0, 12], [0, 6, 3], [-2, 4]):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        run([1] * 9, [-1, 0, 1, -1, 0, 1, 0, 1, 2], starts, [1] * 9, status=status)
        with pytest.raises(ChannelError):
            check_status(status)
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    r = accept_drafts(i, i, i[:1].contiguous(), i)
    assert r.counts.numel() == 0 and r.kept.tolist() == [-1] * 4


def test_captured():
    case = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in random_case([20, 3, 40], 5, 2)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        accept_drafts(*case)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        r = accept_drafts(*case)
    other = random_case([20, 3, 40], 6, 2)
    for a, b in zip(case, other):
        a.copy_(torch.tensor(b, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    want = walk(*other)
    assert r.counts.tolist() == want[0] and r.next_tokens.tolist() == want[1] and r.kept.tolist() == want[2]


@pytest.mark.parametrize("n", [32, 33, 64, 65, 128, 129, 256, 257, 1023, 1024, 1025, 2049])
def test_stream_counts(n):
    run(*random_case([(5 * i) % 7 for i in range(n)], n, 2, pad=n % 3))
