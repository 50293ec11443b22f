"""Waits inside ch_chunk_attention that give up: the call ends, says so in the status word, and leaves
the device and the buffers fit for the next one.  Nothing is made to hang: the limit is set
below what an ordinary wait takes."""
import ctypes as C

import pytest
import torch

from channel_b200 import ChannelError
from channel_b200 import _lib as L
from channel_b200.paged import check_status, prompt_attention, tree_attention
from tests.chunk_util import make

pytestmark = pytest.mark.gpu


@pytest.fixture
def limit():
    """Sets after how many ns a wait gives up."""
    fn = L.load().ch_test_chunk_wait_ns
    fn.restype, fn.argtypes = C.c_uint64, [C.c_uint64]
    usual = fn(0)
    fn(usual)
    yield fn
    fn(usual)


def calls():
    """A chain of 4,096 nodes, whose rows walk their path for some ms, and many units of prompts."""
    tree = make([4096, 5], n_q=2, n_kv=1, dim=64, seed=1)
    parents = torch.cat([torch.arange(-1, 4095), torch.arange(-1, 4)]).int().cuda()
    prompts = make([16 + 37 * i % 700 for i in range(40)], [53 * i % 300 for i in range(40)], n_q=8, n_kv=4, dim=256, seed=2)
    return (lambda status: tree_attention(parents=parents, status=status, **tree)), (lambda status: prompt_attention(status=status, **prompts))


@pytest.mark.parametrize("ns", [0, 1000, 5000, 20000])
def test_a_wait_that_runs_out_ends_the_call(ns, limit):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    tree, prompts = calls()
    want = tree(status), prompts(status)
    check_status(status)
    usual = limit(ns)
    for _ in range(3):
        tree(status)
        with pytest.raises(ChannelError) as e:  # (its rows take longer than any of these limits)
            check_status(status)
        assert e.value.status == L.CH_ETIMEOUT
        prompts(status)
        torch.cuda.synchronize()
        status.zero_()
    limit(usual)
    assert torch.equal(tree(status), want[0]) and torch.equal(prompts(status), want[1])
    check_status(status)
