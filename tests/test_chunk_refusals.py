"""What ch_chunk_attention, ch_accept_drafts and ch_score_rows refuse, without a device: the
checks come before any work."""
import ctypes as C

import pytest
import torch

from channel_b200 import ChannelError
from channel_b200 import _lib as L
from channel_b200.paged import prompt_attention, tree_attention
from channel_b200.sampling import accept_drafts, score_rows

PTR = 1 << 20


def chunk(**kw):
    a = dict(q=PTR, k=PTR, v=PTR, out=PTR, starts=PTR, k_pool=PTR, v_pool=PTR, prefix_table=PTR, table=PTR, lens=PTR,
             q_token_stride=512, q_head_stride=64, k_token_stride=512, k_head_stride=64, v_token_stride=512, v_head_stride=64,
             out_token_stride=512, out_head_stride=64, page_stride=2048, token_stride=128, head_stride=64, table_stride=4,
             n_tokens=5, n_streams=2, n_q=4, n_kv=2, head_dim=64, page_size=16, n_pages=9, table_cols=4, prefix_len=10,
             scale=1.0, dtype=L.CH_F16)
    a.update(kw)
    return L.ChChunkAttnArgs(**a)


@pytest.mark.parametrize("kw", [
    dict(head_dim=96), dict(head_dim=0), dict(n_q=5), dict(n_q=34), dict(n_kv=0), dict(n_q=0), dict(n_q=2048, n_kv=1024),
    dict(n_streams=4097), dict(n_tokens=1 << 31), dict(window=1 << 31), dict(prefix_len=1 << 31), dict(n_pages=1 << 31),
    dict(page_size=4), dict(page_size=24), dict(page_size=512), dict(table_cols=1 << 28), dict(dtype=L.CH_F32), dict(dtype=7),
    dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(starts=0), dict(k_pool=0), dict(v_pool=0), dict(table=0), dict(lens=0),
    dict(prefix_table=0), dict(q=PTR + 8), dict(out=PTR + 2), dict(v_pool=PTR + 4), dict(q_token_stride=100),
    dict(k_head_stride=68), dict(v_token_stride=4), dict(out_head_stride=2), dict(page_stride=2050), dict(token_stride=1),
    dict(head_stride=60)], ids=str)
def test_chunk_attention_arguments(kw):
    lib = L.load()
    a = chunk(**kw)
    assert lib.ch_chunk_attention(C.byref(a), PTR, 1 << 40, None) == L.CH_EINVAL
    assert lib.ch_last_error()


def test_null_records():
    lib = L.load()
    assert lib.ch_chunk_attention(None, None, 0, None) == L.CH_EINVAL
    assert lib.ch_chunk_attention_workspace(None) == 0
    assert lib.ch_accept_drafts(None, None) == L.CH_EINVAL
    assert lib.ch_score_rows(None, None) == L.CH_EINVAL


def test_nothing_to_do():
    lib = L.load()
    assert lib.ch_chunk_attention(C.byref(chunk(n_tokens=0)), None, 0, None) == L.CH_OK
    assert lib.ch_chunk_attention(C.byref(chunk(n_streams=0)), None, 0, None) == L.CH_OK
    assert lib.ch_score_rows(C.byref(L.ChScoreArgs(n_rows=0)), None) == L.CH_OK
    assert lib.ch_accept_drafts(C.byref(L.ChAcceptArgs()), None) == L.CH_OK


@pytest.mark.parametrize("kw", [dict(n_streams=8193), dict(n_tokens=1 << 31), dict(starts=0), dict(counts=0), dict(next=0),
                                dict(kept=0), dict(drafted=0), dict(parents=0), dict(sampled=0)], ids=str)
def test_accept_arguments(kw):
    a = dict(drafted=PTR, parents=PTR, starts=PTR, sampled=PTR, counts=PTR, next=PTR, kept=PTR, n_tokens=4, n_streams=2)
    a.update(kw)
    assert L.load().ch_accept_drafts(C.byref(L.ChAcceptArgs(**a)), None) == L.CH_EINVAL


@pytest.mark.parametrize("kw", [dict(vocab=0), dict(vocab=262145), dict(top=65), dict(top=11, vocab=10), dict(logits=0),
                                dict(targets=0), dict(logprobs=0), dict(entropy=0), dict(ranks=0), dict(top_ids=0),
                                dict(top_logprobs=0), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")),
                                dict(dtype=3), dict(n_rows=1 << 31)], ids=str)
def test_score_arguments(kw):
    a = dict(logits=PTR, targets=PTR, logprobs=PTR, entropy=PTR, ranks=PTR, top_ids=PTR, top_logprobs=PTR, row_stride=100,
             n_rows=2, vocab=100, top=5, softcap=0.0, dtype=L.CH_F32)
    a.update(kw)
    assert L.load().ch_score_rows(C.byref(L.ChScoreArgs(**a)), None) == L.CH_EINVAL


def tensors():
    q, k, v = torch.zeros(6, 4, 64).half(), torch.zeros(6, 2, 64).half(), torch.zeros(6, 2, 64).half()
    pool = torch.zeros(5, 16, 2, 64).half()
    return dict(q=q, k=k, v=v, starts=torch.tensor([0, 2, 6]).int(), k_pool=pool, v_pool=pool.clone(),
                table=torch.zeros(2, 3).int(), lens=torch.zeros(2).int(), prefix_table=torch.zeros(2).int(), prefix_len=20)


@pytest.mark.parametrize("kw", [
    {}, dict(k=torch.zeros(5, 2, 64).half()), dict(k=torch.zeros(6, 2, 64)), dict(v=torch.zeros(6, 1, 64).half()),
    dict(q=torch.zeros(6, 4, 32).half()), dict(q=torch.zeros(6, 4, 128).half()[..., ::2]), dict(q=torch.zeros(6, 256).half()),
    dict(starts=torch.tensor(0).int()), dict(starts=torch.zeros(0).int()), dict(starts=torch.tensor([0, 2, 6])),
    dict(k_pool=None), dict(v_pool=None), dict(k_pool=None, v_pool=None), dict(table=None), dict(lens=None),
    dict(table=torch.zeros(3, 3).int()), dict(lens=torch.zeros(3).int()), dict(prefix_table=None), dict(prefix_len=33),
    dict(prefix_len=-1), dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e39),
    dict(out=torch.zeros(6, 4, 64)), dict(out=torch.zeros(5, 4, 64).half()), dict(window=1 << 33),
    dict(k_pool=torch.zeros(5, 16, 2, 64), v_pool=torch.zeros(5, 16, 2, 64))], ids=lambda kw: ",".join(kw) or "cpu")
def test_chunk_attention_tensors(kw):
    with pytest.raises(ChannelError):
        prompt_attention(**{**tensors(), **kw})


def test_tree_tensors():
    for parents in (None, torch.zeros(7).int(), torch.zeros(6), torch.zeros(6, 1).int()):
        with pytest.raises(ChannelError):
            tree_attention(parents=parents, **tensors())


def test_score_and_accept_tensors():
    x, t = torch.zeros(3, 10), torch.zeros(3).int()
    for a in ((x[0], t), (x, t[:2]), (x, t.long()), (x.t(), torch.zeros(10).int()), (x, t, -1), (x, t, 65), (x, t, 0, float("nan")),
              (x, t)):
        with pytest.raises(ChannelError):
            score_rows(*a)
    i = torch.zeros(4).int()
    for a in ((i, i, i, i), (i, i[:3], i, i), (i, i, i[:0], i), (i.long(), i, i, i), (i, i, i, i.float())):
        with pytest.raises(ChannelError):
            accept_drafts(*a)
