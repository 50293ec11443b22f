"""Page plans, page writes and shared-prefix attention at the ends of their documented ranges."""
import ctypes

import pytest
import torch

from channel_b200 import _lib as L
from tests.test_paged_gpu import attend, attn_args, check, make

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("d", [64, 256])
def test_attention_with_a_workspace_on_16_bytes(d):
    """a workspace on any 16 bytes, of the size asked for and no more"""
    q, k, v, pt, table, lens = [t.cuda() if torch.is_tensor(t) else t for t in
                                make(5, 300, [0, 3, 70, 130, 200], 4, 2, d, 16, torch.float16)]
    n_own, ref, lib = torch.tensor(lens, dtype=torch.int32, device="cuda"), attend(q, k, v, pt, table, lens, 300), L.load()
    out = torch.zeros_like(ref)
    a = attn_args(q=q.data_ptr(), k_pool=k.data_ptr(), v_pool=v.data_ptr(), out=out.data_ptr(), prefix_table=pt.data_ptr(),
                  table=table.data_ptr(), lens=n_own.data_ptr(), q_stream_stride=4 * d, q_head_stride=d, out_stream_stride=4 * d,
                  out_head_stride=d, page_stride=32 * d, token_stride=2 * d, head_stride=d, table_stride=table.stride(0),
                  n_streams=5, head_dim=d, n_pages=k.shape[0], table_cols=table.shape[1], prefix_len=300, scale=d ** -0.5)
    need = lib.ch_prefix_attention_workspace(ctypes.byref(a))
    buf = torch.zeros(need + 1024, dtype=torch.uint8, device="cuda")
    for at in (16, 32, 240, 256, 272):
        buf.zero_()
        out.zero_()
        L.check(lib.ch_prefix_attention(ctypes.byref(a), buf.data_ptr() + at, need, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out, ref)
        assert int(buf[:at].max()) == 0 and int(buf[at + need:].max()) == 0


@gpu
@pytest.mark.parametrize("n,nq,nkv,d,prefix", [
    (17, 1024, 64, 64, 150),    # 192 pairs of kv head and 128 query rows, two for some of the SMs
    (1153, 16, 8, 256, 70),     # 152 of them
    (300, 64, 8, 128, 65),      # 152, and more streams than threads
    (4096, 2, 1, 128, 100)])    # as many streams as a call takes
def test_attention_of_more_prefix_work_than_sms(n, nq, nkv, d, prefix):
    lens = [(5 * i) % 11 for i in range(n)]
    check(*make(n, prefix, lens, nq, nkv, d, 8, torch.float16, seed=n), prefix)
