"""Page plans, page writes and shared-prefix attention at the ends of their documented ranges."""
import ctypes
import math

import pytest
import torch

from channel_b200 import _lib as L
from channel_b200 import paged, sampling
from tests.test_paged_gpu import U, attend, attn_args, check, make

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


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,nkv,d", [(9, 1, 256), (16, 1, 256), (32, 2, 256), (22, 2, 64), (16, 1, 64), (13, 1, 128)])
def test_attention_of_many_query_heads_per_kv_head(nq, nkv, d, dtype):
    """more than 8, with and without a shared prefix, windowed, and one stream alone"""
    lens = [0, 1, 17, 64, 130, 333, 16]
    for prefix, window in ((201, 0), (0, 0), (201, 100)):
        check(*make(7, prefix, lens, nq, nkv, d, 16, dtype, seed=nq), prefix, window)
    check(*make(1, 100, [700], nq, nkv, d, 32, dtype, seed=nq), 100)

@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,nq,nkv,d,prefix,page", [
    (3, 4, 2, 64, 9001, 16), (3, 4, 2, 128, 9001, 16), (16, 64, 64, 128, 8000, 32), (16, 64, 64, 64, 7990, 64),
    (64, 16, 8, 128, 32767, 64)])
def test_attention_long_prefix_of_narrow_heads(n, nq, nkv, d, prefix, page, dtype):
    """many key tiles per unit, and a ragged last one; among them pages that are not in the pool,
    whose tiles have masks of their own"""
    lens = [(37 * i) % 50 for i in range(n)]
    args = make(n, prefix, lens, nq, nkv, d, page, dtype, seed=d + n)
    if n < 64:
        check(*args, prefix)
    q, k, v, pt, table, lens = args
    gone = torch.arange(0, len(pt) - 1, 11)  # every 11th page
    bad = pt.clone()
    bad[gone] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = attend(q, k, v, bad, table, lens, prefix, status=status)
    assert int(status.item()) == 1 << 2
    # the definition over the rest: the positions of those pages are left out
    seen = torch.ones(prefix, dtype=torch.bool)
    for i in gone.tolist():
        seen[i * page:(i + 1) * page] = False
    rows = (pt.long().repeat_interleave(page)[:prefix] * page + torch.arange(prefix) % page)[seen]
    kr, vr, u = k.flatten(0, 1).cuda(), v.flatten(0, 1).cuda(), U[dtype]
    group = nq // nkv
    for b in range(n):
        own = torch.tensor([int(table[b, i // page]) * page + i % page for i in range(lens[b])], dtype=torch.long)
        at = torch.cat([rows, own]).cuda()
        for h in range(nkv):
            p = torch.softmax(q[b, h * group:(h + 1) * group].cuda().double() @ kr[at, h].double().T * d ** -0.5, 1)
            values = vr[at, h].double()
            ref, mag = p @ values, p @ values.abs()
            far = (out[b, h * group:(h + 1) * group].double() - ref).abs() - (u * ref.abs() + (u + 2.0 ** -14) * mag)
            assert float(far.max()) <= 1e-7, (b, h)


@gpu
@pytest.mark.parametrize("window", [0, 60, 120, 300])
@pytest.mark.parametrize("d,prefix", [(128, 200), (256, 200), (64, 0)])
def test_attention_window_of_a_stream_past_its_table(d, prefix, window):
    """T counts the tokens that the table cannot hold: the window ends there, and only what the
    table holds of it is seen"""
    page, held = 16, 48
    lens = [100, 48, 1000, 49, 20, 2**31 - 1]
    q, k, v, pt, table, _ = make(6, prefix, [held] * 6, 4, 2, d, page, torch.float16, seed=window)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = attend(q, k, v, pt, table, lens, prefix, window, status=status).cpu().double()
    u, none = U[torch.float16], 0
    for b, n in enumerate(lens):
        lo, hi = max(0, prefix + n - window) if window else 0, prefix + min(n, held)
        at = [int(pt[i // page]) * page + i % page if i < prefix else
              int(table[b, (i - prefix) // page]) * page + (i - prefix) % page for i in range(lo, hi)]
        none += not at
        for h in range(4):
            p = torch.softmax(k.flatten(0, 1)[at, h // 2].double() @ q[b, h].double() * d ** -0.5, 0)
            values = v.flatten(0, 1)[at, h // 2].double()
            ref, mag = p @ values, p @ values.abs()
            assert bool(((out[b, h] - ref).abs() <= u * ref.abs() + (u + 2.0 ** -14) * mag + 1e-7).all()), (b, h)
    assert none == (2 if window else 0)
    assert int(status.item()) == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sink", [15.0, 16.0, 17.0, 17.5, 19.0])
@pytest.mark.parametrize("n,heads,d,prefix,own", [(2, 64, 64, 32768, 0), (64, 8, 128, 0, 2000), (33, 8, 256, 5000, 900)])
def test_attention_flat_keys_beside_a_large_one(n, heads, d, prefix, own, sink, dtype):
    """One key takes nearly all the weight and has V = 0, so the output is the small weights' part,
    which f16 holds only with its exponent moved.  Weights are off by u of themselves or, under
    the least normal f16 (P moved by 7 or more places, rounded to 2^-24), by 2^-32 of the largest:
    |out - ref| <= u |ref| + (u + 2^-14) sum p|v| / sum p + 2^-32 sum |v| / sum p."""
    page, u = 64, U[dtype]
    shared, mine = -(-prefix // page), -(-own // page)
    k = torch.zeros(shared + n * mine, page, heads, d, dtype=dtype, device="cuda")
    v = torch.full_like(k, 16.0)
    first = [0] if prefix else [b * mine for b in range(n)]
    k[first, 3, :, 0] = sink
    v[first, 3] = 0.0
    q = torch.zeros(n, heads, d, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    table = (shared + torch.arange(n * mine, dtype=torch.int32, device="cuda")).view(n, mine)
    pt, lens = torch.arange(shared, dtype=torch.int32, device="cuda"), torch.full((n,), own, dtype=torch.int32, device="cuda")
    out = paged.prefix_attention(q, k, v, table, lens, pt, prefix, scale=1.0).double()
    count, p = prefix + own - 1, math.exp(-sink)
    whole = 1 + count * p
    ref = 16.0 * count * p / whole
    bound = u * ref + (u + 2.0 ** -14) * ref + 2.0 ** -32 * 16 * count / whole
    assert float((out - ref).abs().max()) <= bound


def odd_strides(t):
    """t with an odd stride wherever a dimension is 1 (never used; torch may give any number there)"""
    return t.as_strided(t.shape, [2 * i + 3 if n == 1 else s for i, (n, s) in enumerate(zip(t.shape, t.stride()))])


@gpu
@pytest.mark.parametrize("n,nq,nkv,pages_of_one", [(1, 1, 1, True), (1, 4, 2, False), (3, 1, 1, False), (5, 4, 1, True)])
def test_strides_of_dimensions_of_one(n, nq, nkv, pages_of_one):
    d, page, lens = 64, 64, [7] + [0] * (n - 1)
    q, k, v, pt, table, lens = make(n, 0, lens, nq, nkv, d, page, torch.float16)
    if pages_of_one:  # a pool of one page
        k, v, table = k[table[0, :1].long()], v[table[0, :1].long()], torch.zeros_like(table)
    dev = [t.cuda() for t in (q, k, v, table)]
    own = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref = paged.prefix_attention(*dev, own)
    out = paged.prefix_attention(*map(odd_strides, dev), own, out=odd_strides(torch.zeros_like(dev[0])))
    assert torch.equal(out, ref) and float(out[0].abs().max()) > 0
    new = torch.randn(n, nkv, d, device="cuda")
    slots = torch.arange(10, 10 + n, dtype=torch.int32, device="cuda")
    for pools in (dev[1:3], [t.flatten(0, 1)[:, None] for t in dev[1:3]]):  # pages of 64, of one token
        one = [t.clone() for t in pools]
        two = [t.clone() for t in pools]
        paged.kv_write(new, new, slots, *one)
        paged.kv_write(odd_strides(new), odd_strides(new), slots, *map(odd_strides, two))
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(one, two))
        assert torch.equal(one[0].flatten(0, 1)[10:10 + n], new.half())


@gpu
def test_plan_of_a_table_of_one_column():
    lens, new = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 3, 16], [1, 1, 0]))
    table = torch.full((3, 1), 9, dtype=torch.int32, device="cuda")
    free = torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    plan = paged.plan_pages(lens, new, odd_strides(table), free, 16, 2)
    assert table[:, 0].tolist() == [5, 9, 9] and plan.slots.tolist() == [80, 147]


# ---- what the wrappers refuse, always as a ChannelError -----------------------------------------


def test_wrappers_refuse_other_dimensions():
    z, i = torch.zeros, torch.int32
    pool, k, slots = z(4, 16, 2, 64, dtype=torch.float16), z(5, 2, 64, dtype=torch.float16), z(5, dtype=i)
    for args in [(k[0], k[0], slots, pool, pool), (k, k[0], slots, pool, pool), (k[None], k[None], slots, pool, pool),
                 (k, k, slots, pool[0], pool[0]), (k, k, z((), dtype=i), pool, pool)]:
        with pytest.raises(L.ChannelError):
            paged.kv_write(*args)
    q, table, lens = z(3, 4, 64, dtype=torch.float16), z(3, 2, dtype=i), z(3, dtype=i)
    for args, kw in [((q[0], pool, pool, table, lens), {}), ((q, pool, pool, table[0], lens), {}),
                     ((q, pool, pool, table, z((), dtype=i)), {}),
                     ((q, pool, pool, table, lens), dict(prefix_table=z((), dtype=i), prefix_len=5))]:
        with pytest.raises(L.ChannelError):
            paged.prefix_attention(*args, **kw)
    for args in [(z((), dtype=i), lens, table, lens, 16, 4), (lens, lens, table, z((), dtype=i), 16, 4)]:
        with pytest.raises(L.ChannelError):
            paged.plan_pages(*args)


@gpu
def test_wrappers_refuse_sizes_that_no_field_holds():
    def z(*shape, dtype=torch.int32):
        return torch.zeros(*shape, dtype=dtype, device="cuda")
    pool, q = z(4, 16, 2, 64, dtype=torch.float16), z(3, 4, 64, dtype=torch.float16)
    table, lens = z(3, 2), z(3)
    for kw in (dict(window=1 << 32), dict(window=0.5), dict(scale=1e300)):
        with pytest.raises(L.ChannelError, match="out of range"):
            paged.prefix_attention(q, pool, pool, table, lens, **kw)
    for args in [(lens, lens, table, lens, 1 << 32, 4), (lens, lens, table, lens, 16, 4, 1 << 32),
                 (lens, lens, table, lens, 16, 1 << 40), (z(()), lens, table, lens, 16, 4), (z(()), z(()), table, lens, 16, 4),
                 (z(3, 1), z(3, 1), table, lens, 16, 4)]:
        with pytest.raises(L.ChannelError):
            paged.plan_pages(*args)
    with pytest.raises(L.ChannelError, match="out of range"):
        sampling.sample_rows(z(2, 9, dtype=torch.float32), z(2, dtype=torch.float32), softcap=1e300)


def test_wrappers_refuse_tensors_that_require_gradients():
    z, i = torch.zeros, torch.int32
    pool, k, q = (z(*s, dtype=torch.float16) for s in ((4, 16, 2, 64), (5, 2, 64), (3, 4, 64)))
    slots, table, lens = z(5, dtype=i), z(3, 2, dtype=i), z(3, dtype=i)
    x, u = z(2, 9), z(2)

    def g(t):
        return t.clone().requires_grad_()
    for call in (lambda: paged.kv_write(g(k), k, slots, pool, pool), lambda: paged.kv_write(k, g(k), slots, pool, pool),
                 lambda: paged.kv_write(k, k, slots, pool, g(pool)), lambda: sampling.sample_rows(g(x), u),
                 lambda: paged.prefix_attention(g(q), pool, pool, table, lens),
                 lambda: paged.prefix_attention(q, g(pool), pool, table, lens),
                 lambda: paged.prefix_attention(q, pool, g(pool), table, lens)):
        with pytest.raises(L.ChannelError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(L.ChannelError, match="device"):  # these are on the CPU
            call()


# ---- page plan ----------------------------------------------------------------------------------


@gpu
def test_plan_of_slots_past_31_bits():
    """a page whose tokens have no slot number below 2^31: not written, and reported"""
    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    top = (1 << 27) - 1  # the last page of 16 with slots below 2^31
    for first, new, slots, bad in (([3, top], 18, [*range(48, 64), 2**31 - 16, 2**31 - 15], False),
                                   ([top, top + 1], 18, [*range(2**31 - 16, 2**31), -1, -1], True),
                                   ([2**31 - 1, 0], 17, [-1] * 16 + [0], True)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        table = torch.full((1, 2), -1, dtype=torch.int32, device="cuda")
        plan = paged.plan_pages(ints(0), ints(new), table, ints(*first), 16, new, status=status)
        assert plan.slots.tolist() == slots and table.tolist() == [first]
        assert int(status.item()) == (1 << 5 if bad else 0)
        # the same page already in the table
        status.zero_()
        plan = paged.plan_pages(ints(16), ints(new - 16), ints(5, first[1])[None], ints(first[1]), 16, new - 16, status=status)
        assert plan.slots.tolist() == slots[16:] and int(status.item()) == (1 << 5 if slots[16] < 0 else 0)
    for prefix, bad in ((2**31 - 3, False), (2**31 - 2, True)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        plan = paged.plan_pages(ints(0), ints(3), ints(-1)[None], ints(0), 16, 3, prefix, status=status)
        assert plan.positions.tolist() == [min(prefix + i, 2**31 - 1) for i in range(3)]
        assert int(status.item()) == (1 << 5 if bad else 0)
