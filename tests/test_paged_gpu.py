"""Page plans, page writes and shared-prefix attention (ch_page_plan, ch_paged_kv_write,
ch_prefix_attention) against plain implementations in 64 bits."""
import numpy as np
import pytest
import torch

from channel_b200 import _lib as L
from channel_b200 import paged

gpu = pytest.mark.gpu
# unit roundoff of the 16-bit types
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


# ---- page plan ----------------------------------------------------------------------


def plain_plan(lens, new, table, free, page, max_tokens, prefix):
    """the plan token by token"""
    table = table.copy()
    slots, pos, rows = (np.full(max_tokens, -1, np.int64) for _ in range(3))
    starts, taken, at, bad = [0], 0, 0, False
    for b, (n, add) in enumerate(zip(lens.tolist(), new.tolist())):
        bad |= n < 0 or add < 0
        n, add = max(n, 0), max(add, 0)
        bad |= -(-(n + add) // page) > table.shape[1]
        for col in range(-(-n // page), -(-(n + add) // page)):
            if col >= table.shape[1]:
                break
            table[b, col] = free[taken] if taken < len(free) else -1
            taken += 1
        for i in range(n, n + add):
            if at < max_tokens:
                p = table[b, i // page] if i // page < table.shape[1] else -1
                slots[at] = p * page + i % page if p >= 0 else -1
                pos[at], rows[at] = prefix + i, b
            at += 1
        starts.append(at)
    bad |= taken > len(free) or at > max_tokens
    return dict(table=table, lens=np.maximum(lens, 0) + np.maximum(new, 0), starts=np.array(starts), slots=slots,
                positions=pos, rows=rows, counts=np.array([at, taken])), bad


def run_plan(lens, new, cols, page, max_tokens, prefix, n_free, seed=0, wide=0):
    rng = np.random.default_rng(seed)
    lens, new = np.asarray(lens, np.int32), np.asarray(new, np.int32)
    table = rng.integers(0, 5000, (len(lens), cols + wide)).astype(np.int32)
    free = rng.permutation(20000)[:n_free].astype(np.int32)
    ref, bad = plain_plan(lens, new, table[:, :cols], free, page, max_tokens, prefix)
    whole = torch.from_numpy(table).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = paged.plan_pages(torch.from_numpy(lens).cuda(), torch.from_numpy(new).cuda(), whole[:, :cols],
                           torch.from_numpy(free).cuda(), page, max_tokens, prefix, status=status)
    for k, v in ref.items():
        assert np.array_equal(getattr(got, k).cpu().numpy(), v), k
    assert np.array_equal(whole[:, cols:].cpu().numpy(), table[:, cols:])
    assert bool(int(status.item()) & (1 << 5)) == bad
    return status


@gpu
@pytest.mark.parametrize("page", [1, 8, 16, 64, 256])
@pytest.mark.parametrize("n", [1, 2, 37, 64, 1000])
def test_plan(page, n):
    rng = np.random.default_rng(n + page)
    lens = rng.integers(0, 700, n)
    for new in (np.ones(n, int), np.zeros(n, int), rng.integers(0, 90, n)):
        run_plan(lens, new, 800 // page + 2, page, int(new.sum()) + int(rng.integers(0, 9)), 100, 20000 if page > 1 else
                 20000, seed=n, wide=3 if n == 37 else 0)


@gpu
def test_plan_long_prompts_and_many_streams():
    run_plan([0, 5, 0], [40001, 0, 70000], 70000 // 16 + 1, 16, 110001, 2048, 20000)
    rng = np.random.default_rng(1)
    run_plan(rng.integers(0, 30, 8192), rng.integers(0, 3, 8192), 4, 16, 20000, 0, 20000)


@gpu
def test_plan_shortages():
    run_plan([16, 3, 40], [16, 30, 1], 4, 16, 47, 0, 1)        # too few pages
    run_plan([16, 3, 40], [16, 30, 1], 4, 16, 47, 0, 0)        # none
    run_plan([16, 3, 40], [16, 90, 1], 3, 16, 107, 0, 50)      # too few columns
    run_plan([16, 3, 40], [16, 30, 1], 4, 16, 20, 0, 50)       # too few token rows
    run_plan([16, -3, 40], [16, 30, -1], 4, 16, 50, 0, 50)     # negative lengths
    run_plan([100, 3], [5, 5], 2, 16, 10, 0, 50)               # a stream that is already past its table
    st = run_plan([4, 4], [1, 1], 2, 16, 2, 0, 0)              # nothing short: no page is needed
    paged.check_status(st)
    st = run_plan([16], [1], 2, 16, 1, 0, 0)
    with pytest.raises(L.ChannelError, match="ran out"):
        paged.check_status(st)
    assert int(st.item()) == 0


@gpu
def test_plan_of_no_streams():
    run_plan([], [], 2, 16, 3, 0, 5)


# ---- page writes ----------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("src,dst", [(torch.float32, torch.float16), (torch.float32, torch.bfloat16),
                                     (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("n,nkv,dim,page", [(1, 1, 64, 8), (5, 8, 256, 16), (130, 2, 128, 32), (67, 3, 72, 1)])
def test_write(src, dst, n, nkv, dim, page):
    g = torch.Generator("cuda").manual_seed(n)
    pages = n // page + 5
    qkv = torch.randn(n, 3, nkv, dim + 8, generator=g, device="cuda").to(src)
    qkv[0, 0, 0, 0], qkv[-1, 1, 0, 1] = float("inf"), float("nan")
    k, v = qkv[:, 0, :, :dim], qkv[:, 1, :, 8:]
    # pools with a gap after every token's heads
    pool = torch.randn(2, pages, page, nkv + 1, dim, generator=g, device="cuda").to(dst)
    before = pool.clone()
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n].int()
    if n > 2:
        slots[1] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.kv_write(k, v, slots, pool[0, :, :, :nkv], pool[1, :, :, :nkv], status)
    ref = before.cpu().clone()
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            ref[0, s // page, s % page, :nkv] = k[t].cpu().double().to(dst) if src == dst else k[t].cpu().to(dst)
            ref[1, s // page, s % page, :nkv] = v[t].cpu().double().to(dst) if src == dst else v[t].cpu().to(dst)
    a, b = pool.cpu().view(torch.int16), ref.view(torch.int16)
    same = (a == b) | (pool.cpu().isnan() & ref.isnan())
    assert bool(same.all())
    assert int(status.item()) == 0


@gpu
def test_write_slot_outside_the_pool():
    k = torch.ones(3, 1, 64, dtype=torch.float16, device="cuda")
    pool = torch.zeros(2, 2, 8, 1, 64, dtype=torch.float16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.kv_write(k, k, torch.tensor([15, 16, -7], dtype=torch.int32, device="cuda"), pool[0], pool[1], status)
    assert float(pool.sum()) == 128.0 and float(pool[:, 1, 7].sum()) == 128.0
    with pytest.raises(L.ChannelError, match="outside its pool"):
        paged.check_status(status)


# ---- shared-prefix attention --------------------------------------------------------------


def plain_attention(q, k, v, prefix_table, prefix, table, lens, window, scale, page):
    """out and sum p|v| / sum p (what rounded weights can move the output by), in 64 bits"""
    n, nq, d = q.shape
    group = nq // k.shape[2]
    out, mag = torch.zeros(n, nq, d, dtype=torch.float64), torch.zeros(n, nq, d, dtype=torch.float64)
    shared = [prefix_table[i // page] * page + i % page for i in range(prefix)]
    kr, vr = k.flatten(0, 1), v.flatten(0, 1)
    for b in range(n):
        at = shared + [int(table[b][i // page]) * page + i % page for i in range(lens[b])]
        at = at[max(0, len(at) - window):] if window else at
        if not at:
            continue
        keys, values = kr[at].double(), vr[at].double()
        for h in range(nq):
            p = torch.softmax(keys[:, h // group] @ q[b, h].double() * scale, 0)
            out[b, h] = p @ values[:, h // group]
            mag[b, h] = p @ values[:, h // group].abs()
    return out, mag


def make(n, prefix, lens, nq, nkv, d, page, dtype, seed=0, spread=2.5):
    """inputs on the host; stale rows (past a prefix or a stream's end) are NaN"""
    g = torch.Generator().manual_seed(seed)
    shared = -(-prefix // page)
    need = [-(-x // page) for x in lens]
    pages = shared + sum(need) + 3
    k, v = (torch.randn(pages, page, nkv, d, generator=g).to(dtype) for _ in range(2))
    q = (spread * torch.randn(n, nq, d, generator=g)).to(dtype)
    order = torch.randperm(pages, generator=g).tolist()
    prefix_table, rest = order[:shared], order[shared:]
    table = torch.full((n, max(need + [1])), -1, dtype=torch.int32)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for i in range(prefix):
        used[prefix_table[i // page], i % page] = True
    for b in range(n):
        mine, rest = rest[:need[b]], rest[need[b]:]
        table[b, :need[b]] = torch.tensor(mine, dtype=torch.int32)
        for i in range(lens[b]):
            used[mine[i // page], i % page] = True
    k[~used] = float("nan")
    v[~used] = float("nan")
    return q, k, v, torch.tensor(prefix_table, dtype=torch.int32), table, lens


def attend(q, k, v, pt, table, lens, prefix, window=0, **kw):
    return paged.prefix_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(),
                                  torch.tensor(lens, dtype=torch.int32, device="cuda"), pt.cuda(), prefix, window, **kw)


def check(q, k, v, pt, table, lens, prefix, window=0, scale=None, **kw):
    """|out - ref| <= u |ref| (rounding of out) + (u + 2^-14) sum p|v| / sum p (weights rounded
    to the type before the product with V; scores and sums in f32, whose errors of a few
    2^-24 of sum |q k| stay far below 2^-14)"""
    page = k.shape[1]
    s = q.shape[2] ** -0.5 if scale is None else scale
    ref, mag = plain_attention(q, k, v, pt.tolist(), prefix, table, lens, window, s, page)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = attend(q, k, v, pt, table, lens, prefix, window, scale=scale, status=status, **kw)
    u = U[q.dtype]
    far = (got.cpu().double() - ref).abs() - (u * ref.abs() + (u + 2.0 ** -14) * mag)
    assert torch.isfinite(got).all()
    assert float(far.max()) <= 1e-7, f"{float(far.max()):.3g} over the bound at {int(far.argmax())}"
    assert int(status.item()) == 0
    return got


HEADS = [(4, 2, 256), (8, 1, 256), (16, 8, 256), (8, 2, 128), (6, 2, 64), (16, 1, 128), (3, 3, 64)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,nkv,d", HEADS)
def test_attention_heads(nq, nkv, d, dtype):
    lens = [0, 1, 17, 64, 130]
    check(*make(5, 201, lens, nq, nkv, d, 16, dtype), 201)


@gpu
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 127, 128, 129, 500])
def test_attention_pages(page, prefix):
    lens = [0, 1, 15, 16, 17, 255, 256, 300]
    check(*make(8, prefix, lens, 4, 2, 128, page, torch.float16, seed=page + prefix), prefix)


@gpu
@pytest.mark.parametrize("n", [1, 2, 31, 64, 65, 130])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_streams(n, dtype):
    lens = [(37 * i) % 90 for i in range(n)]
    check(*make(n, 777, lens, 4, 2, 256, 32, dtype, seed=n), 777)


@gpu
def test_attention_long():
    check(*make(3, 9000, [0, 5000, 1], 2, 1, 256, 64, torch.bfloat16), 9000)
    check(*make(2, 1, [9001, 3], 8, 1, 64, 16, torch.float16), 1)


@gpu
@pytest.mark.parametrize("window", [1, 7, 64, 100, 128, 500, 5000])
def test_attention_window(window):
    lens = [0, 1, 50, 99, 100, 101, 300, 640]
    check(*make(8, 333, lens, 4, 2, 256, 16, torch.float16, seed=window), 333, window)
    check(*make(8, 0, lens, 4, 1, 64, 16, torch.bfloat16, seed=window), 0, window)


@gpu
def test_attention_sees_nothing():
    q, k, v, pt, table, lens = make(3, 0, [0, 5, 0], 4, 2, 128, 16, torch.float16)
    out = attend(q, k, v, pt, table, lens, 0)
    assert float(out[0].abs().max()) == 0 and float(out[2].abs().max()) == 0 and float(out[1].abs().max()) > 0
    q, k, v, pt, table, lens = make(2, 0, [0, 0], 4, 2, 128, 16, torch.float16)
    assert float(attend(q, k, v, pt, table, lens, 0).abs().max()) == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_poison_outside_the_window(dtype):
    """NaN and infinities at positions that a stream's window hides do not reach it, although
    other streams see them"""
    lens, prefix, window = [0, 40, 200, 260], 300, 250
    q, k, v, pt, table, lens = make(4, prefix, lens, 4, 2, 256, 16, dtype)
    clean = attend(q, k, v, pt, table, lens, prefix, window)
    # prefix positions 60 and 70: stream 0 sees [50, 300), stream 1 [90, 340), the others less
    for i, x in ((60, float("nan")), (70, float("inf"))):
        v[pt[i // 16], i % 16] = x
        k[pt[i // 16], i % 16] = x
    got = attend(q, k, v, pt, table, lens, prefix, window)
    assert torch.isnan(got[0]).all()
    bound = 2 * U[dtype] * (clean[1:].abs().double() + 4)
    assert bool(((got[1:].double() - clean[1:].double()).abs() <= bound).all())


@gpu
def test_attention_large_scores():
    """score spreads far past what exp holds: the running maximum decides"""
    check(*make(6, 300, [0, 3, 9, 70, 130, 200], 4, 2, 128, 16, torch.float16, spread=60.0), 300)
    q, k, v, pt, table, lens = make(2, 200, [9, 60], 4, 2, 128, 16, torch.bfloat16, spread=1.0)
    check(q, k, v, pt, table, lens, 200, scale=-30.0)
    check(q, k, v, pt, table, lens, 200, scale=0.0)


@gpu
def test_attention_strides_and_out():
    """q as a slice of the fused q|k|v rows, pools as halves of one tensor, a strided out"""
    q, k, v, pt, table, lens = make(5, 100, [3, 0, 40, 77, 16], 4, 2, 128, 16, torch.float16)
    ref = attend(q, k, v, pt, table, lens, 100)
    fused = torch.randn(5, 8, 128).half().cuda()
    fused[:, 1:5] = q.cuda()
    both = torch.zeros(k.shape[0], 16, 5, 128, dtype=torch.float16, device="cuda")
    both[:, :, 0:2], both[:, :, 2:4] = k.cuda(), v.cuda()
    wide = torch.full((5, 6, 136), 7.0, dtype=torch.float16, device="cuda")
    tw = torch.full((5, 40), -1, dtype=torch.int32, device="cuda")
    tw[:, :table.shape[1]] = table.cuda()
    out = paged.prefix_attention(fused[:, 1:5], both[:, :, 0:2], both[:, :, 2:4], tw,
                                 torch.tensor(lens, dtype=torch.int32, device="cuda"), pt.cuda(), 100,
                                 out=wide[:, 1:5, :128])
    assert torch.equal(out, ref) and out.data_ptr() == wide[:, 1:5].data_ptr()
    assert float((wide[:, 0] - 7).abs().max()) == 0 and float((wide[..., 128:] - 7).abs().max()) == 0


@gpu
def test_attention_bad_pages_and_lengths():
    """a page index outside the pool leaves its positions out and is reported; a length past
    the table is cut"""
    q, k, v, pt, table, lens = make(4, 64, [40, 40, 0, 20], 4, 2, 128, 16, torch.float16)
    good = attend(q, k, v, pt, table, lens, 64)
    bad = table.clone()
    bad[0, 1], bad[1, 0] = -5, 1 << 30
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = attend(q, k, v, pt, bad, lens, 64, status=status)
    assert torch.isfinite(out).all() and torch.equal(out[2:], good[2:])
    with pytest.raises(L.ChannelError):
        paged.check_status(status)
    # what stream 0 sees without its second page, stream 1 without its first
    kr, vr = k.clone(), v.clone()
    t0 = torch.tensor([[table[0, 0], table[0, 2]]], dtype=torch.int32)
    t1 = torch.tensor([[table[1, 1], table[1, 2]]], dtype=torch.int32)
    for b, t in ((0, t0), (1, t1)):
        ref, mag = plain_attention(q[b:b + 1], kr, vr, pt.tolist(), 64, t, [24], 0, 128 ** -0.5, 16)
        u = U[torch.float16]
        assert bool(((out[b:b + 1].cpu().double() - ref).abs() <= u * ref.abs() + (u + 2.0 ** -14) * mag + 1e-7).all())
    ptb = pt.clone()
    ptb[2] = -1
    out = attend(q, k, v, ptb, table, lens, 64, status=status)
    ref, mag = plain_attention(q, k, v, pt[[0, 1, 3]].tolist(), 48, table, lens, 0, 128 ** -0.5, 16)
    assert bool(((out.cpu().double() - ref).abs() <= u * ref.abs() + (u + 2.0 ** -14) * mag + 1e-7).all())
    assert int(status.item()) & (1 << 2)
    out = attend(q, k, v, pt, table, [48, 1 << 30, -4, 20], 64)  # streams 0 and 1 end in stale rows
    assert torch.equal(out[2:], good[2:])


@gpu
def test_attention_on_another_stream_and_in_a_graph():
    q, k, v, pt, table, lens = make(6, 300, [0, 3, 9, 70, 130, 200], 4, 2, 256, 16, torch.float16)
    ref = attend(q, k, v, pt, table, lens, 300)
    args = [t.cuda() for t in (q, k, v, table)] + [torch.tensor(lens, dtype=torch.int32, device="cuda"), pt.cuda(), 300]
    out = torch.zeros_like(args[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.prefix_attention(*args, out=out)
    side.synchronize()
    assert torch.equal(out, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.prefix_attention(*args, out=out)
    for shift in (0, 1):  # the same graph with other lengths
        now = [max(0, x - shift) for x in lens]
        args[4].copy_(torch.tensor(now, dtype=torch.int32))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, attend(q, k, v, pt, table, now, 300))


@gpu
def test_attention_is_the_same_every_time():
    q, k, v, pt, table, lens = make(64, 2000, [(91 * i) % 700 for i in range(64)], 4, 2, 256, 16, torch.bfloat16)
    first = attend(q, k, v, pt, table, lens, 2000)
    for _ in range(5):
        assert torch.equal(first, attend(q, k, v, pt, table, lens, 2000))


@gpu
def test_attention_pool_past_32_bit_offsets():
    """pages whose elements lie past 2^31 in the pool"""
    pages = (1 << 31) // (64 * 8 * 256) + 8
    k = torch.empty(pages, 64, 8, 256, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    last = list(range(pages - 6, pages))
    g = torch.Generator("cuda").manual_seed(2)
    k[last] = torch.randn(6, 64, 8, 256, generator=g, device="cuda").half()
    v[last] = torch.randn(6, 64, 8, 256, generator=g, device="cuda").half()
    q = (2.5 * torch.randn(2, 16, 256, generator=g, device="cuda")).half()
    lens = [100, 30]
    pt = torch.tensor(last[:3], dtype=torch.int32)
    table = torch.tensor([last[3:5], [last[5], -1]], dtype=torch.int32)
    new = torch.randn(2, 8, 256, generator=g, device="cuda").half()
    slots = torch.tensor([last[4] * 64 + 35, last[5] * 64 + 29], dtype=torch.int32, device="cuda")
    paged.kv_write(new, new, slots, k, v)
    out = paged.prefix_attention(q, k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), pt.cuda(), 150)
    small_k, small_v = k[last].cpu(), v[last].cpu()
    assert torch.equal(small_k[4, 35], new[0].cpu())
    ref, mag = plain_attention(q.cpu(), small_k, small_v, [0, 1, 2], 150, torch.tensor([[3, 4], [5, -1]]), lens, 0, 1 / 16, 64)
    u = U[torch.float16]
    assert bool(((out.cpu().double() - ref).abs() <= u * ref.abs() + (u + 2.0 ** -14) * mag + 1e-7).all())


# ---- refusals (no GPU needed: the checks come before any CUDA call) ----------------------------


def attn_args(**kw):
    one = 4096  # never dereferenced
    base = dict(q=one, k_pool=one, v_pool=one, out=one, prefix_table=one, table=one, lens=one, q_stream_stride=512,
                q_head_stride=128, out_stream_stride=512, out_head_stride=128, page_stride=4096, token_stride=256,
                head_stride=128, table_stride=4, n_streams=2, n_q=4, n_kv=2, head_dim=128, page_size=16, n_pages=8,
                table_cols=4, prefix_len=20, window=0, scale=1.0, dtype=L.CH_F16, status=None)
    base.update(kw)
    return L.ChPrefixAttnArgs(**base)


@pytest.mark.parametrize("bad,why", [
    (dict(head_dim=96), "head_dim"), (dict(n_q=5), "n_q must"), (dict(n_q=34), "n_q must"), (dict(n_kv=0), "n_q must"),
    (dict(page_size=24), "page_size"), (dict(page_size=4), "page_size"), (dict(page_size=512), "page_size"),
    (dict(dtype=L.CH_F32), "dtype"), (dict(dtype=9), "dtype"), (dict(q=None), "NULL"), (dict(lens=None), "NULL"),
    (dict(prefix_table=None), "NULL"), (dict(table=None), "NULL"), (dict(token_stride=260), "multiples of 8"),
    (dict(q_head_stride=132), "multiples of 8"), (dict(q=4100), "aligned"), (dict(v_pool=4104), "aligned"),
    (dict(n_streams=70000), "streams"), (dict(prefix_len=1 << 31), "2^31")])
def test_attention_refuses(bad, why):
    import ctypes as C
    lib = L.load()
    a = attn_args(**bad)
    assert lib.ch_prefix_attention(C.byref(a), 4096, 1 << 40, None) == L.CH_EINVAL
    assert why in lib.ch_last_error().decode()


def test_attention_refuses_a_short_workspace():
    import ctypes as C
    lib = L.load()
    a = attn_args()
    need = lib.ch_prefix_attention_workspace(C.byref(a))
    if need:
        assert lib.ch_prefix_attention(C.byref(a), 4096, need - 1, None) == L.CH_EINVAL
        assert lib.ch_prefix_attention(C.byref(a), None, need, None) == L.CH_EINVAL
        assert lib.ch_prefix_attention(C.byref(a), 4097, need, None) == L.CH_EINVAL
    assert lib.ch_prefix_attention(None, None, 0, None) == L.CH_EINVAL
    assert lib.ch_prefix_attention_workspace(C.byref(attn_args(head_dim=100))) == 0


@pytest.mark.parametrize("bad,why", [
    (dict(page_size=12), "page_size"), (dict(page_size=0), "page_size"), (dict(n_streams=8193), "streams"),
    (dict(lens=None), "NULL"), (dict(counts=None), "NULL"), (dict(slots=None), "NULL"), (dict(table=None), "table"),
    (dict(free_pages=None), "free_pages"), (dict(table_stride=3), "table_stride"), (dict(lens_out=64), "lens_out"),
    (dict(n_free=1 << 31), "2^31")])
def test_plan_refuses(bad, why):
    import ctypes as C
    lib = L.load()
    base = dict(lens=64, new_tokens=128, free_pages=256, table=512, lens_out=1024, starts=2048, slots=4096,
                positions=8192, rows=16384, counts=32768, table_stride=4, n_streams=2, table_cols=4, n_free=5,
                page_size=16, max_tokens=8, prefix_len=0, status=None)
    base.update(bad)
    assert lib.ch_page_plan(C.byref(L.ChPagePlanArgs(**base)), None) == L.CH_EINVAL
    assert why in lib.ch_last_error().decode()
    assert lib.ch_page_plan(None, None) == L.CH_EINVAL


@pytest.mark.parametrize("bad,why", [
    (dict(head_dim=12), "head_dim"), (dict(page_size=0), "page_size"), (dict(k=None), "NULL"), (dict(slots=None), "NULL"),
    (dict(token_stride=4), "multiples of 8"), (dict(v=4100), "aligned"), (dict(src_dtype=L.CH_BF16), "CH_F32"),
    (dict(dst_dtype=L.CH_F32), "CH_F32"), (dict(n_pages=1 << 31), "2^31")])
def test_write_refuses(bad, why):
    import ctypes as C
    lib = L.load()
    base = dict(k=4096, v=4096, k_pool=4096, v_pool=4096, slots=64, k_token_stride=256, k_head_stride=128,
                v_token_stride=256, v_head_stride=128, page_stride=4096, token_stride=256, head_stride=128, n_tokens=2,
                n_kv=2, head_dim=128, page_size=16, n_pages=4, src_dtype=L.CH_F16, dst_dtype=L.CH_F16, status=None)
    base.update(bad)
    assert lib.ch_paged_kv_write(C.byref(L.ChKvWriteArgs(**base)), None) == L.CH_EINVAL
    assert why in lib.ch_last_error().decode()
    assert lib.ch_paged_kv_write(None, None) == L.CH_EINVAL


def test_wrappers_refuse():
    z, i = torch.zeros, torch.int32
    pool = z(4, 16, 2, 64, dtype=torch.float16)
    q, table, lens = z(3, 4, 64, dtype=torch.float16), z(3, 2, dtype=i), z(3, dtype=i)
    for args, kw in [((q.float(), pool, pool, table, lens), {}), ((q, pool, pool.float(), table, lens), {}),
                     ((q, pool, pool[:2], table, lens), {}), ((q, pool, pool, table.long(), lens), {}),
                     ((q, pool, pool, table[:2], lens), {}), ((q[..., :32], pool, pool, table, lens), {}),
                     ((q, pool, pool, table, lens), dict(prefix_len=3)),
                     ((q, pool, pool, table, lens), dict(prefix_table=z(1, dtype=i), prefix_len=17)),
                     ((q, pool, pool, table, lens), dict(out=q.float())),
                     ((q, pool, pool, table, lens), {})]:  # the last: tensors on the CPU
        with pytest.raises(L.ChannelError):
            paged.prefix_attention(*args, **kw)
    k = z(5, 2, 64, dtype=torch.float16)
    for args in [(k, k[:4], z(5, dtype=i), pool, pool), (k, k, z(4, dtype=i), pool, pool), (k, k, z(5), pool, pool),
                 (k[:, :1], k[:, :1], z(5, dtype=i), pool, pool), (k, k, z(5, dtype=i), pool, pool)]:
        with pytest.raises(L.ChannelError):
            paged.kv_write(*args)
    for args in [(lens, lens[:2], table, lens, 16, 4), (lens, lens, table[:2], lens, 16, 4),
                 (lens, lens, table.long(), lens, 16, 4), (lens, lens, table, lens, 16, 4)]:
        with pytest.raises(L.ChannelError):
            paged.plan_pages(*args)


def test_packed_arguments_match_the_structures():
    """the wrappers' packed records have the field offsets of the ctypes structures"""
    import ctypes as C

    from channel_b200 import sampling
    for fmt, kind in ((paged._PLAN, L.ChPagePlanArgs), (paged._WRITE, L.ChKvWriteArgs), (paged._ATTEND, L.ChPrefixAttnArgs),
                      (sampling._ROWS, L.ChSampleRowsArgs)):
        assert fmt.size == C.sizeof(kind)
        values = [float(i + 1) if t is C.c_float else i + 1 for i, (_, t) in enumerate(kind._fields_)]
        got = kind.from_buffer_copy(fmt.pack(*values))
        assert [getattr(got, n) for n, _ in kind._fields_] == values
