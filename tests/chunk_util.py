"""A plain form in 64 bits of ch_chunk_attention, and the inputs of its tests."""
import math

import torch


def attend64(q, k, v, starts, parents=None, k_pool=None, v_pool=None, table=None, lens=None, prefix_table=None,
             prefix_len=0, window=0, scale=None):
    """(out, bound on what rounding may add per half step of the weights, of the scores) in
    float64; rows of no stream are NaN.  Every visible key is looked up on its own."""
    rows, n_q, dim = q.shape
    n_kv = k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    out, mass, drift = (torch.full((rows, n_q, dim), math.nan, dtype=torch.float64, device=q.device) for _ in range(3))
    starts = starts.tolist()
    page = k_pool.shape[1] if k_pool is not None else 1
    for b in range(len(starts) - 1):
        lo, hi = min(max(starts[b], 0), rows), min(max(starts[b + 1], 0), rows)
        before = prefix_len + (max(int(lens[b]), 0) if lens is not None else 0)
        ks, vs, at = [], [], []
        for pages, count, first in ((prefix_table, prefix_len, 0),
                                    (table[b] if table is not None else None, before - prefix_len, prefix_len)):
            if pages is None:
                continue
            pages = pages.tolist()
            for i in range(min(count, len(pages) * page)):
                if 0 <= pages[i // page] < k_pool.shape[0]:
                    ks.append(k_pool[pages[i // page], i % page])
                    vs.append(v_pool[pages[i // page], i % page])
                    at.append(first + i)
        old_k = torch.stack(ks).double() if ks else k[:0]
        old_v = torch.stack(vs).double() if vs else v[:0]
        at = torch.tensor(at, device=q.device, dtype=torch.long)
        for i in range(hi - lo):
            path = list(range(i + 1))
            if parents is not None:
                path, j = [], i
                while j >= 0:
                    path.append(j)
                    up = int(parents[lo + j])
                    j = up if up < j else -1
                path.reverse()
            position = before + len(path) - 1
            low = position + 1 - window if window else 0
            path = [j for d, j in enumerate(path) if before + d >= low]
            index = torch.tensor(path, device=q.device, dtype=torch.long) + lo
            old = at >= low
            kk, vv = torch.cat([old_k[old], k[index]]), torch.cat([old_v[old], v[index]])
            group = n_q // n_kv
            kk, vv = kk.repeat_interleave(group, 1), vv.repeat_interleave(group, 1)
            s = torch.einsum("hd,khd->hk", q[lo + i], kk) * scale
            p = torch.softmax(s, 1)
            out[lo + i] = torch.einsum("hk,khd->hd", p, vv)
            mass[lo + i] = torch.einsum("hk,khd->hd", p, vv.abs())
            size = torch.einsum("hd,khd->hk", q[lo + i].abs(), kk.abs()).amax(1) * abs(scale)
            drift[lo + i] = mass[lo + i] * size[:, None]
    return out, mass, drift


def tolerance(ref, mass, drift, dtype, dim):
    """|out - ref| in exact arithmetic but for: the result rounded once (half a step of it); the
    weights rounded to the type (half a step each, so of sum p |v|, and as much again where two
    differ); and scores summed in f32, at most dim roundings of 2^-24 each of sum |q k|, which a
    weight feels e-fold in the sums above and below the line; 2^-20 of sum p |v| for the f32 sums
    of up to a few thousand weights, added tile by tile."""
    half = torch.finfo(dtype).eps / 2
    return half * ref.abs() + 2 * half * mass + 2 * dim * 2.0 ** -24 * drift + 2.0 ** -20 * mass


def check_close(out, ref, mass, drift, what=""):
    there = ~torch.isnan(mass)
    off = (out.double() - ref).abs()[there]
    tol = tolerance(ref, mass, drift, out.dtype, out.shape[-1])[there]
    tiny = torch.finfo(out.dtype).smallest_normal  # results below the type's normal range keep its step
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert bool((off <= tol + tiny).all()), f"{what}: {worst:.3e} over the bound, {int((~(off <= tol + tiny)).sum())} values"


def make(new, old=None, prefix=0, n_q=4, n_kv=2, dim=64, page=16, dtype=torch.float16, pad=0, seed=0, spread=2.0, stale=None,
         spare=3):
    """Packed tensors (slices of one fused tensor), pools with pages anywhere; what no token owns
    holds `stale`."""
    g = torch.Generator("cuda").manual_seed(seed)
    total = sum(new)
    qkv = torch.randn(total + pad, n_q + 2 * n_kv, dim, generator=g, device="cuda")
    qkv[:, :n_q] *= spread
    qkv = qkv.to(dtype)
    if stale is not None:
        qkv[total:, n_q:] = stale
    starts = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    s = dict(q=qkv[:, :n_q], k=qkv[:, n_q:n_q + n_kv], v=qkv[:, n_q + n_kv:], starts=starts)
    if old is None and not prefix:
        return s
    old = old or [0] * len(new)
    shared, need = -(-prefix // page), [-(-n // page) for n in old]
    pages = shared + sum(need) + spare
    cols = max(1, max(need))
    order = torch.randperm(pages, generator=g, device="cuda").int()
    pools = [torch.randn(pages, page, n_kv, dim, generator=g, device="cuda").to(dtype) for _ in range(2)]
    table = torch.full((len(new), cols), -1, dtype=torch.int32, device="cuda")
    used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    at = shared
    for i in range(prefix):
        used[int(order[i // page]), i % page] = True
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        for i in range(old[b]):
            used[int(order[at + i // page]), i % page] = True
        at += n
    if stale is not None:
        for p in pools:
            p[~used] = stale
    s.update(k_pool=pools[0], v_pool=pools[1], table=table, lens=torch.tensor(old, dtype=torch.int32, device="cuda"))
    if prefix:
        s.update(prefix_table=order[:shared].contiguous(), prefix_len=prefix)
    return s


def random_parents(new, seed=0, back=5, roots=0.0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in new:
        for i in range(n):
            lone = i == 0 or float(torch.rand(1, generator=g)) < roots
            out.append(-1 if lone else int(torch.randint(max(0, i - back), i, (1,), generator=g)))
    return torch.tensor(out, dtype=torch.int32, device="cuda")
