// chunk_attn.cuh -- what the kernels of ch_chunk_attention share: the arguments, which keys a
// query row sees, and one row computed on its own by a warp.
#pragma once
#include "common.cuh"
#include "kernels.cuh"
#include "tcgen05.cuh"

namespace ch {

// Nodes of a stream's tree (`most`, where there are parents).  A row walks its path anew for every
// tile of new keys, so a chain costs the square of its length; a larger tree is reported and left out.
constexpr uint32_t kMaxNodes = 4096;

struct ChunkArgs {
  const void *q, *k, *v, *k_pool, *v_pool;
  void *out;
  const int32_t *starts, *parents, *prefix_table, *table, *lens;
  long long qs, qh, ks, kh, vs, vh, os, oh;  // token and head strides
  long long page, token, head, ts;           // pool and table strides
  uint32_t n_tokens, n, nq, nkv, group, shift, n_pages, cols, prefix, window, most;
  float scale;
  uint32_t *status;
  uint64_t wait_ns;  // after which a wait inside the kernel gives up
};

// A stream's new tokens [first, first + count) of the packed rows and its cached ones: `cached` of
// them can be read (those in the table's columns), `before` positions lie ahead of the new ones.
struct ChunkStream {
  uint32_t first, count, cached;
  long long before;
};
CH_DEV ChunkStream chunk_stream(const ChunkArgs &a, uint32_t b) {
  ChunkStream s;
  const long long lo = a.starts[b], hi = a.starts[b + 1], top = a.n_tokens;
  s.first = (uint32_t)min(max(lo, 0ll), top);
  const uint32_t end = (uint32_t)min(max(hi, 0ll), top);
  s.count = end > s.first ? end - s.first : 0u;
  if (s.count > a.most) s.count = 0u;
  const long long len = a.lens ? max(a.lens[b], 0) : 0;
  s.cached = (uint32_t)min(len, (long long)a.cols << a.shift);
  s.before = a.prefix + len;
  return s;
}
// The first visible index of the prefix's, the cached and the new tokens for a row at position
// `at`; at or past a run's end: none of it.
struct ChunkLow {
  uint32_t prefix, cached, fresh;
};
CH_DEV ChunkLow chunk_low(const ChunkArgs &a, const ChunkStream &s, long long at) {
  const long long lo = a.window ? max(at + 1 - (long long)a.window, 0ll) : 0ll;
  ChunkLow l;
  l.prefix = (uint32_t)min(lo, (long long)a.prefix);
  l.cached = (uint32_t)min(max(lo - a.prefix, 0ll), (long long)s.cached);
  l.fresh = (uint32_t)max(lo - s.before, 0ll);
  return l;
}
// node above node i of the stream whose rows start at `first`, -1 at a root (or where the parent
// is not an earlier node)
CH_DEV int32_t chunk_parent(const ChunkArgs &a, uint32_t first, uint32_t i) {
  const int32_t p = a.parents[first + i];
  return p >= 0 && (uint32_t)p < i ? p : -1;
}
// what breaks the rules into the status word: starts (by the threads of one CTA), and the parent of
// node i
CH_DEV void chunk_report(const ChunkArgs &a) {
  if (!a.status) return;
  bool bad = false;
  for (uint32_t b = threadIdx.x; b < a.n; b += blockDim.x)
    bad |= a.starts[b] < 0 || a.starts[b + 1] < a.starts[b] || a.starts[b + 1] > (long long)a.n_tokens ||
           (long long)a.starts[b + 1] - a.starts[b] > (long long)a.most;
  if (bad) atomicOr(a.status, DEV_ERR_BAD_LIST);
}
CH_DEV void chunk_report_parent(const ChunkArgs &a, uint32_t first, uint32_t i) {
  const int32_t p = a.parents[first + i];
  if (a.status && (p < -1 || p >= (int32_t)i)) atomicOr(a.status, DEV_ERR_BAD_LIST);
}
CH_DEV uint32_t chunk_depth(const ChunkArgs &a, uint32_t first, uint32_t i) {
  uint32_t d = 0;
  for (int32_t j = chunk_parent(a, first, i); j >= 0; j = chunk_parent(a, first, (uint32_t)j)) d++;
  return d;
}

// K and V rows of a position for one kv head; null where its page is not in the pool (which is reported)
template <typename T>
struct ChunkKey {
  const T *k, *v;
};
// at(x), x = 0 .. n - 1, of every run of positions that new token i of stream s sees: run(n, at) returns
// false to end the walk.  The last run is the stream's new tokens, in a tree one run per node.
template <typename T, typename F>
CH_DEV void chunk_visible(const ChunkArgs &a, const ChunkStream &s, uint32_t b, uint32_t i, uint32_t h, F run) {
  auto paged = [&](const int32_t *table, uint32_t j) {
    const int32_t page = table[j >> a.shift];
    if (page < 0 || (uint32_t)page >= a.n_pages) {
      if (a.status && (threadIdx.x & 31) == 0) atomicOr(a.status, DEV_ERR_BAD_LIST);
      return ChunkKey<T>{nullptr, nullptr};
    }
    const long long at = page * a.page + (long long)(j & ((1u << a.shift) - 1)) * a.token + h * a.head;
    return ChunkKey<T>{static_cast<const T *>(a.k_pool) + at, static_cast<const T *>(a.v_pool) + at};
  };
  auto fresh = [&](uint32_t j) {
    const long long at = (long long)s.first + j;
    return ChunkKey<T>{static_cast<const T *>(a.k) + at * a.ks + h * a.kh, static_cast<const T *>(a.v) + at * a.vs + h * a.vh};
  };
  const uint32_t depth = a.parents && a.window ? chunk_depth(a, s.first, i) : 0u;
  const ChunkLow lo = chunk_low(a, s, s.before + (a.parents ? depth : i));
  if (!run(a.prefix - lo.prefix, [&](uint32_t x) { return paged(a.prefix_table, lo.prefix + x); })) return;
  if (!run(s.cached - lo.cached, [&](uint32_t x) { return paged(a.table + b * a.ts, lo.cached + x); })) return;
  if (a.parents) {  // the path to the root, down to the first depth in the window
    int32_t j = (int32_t)i;
    for (uint32_t d = depth; j >= 0 && (!a.window || d + 1 > lo.fresh); d--, j = chunk_parent(a, s.first, (uint32_t)j))
      if (!run(1u, [&](uint32_t) { return fresh((uint32_t)j); })) return;
  } else {
    run(i + 1 - lo.fresh, [&](uint32_t x) { return fresh(lo.fresh + x); });
  }
}

// Whether a row of results up to x in magnitude needs a second look: NaN, or past the type's largest number.
// An infinity of f16 results is one of the values; the sums of bf16 ones may have left f32.
CH_DEV bool suspect(float x, const __half *) { return !(x <= 65504.f) && x != INFINITY; }
CH_DEV bool suspect(float x, const __nv_bfloat16 *) { return !(x <= 3.38953139e38f); }

// out row of new token i of stream s and q head hq, by one warp, key after key from the visible
// ones only: EPL dims per lane.  Where the sum of weighted values leaves f32, which bf16 values can make
// it do, it is taken again of values 2^32 smaller.
template <typename T, int D>
__device__ __noinline__ void chunk_row(const ChunkArgs &a, const ChunkStream &s, uint32_t b, uint32_t i, uint32_t hq) {
  constexpr int EPL = D / 32;
  const int lane = threadIdx.x & 31;
  const uint32_t h = hq / a.group, row = s.first + i;
  const T *q = static_cast<const T *>(a.q) + row * a.qs + hq * a.qh + lane * EPL;
  float qr[EPL], o[EPL], m, sum, shrink = 1.f;
  uint32_t odd;  // columns with a value that is not finite
#pragma unroll
  for (int e = 0; e < EPL; e++) qr[e] = to_f32(q[e]);
  auto key = [&](const T *k, const T *v) {
    if (sum != sum) return;  // all of the row is NaN
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; e++) x = fmaf(qr[e], to_f32(k[lane * EPL + e]), x);
    x = warp_sum(x) * a.scale;
    if (x == -INFINITY) return;
    const float m1 = fmaxf(m, x), c = m1 == m ? 1.f : expf(m - m1), p = expf(x - m1);
    sum = sum * c + p;
#pragma unroll
    for (int e = 0; e < EPL; e++) {  // (an infinity stays one, however small its weight)
      const float y = to_f32(v[lane * EPL + e]) * shrink, kept = isinf(o[e]) ? o[e] : o[e] * c;
      o[e] = isinf(y) ? kept + y : fmaf(p, y, kept);
      odd |= isfinite(y) ? 0u : 1u << e;
    }
    m = m1;
  };
  for (;;) {
    m = -INFINITY, sum = 0.f, odd = 0u;
#pragma unroll
    for (int e = 0; e < EPL; e++) o[e] = 0.f;
    chunk_visible<T>(a, s, b, i, h, [&](uint32_t n, auto at) {
      for (uint32_t x = 0; x < n; x++)
        if (const ChunkKey<T> at_x = at(x); at_x.k) key(at_x.k, at_x.v);
      return true;
    });
    bool over = false;
#pragma unroll
    for (int e = 0; e < EPL; e++) over |= sum == sum && !isfinite(o[e]) && !(odd >> e & 1);
    if (shrink != 1.f || !__any_sync(0xffffffffu, over)) break;
    shrink = 0x1p-32f;
  }
  T *out = static_cast<T *>(a.out) + row * a.os + hq * a.oh + lane * EPL;
  uint32_t packed[EPL / 2];
#pragma unroll
  for (int e = 0; e < EPL / 2; e++) {
    const float x = sum == 0.f ? 0.f : o[2 * e] / sum / shrink, y = sum == 0.f ? 0.f : o[2 * e + 1] / sum / shrink;
    packed[e] = pack2(x, y, static_cast<const T *>(nullptr));
  }
  if constexpr (EPL == 8)
    *reinterpret_cast<uint4 *>(out) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
  else if constexpr (EPL == 4)
    *reinterpret_cast<uint2 *>(out) = make_uint2(packed[0], packed[1]);
  else
    *reinterpret_cast<uint32_t *>(out) = packed[0];
}

// Columns of an out row that the tensor cores left NaN or infinite although its sum is finite, by one
// warp.  In one of NaN a weight of 0 met a value that is not finite: of a key that the row sees (its weight
// was below the type's range) or of another one of the tile.  What the row sees says what is right: NaN for
// a NaN or infinities of both signs, otherwise the infinity.  Without any (an infinite column then is one
// whose sum left f32, or left the type's range by the rounding of the weights) the row is computed again.  A row of NaN
// throughout may have a sum that is NaN, and then no infinity: unless it is to be NaN either way it is
// computed again too.  Only values are read until all columns are settled, and `hint` first: the key that
// settled an earlier row of the stream and kv head, which a later one sees too where there is neither a
// window nor a tree (8,192 tokens of 256-dim heads with one NaN in the middle 14 ms, without it 33).
template <typename T, int D>
__device__ __noinline__ void chunk_mend(const ChunkArgs &a, const ChunkStream &s, uint32_t b, uint32_t i, uint32_t hq,
                                        ChunkKey<T> &hint) {
  constexpr int EPL = D / 32;
  constexpr uint32_t kAhead = 4;  // keys whose values are on their way together
  struct alignas(2 * EPL) Vec {
    uint32_t w[EPL / 2];
  };
  const int lane = threadIdx.x & 31;
  const uint32_t h = hq / a.group, row = s.first + i;
  T *out = static_cast<T *>(a.out) + row * a.os + hq * a.oh + lane * EPL;
  uint32_t lost = 0, far = 0, up = 0, down = 0, nan = 0;  // of this lane's columns: NaN, infinite; what was seen
#pragma unroll
  for (int e = 0; e < EPL; e++) {
    const float x = to_f32(out[e]);
    lost |= isnan(x) ? 1u << e : 0u, far |= isinf(x) ? 1u << e : 0u;
  }
  const uint32_t open = lost | far;
  if (!__any_sync(0xffffffffu, open)) return;
  const bool whole = __all_sync(0xffffffffu, lost == (1u << EPL) - 1);
  auto look = [&](const ChunkKey<T> &key) {
    const T *q = static_cast<const T *>(a.q) + row * a.qs + hq * a.qh + lane * EPL;
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; e++) x = fmaf(to_f32(q[e]), to_f32(key.k[lane * EPL + e]), x);
    if (warp_sum(x) * a.scale == -INFINITY) return;  // (counts as a key that is not seen)
#pragma unroll
    for (int e = 0; e < EPL; e++) {
      const float v = to_f32(key.v[lane * EPL + e]);
      nan |= isnan(v) ? 1u << e : 0u, up |= v == INFINITY ? 1u << e : 0u, down |= v == -INFINITY ? 1u << e : 0u;
    }
  };
  auto settled = [&]() { return !__any_sync(0xffffffffu, (lost & ~(nan | (up & down))) | (far & ~(nan | up | down))); };
  if (hint.k) look(hint);
  if (settled()) return;
  chunk_visible<T>(a, s, b, i, h, [&](uint32_t n, auto at) {
    for (uint32_t x0 = 0; x0 < n; x0 += kAhead) {
      Vec v[kAhead];
#pragma unroll
      for (uint32_t u = 0; u < kAhead; u++) {
        const ChunkKey<T> key = x0 + u < n ? at(x0 + u) : ChunkKey<T>{nullptr, nullptr};
        v[u] = key.v ? *reinterpret_cast<const Vec *>(key.v + lane * EPL) : Vec{};
      }
      uint32_t hits = 0;
#pragma unroll
      for (uint32_t u = 0; u < kAhead; u++)
#pragma unroll
        for (int e = 0; e < EPL; e++)
          if ((open >> e & 1) && !isfinite(to_f32(reinterpret_cast<const T *>(v[u].w)[e]))) hits |= 1u << u;
      hits = __reduce_or_sync(0xffffffffu, hits);
      if (!hits) continue;
      for (; hits; hits &= hits - 1) {
        const ChunkKey<T> key = at(x0 + __ffs(hits) - 1);
        look(key);
        if (settled()) {
          if (!a.window && !a.parents) hint = key;
          return false;
        }
      }
    }
    return true;
  });
  const uint32_t one = whole ? 0u : open & ~nan & (up ^ down);
  if (__any_sync(0xffffffffu, open & ~(nan | one | (up & down)))) {
    chunk_row<T, D>(a, s, b, i, hq);
    return;
  }
#pragma unroll
  for (int e = 0; e < EPL; e++)
    if (one >> e & 1) {
      const uint32_t word = pack2(up >> e & 1 ? INFINITY : -INFINITY, 0.f, static_cast<const T *>(nullptr));
      *reinterpret_cast<uint16_t *>(out + e) = (uint16_t)word;
    }
}

}  // namespace ch
