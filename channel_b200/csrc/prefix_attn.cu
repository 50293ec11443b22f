// prefix_attn.cu -- attention of one query token per stream over a prompt that all streams
// share and each stream's own tokens, both in pages (ch_prefix_attention).
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - m),
// over the visible positions j; m is the running maximum, and sums are f32.
#include <algorithm>
#include <cstring>
#include <string>
#include <type_traits>

#include "../../include/channel_cuda.h"
#include "prefix_tc.cuh"

namespace ch {
int set_last_error(int code, const std::string &msg);

namespace {
CH_DEV void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
CH_DEV void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
CH_DEV uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
CH_DEV void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const __half *) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
CH_DEV void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const __nv_bfloat16 *) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// ---------------------------------------------------------------------------
// Positions read stream by stream.  HBM-bound: each K and V row is used by the `group`
// query rows of its kv head only, so what counts is bytes in flight.  A warp is a unit of
// its own: it takes an equal run of the 16-key tiles of all (stream, kv head) pairs, laid
// end to end, and streams them through a private ring of row copies (lane l < 16 copies K
// row l of a tile, lane 16 + l its V row), so no barrier couples the warps and tiles of the
// next pair are in flight while one pair ends.  A tile takes
//   S^T (16 keys x 8 rows) = K (16 x D) Q^T,   O^T (D x 8 rows) += V^T (D x 16 keys) P^T,
// with K and V as the 16-row A operand of mma.m16n8k16 (the query rows, at most 8 or 16, are
// its narrow side) and P^T from S^T by two 8 x 8 register transposes.  P is rounded to the
// type of V (what the tensor core takes), in f16 times 2^15 (at most 32,768 then), so that
// weights far below the run's largest one do not fall under the type's least; its sum is kept in
// f32 before rounding.  The running maximum, in units of log2, is per warp; each cut pair leaves (O, m, l) in the
// workspace and attend_join_kernel adds the parts.
//
// Measured (8 kv heads of 256, two q heads each, with the shared prefix of prefix_tc.cuh beside
// it in the same launch, and the join): 64 streams of 1 to 1,023 own tokens behind 4,096 shared
// ones 61 to 62 us (303 MB, 4.9 TB/s; a kernel per row 1,648 us), behind 32,768 with 1 to 2,047 own
// ones 138 to 141 us (5.8 TB/s), a window of 1,024 67 to 70 us; 37 streams of 32 q on 8 kv heads of 128
// 26 us, 4 streams behind 192 tokens 12 us.  The small ones are the latency of one launch with a join.
constexpr uint32_t kTile = 16;  // keys
template <typename T>
constexpr float kOwnBias = std::is_same<T, __half>::value ? 15.f : 0.f;  // log2 of the factor on P
template <int D>
struct Own {
  static constexpr int kWarps = D == 256 ? 6 : 8;
  static constexpr int kStages = D == 64 ? 5 : D == 128 ? 3 : 2;
  static constexpr uint32_t kPitch = D * 2 + 16;  // 8 rows of a fragment load hit distinct banks
  static constexpr uint32_t kStage = 2 * kTile * kPitch;
  static constexpr uint32_t kRing = kWarps * kStages * kStage;
  static constexpr int kThreads = kWarps * 32 > kTcThreads ? kWarps * 32 : kTcThreads;
  // shared memory: the prefix unit's or the rings, then start[n + 1]
  static constexpr uint32_t kOffStart = Tc<D>::kBytes > kRing ? Tc<D>::kBytes : kRing;
};
constexpr uint32_t kMaxStreams = 4096;

// How the work is dealt to the CTAs, the same in each (computed from lens by all of them).
// The prefix is n_kv * row tiles * splits units for CTAs 0, 1, ...; the 16-key tiles of the
// streams go to the warps in equal runs, longer ones (y tiles) to the CTAs without a unit and
// shorter ones (x) to those with one, by the units' cost.
struct Deal {
  uint32_t splits;  // of the prefix
  uint32_t units, unit_ctas;
  uint32_t y_runs, y, x;  // runs 0 .. y_runs - 1 have y tiles, the rest x
};
struct Work {       // in the caller's workspace
  uint32_t *start;  // [n + 1] first tile of a stream, per kv head
  Deal *deal;
  float *o;    // [segments][group][D]; segment = run + pair, pair = stream * n_kv + head
  float2 *ml;  // [segments][group]: maximum, sum
};
// What a 64-key tile of the prefix and a unit's start and end cost, in 16-key tiles.  By
// bytes a tile costs 4; measured best is 3 (64 streams behind 4K / 32K tokens: 64 / 143 us,
// with 4: 66 / 148, with 5: 67 / 157), because a unit's CTA has its SM's copies to itself.
constexpr uint32_t kCostTile = 3, kCostUnit = 24;

// own: 16-key tiles of all streams and kv heads (below 2^31).  The shares are estimates in
// f32, the same in every CTA; y is then what exactly covers all tiles.
CH_DEV Deal deal_work(uint32_t own, uint32_t ptiles, uint32_t per_split, uint32_t max_splits, uint32_t ctas,
                      uint32_t warps) {
  Deal d;
  const float prefix = (float)ptiles * per_split * kCostTile;
  d.splits = 0;
  if (ptiles) {
    const float want = ceilf(prefix * ctas / ((own + prefix) * per_split));
    d.splits = max(1u, min(min(max_splits, ptiles), (uint32_t)want));
  }
  d.units = d.splits * per_split;
  d.unit_ctas = min(d.units, ctas);
  const uint32_t rest = ctas - d.unit_ctas, x_runs = d.unit_ctas * warps;
  d.y_runs = rest * warps;
  // a CTA's cost of its units, and the even share of everything
  const float used = d.units ? (prefix + (float)d.units * kCostUnit) / d.unit_ctas : 0.f;
  const float share = (own + used * d.unit_ctas) / ctas;
  d.y = 0;
  if (rest == 0) {
    d.x = (own + x_runs - 1) / x_runs;
  } else {
    d.x = used < share ? (uint32_t)((share - used) / warps) : 0u;
    if (own > d.x * x_runs) d.y = (own - d.x * x_runs + d.y_runs - 1) / d.y_runs;
  }
  return d;
}

// Registers: room for the join's CTAs beside it (they wait on the SM while this kernel runs),
// but not where 16 query rows need them all.
constexpr int attend_bound(int D, int NR) { return D == 256 && NR == 2 ? 256 : 320; }

template <typename T, int D, int NR>
__global__ void __launch_bounds__(attend_bound(D, NR), 1)
    attend_kernel(const PrefixArgs a, const Work w, const PrefixParts pp, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap vmap) {
  using O = Own<D>;
  constexpr int kThreads = O::kThreads, kSteps = D / 16;
  extern __shared__ uint8_t smem_dyn[];
  uint8_t *smem = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
  uint32_t *start = reinterpret_cast<uint32_t *>(smem + O::kOffStart);  // [n + 1]
  __shared__ TcBars tc_bars;
  __shared__ __align__(8) uint64_t bars[O::kWarps][O::kStages];
  __shared__ uint32_t masks[O::kWarps][O::kStages], sums[kThreads / 32], lo_min;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;

  grid_dep_wait();  // the kernel in front may still be running
  // ---- tiles per stream, summed over the streams; the first position any stream sees ----
  const uint32_t per_thread = (a.n + kThreads - 1) / kThreads, b0 = min(a.n, tid * per_thread), b1 = min(a.n, b0 + per_thread);
  uint32_t mine = 0, low = 0xFFFFFFFFu;
  auto tiles_of = [&](uint32_t b) {
    uint32_t lo, hi;
    visible(a, b, lo, hi);
    low = min(low, lo);
    lo = max(lo, a.from);
    return hi > lo ? (hi - lo + kTile - 1) / kTile : 0u;
  };
  if (tid == 0) lo_min = 0xFFFFFFFFu;
  for (uint32_t b = b0; b < b1; b++) {
    const uint32_t n = tiles_of(b);
    start[b] = n;
    mine += n;
  }
  uint32_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) sums[warp] = inc;
  if (warp < O::kWarps && lane < O::kStages) mbar_init(&bars[warp][lane], 1);
  fence_mbar_init();
  __syncthreads();
  low = __reduce_min_sync(0xffffffffu, low);
  if (lane == 0) atomicMin(&lo_min, low);
  uint32_t at = inc - mine, all = 0;
  for (int k = 0; k < kThreads / 32; k++) {
    if (k < warp) at += sums[k];
    all += sums[k];
  }
  for (uint32_t b = b0; b < b1; b++) {
    const uint32_t n = start[b];
    start[b] = at;
    at += n;
  }
  if (tid == 0) start[a.n] = all;
  __syncthreads();
  const uint32_t zlo = min(lo_min, a.prefix), tile0 = zlo / kKeys;
  const uint32_t ptiles = pp.max_splits && zlo < a.prefix ? (a.prefix + kKeys - 1) / kKeys - tile0 : 0u;
  const uint32_t row_tiles = (a.n * a.group + kRows - 1) / kRows;
  const uint32_t total = all * a.nkv;
  const Deal d = deal_work(total, ptiles, a.nkv * row_tiles, pp.max_splits, gridDim.x, O::kWarps);
  if (blockIdx.x == gridDim.x - 1) {
    for (uint32_t b = tid; b <= a.n; b += kThreads) w.start[b] = start[b];
    if (tid == 0) *w.deal = d;
  }
  grid_dep_launch();

  // ---- the shared prefix ----
  bool dead = false;  // a wait gave up
  for (uint32_t u = blockIdx.x; u < d.units; u += gridDim.x) {
    const uint32_t h = u % a.nkv, rt = (u / a.nkv) % row_tiles, split = u / (a.nkv * row_tiles);
    const uint32_t i0 = split * (ptiles / d.splits) + min(split, ptiles % d.splits);
    const uint32_t i1 = i0 + ptiles / d.splits + (split < ptiles % d.splits);
    dead = dead || !prefix_unit<T, D>(a, pp, kmap, vmap, smem, tc_bars, h, rt, split, tile0 + i0, i1 - i0, zlo);
    const uint32_t rows = a.n * a.group, gr = rt * kRows + tid;
    if (dead && tid < (int)kRows && gr < rows) pp.ml[((size_t)split * a.nkv + h) * rows + gr] = make_float2(0.f, NAN);
  }

  // ---- this warp's run of the streams' own tiles; consecutive runs lie on different SMs, so
  // that few tiles spread over all of them ----
  if (warp >= O::kWarps) return;  // (no barrier of the CTA from here on)
  const bool with_unit = blockIdx.x < d.unit_ctas;
  const uint32_t run = with_unit ? d.y_runs + warp * d.unit_ctas + blockIdx.x
                                 : warp * (gridDim.x - d.unit_ctas) + blockIdx.x - d.unit_ctas;
  const uint32_t per = with_unit ? d.x : d.y;
  const uint32_t first = with_unit ? d.y_runs * d.y + (run - d.y_runs) * d.x : run * d.y;
  if (per == 0 || first >= total) return;
  uint32_t left = min(per, total - first);

  struct Cursor {
    uint32_t b, h, i, tiles, lo, hi;
  };
  auto enter = [&](Cursor &c, bool bounds) {
    c.tiles = start[c.b + 1] - start[c.b];
    if (!bounds) return;
    visible(a, c.b, c.lo, c.hi);
    c.lo = max(c.lo, a.from);
  };
  Cursor ld;
  {
    uint32_t lo = 0, hi = a.n;
    while (lo + 1 < hi) {
      const uint32_t mid = (lo + hi) >> 1;
      if (start[mid] * a.nkv <= first) lo = mid; else hi = mid;
    }
    ld.b = lo;
    while (start[ld.b + 1] == start[ld.b]) ld.b++;
    enter(ld, true);
    const uint32_t rem = first - start[ld.b] * a.nkv;
    ld.h = rem / ld.tiles;
    ld.i = rem % ld.tiles;
  }
  auto advance = [&](Cursor &c, bool bounds) {
    if (++c.i < c.tiles) return;
    c.i = 0;
    if (++c.h < a.nkv) return;
    c.h = 0;
    do c.b++;
    while (c.b < a.n && start[c.b + 1] == start[c.b]);
    if (c.b < a.n) enter(c, bounds);
  };
  Cursor cu = ld;
  auto give_up = [&]() {  // the rest of the run: sums of NaN, as for a prefix unit
    for (; left; left--) {
      const unsigned long long seg = (unsigned long long)run + cu.b * a.nkv + cu.h;
      if ((cu.i + 1 == cu.tiles || left == 1) && lane < (int)a.group) w.ml[seg * a.group + lane] = make_float2(0.f, NAN);
      advance(cu, false);
    }
  };
  if (dead) return give_up();
  uint32_t qf[NR][kSteps][2];
  float o[NR][kSteps][4], m[NR][2], l[NR][2];
  const float scale2 = a.scale * 1.44269504088896341f;
  const T *tag = nullptr;
  auto begin_pair = [&]() {  // the pair's query rows and empty sums
#pragma unroll
    for (int r = 0; r < NR; r++) {
      const uint32_t qr = r * 8 + g;
      const T *q = static_cast<const T *>(a.q) + cu.b * a.qs + (cu.h * a.group + qr) * a.qh + 2 * t4;
#pragma unroll
      for (int k = 0; k < kSteps; k++) {
        qf[r][k][0] = qr < a.group ? *reinterpret_cast<const uint32_t *>(q + 16 * k) : 0u;
        qf[r][k][1] = qr < a.group ? *reinterpret_cast<const uint32_t *>(q + 16 * k + 8) : 0u;
#pragma unroll
        for (int e = 0; e < 4; e++) o[r][k][e] = 0.f;
      }
      m[r][0] = m[r][1] = -INFINITY;
      l[r][0] = l[r][1] = 0.f;
    }
  };
  begin_pair();  // these reads and the first page reads are in flight together
  bool fresh = false;
  uint8_t *ring = smem + warp * O::kStages * O::kStage;
  const T *pool = static_cast<const T *>(lane < 16 ? a.k : a.v);
  uint32_t to_load = left;
  // A tile on its way: its page index as read (looked at only when the copies go out, so that
  // the reads of several tiles are in flight together)
  struct Tile {
    int32_t page;
    uint32_t row, h;
    bool in;
  };
  auto look_up = [&]() {
    Tile t;
    const uint32_t j = ld.lo + ld.i * kTile + (lane & 15);
    t.in = j < ld.hi;
    t.h = ld.h;
    const bool shared = j < a.prefix;
    const uint32_t i = shared ? j : j - a.prefix;
    t.row = i & ((1u << a.shift) - 1);
    t.page = -1;
    if (t.in) t.page = shared ? a.prefix_table[i >> a.shift] : a.table[ld.b * a.ts + (i >> a.shift)];
    return t;
  };
  auto issue = [&](const Tile &t, int s) {
    uint8_t *dst = ring + s * O::kStage + lane * O::kPitch;
    const bool there = t.page >= 0 && (uint32_t)t.page < a.n_pages;
    const uint32_t have = __ballot_sync(0xffffffffu, there);
    if (!there) {  // not copied: zeros, so that a weight of 0 meets no stale bits
      if (t.in && a.status) atomicOr(a.status, DEV_ERR_BAD_LIST);
      for (uint32_t c = 0; c < D * 2; c += 16) *reinterpret_cast<uint4 *>(dst + c) = make_uint4(0, 0, 0, 0);
      fence_proxy_async();
    }
    if (lane == 0) {
      masks[warp][s] = have & 0xFFFFu;
      mbar_arrive_expect_tx(&bars[warp][s], __popc(have) * D * 2);
    }
    __syncwarp();
    if (there) bulk_g2s(dst, pool + t.page * a.page + (long long)t.row * a.token + t.h * a.head, D * 2, &bars[warp][s]);
  };
  Tile ahead[O::kStages];
#pragma unroll
  for (int s = 0; s < O::kStages; s++)
    if ((uint32_t)s < to_load) {
      ahead[s] = look_up();
      advance(ld, true);
    }
#pragma unroll
  for (int s = 0; s < O::kStages; s++)
    if ((uint32_t)s < to_load) issue(ahead[s], s);
  to_load -= min(to_load, (uint32_t)O::kStages);
  Tile next;
  auto read_ahead = [&]() {
    if (!to_load) return;
    next = look_up();
    advance(ld, true);
  };
  read_ahead();

  const uint32_t frag = smem_u32(ring);
  // fragment addresses of this lane: K rows by key, V columns by key
  const uint32_t k_at = ((lane & 7) + ((lane >> 3) & 1) * 8) * O::kPitch + (lane >> 4) * 16;
  const uint32_t v_at = (kTile + (lane & 7) + (lane >> 4) * 8) * O::kPitch + ((lane >> 3) & 1) * 16;
  int stage = 0;
  uint32_t parity = 0;
  for (; left; left--) {
    if (fresh) {
      fresh = false;
      begin_pair();
    }
    const bool ok = mbar_wait_bounded(&bars[warp][stage], parity, a.status);
    if (!__all_sync(0xffffffffu, ok)) {  // reported; the copies still in flight get a wait of their own
      for (int k = 0; k < O::kStages && (uint32_t)k < left; k++) {
        mbar_wait_bounded(&bars[warp][stage], parity, a.status);
        if (++stage == O::kStages) stage = 0, parity ^= 1;
      }
      return give_up();
    }
    const uint32_t base = frag + stage * O::kStage, mask = masks[warp][stage];
    float s[NR][2][4];
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
      for (int e = 0; e < 4; e++) s[r][0][e] = s[r][1][e] = 0.f;
#pragma unroll
    for (int k = 0; k < kSteps; k++) {
      uint32_t f[4];
      ldsm_x4(base + k_at + k * 32, f);
#pragma unroll
      for (int r = 0; r < NR; r++) mma16(s[r][k & 1], f, qf[r][k][0], qf[r][k][1], tag);
    }
    const bool on0 = (mask >> g) & 1, on1 = (mask >> (g + 8)) & 1;
    uint32_t p[NR][2];
#pragma unroll
    for (int r = 0; r < NR; r++) {
#pragma unroll
      for (int c = 0; c < 2; c++) {  // query row r * 8 + 2 * t4 + c, keys g and g + 8
        const float s0 = on0 ? (s[r][0][c] + s[r][1][c]) * scale2 : -INFINITY;
        const float s1 = on1 ? (s[r][0][c + 2] + s[r][1][c + 2]) * scale2 : -INFINITY;
        float top = fmaxf(s0, s1);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float m1 = fmaxf(m[r][c], top), ref = m1 == -INFINITY ? 0.f : m1;
        const float keep = exp2_approx(m[r][c] - ref);
        m[r][c] = m1;
        const float below = ref - kOwnBias<T>, p0 = exp2_approx(s0 - below), p1 = exp2_approx(s1 - below);
        l[r][c] = l[r][c] * keep + (p0 + p1);
        s[r][0][c] = p0;
        s[r][0][c + 2] = p1;
        s[r][1][c] = keep;
      }
      p[r][0] = transpose8x8(pack2(s[r][0][0], s[r][0][1], tag));
      p[r][1] = transpose8x8(pack2(s[r][0][2], s[r][0][3], tag));
      if (__any_sync(0xffffffffu, s[r][1][0] != 1.f || s[r][1][1] != 1.f)) {
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
          o[r][k][0] *= s[r][1][0], o[r][k][1] *= s[r][1][1];
          o[r][k][2] *= s[r][1][0], o[r][k][3] *= s[r][1][1];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kSteps; k++) {
      uint32_t f[4];
      ldsm_x4_trans(base + v_at + k * 32, f);
#pragma unroll
      for (int r = 0; r < NR; r++) mma16(o[r][k], f, p[r][0], p[r][1], tag);
    }
    __syncwarp();
    if (to_load) {
      issue(next, stage);
      to_load--;
      read_ahead();
    }
    if (++stage == O::kStages) stage = 0, parity ^= 1;

    if (cu.i + 1 == cu.tiles || left == 1) {  // the pair, or this warp's run, ends
      const unsigned long long seg = (unsigned long long)run + cu.b * a.nkv + cu.h;
      float *po = w.o + seg * a.group * D;
      float2 *pm = w.ml + seg * a.group;
#pragma unroll
      for (int r = 0; r < NR; r++) {
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float sum = l[r][c];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
          const uint32_t qr = r * 8 + 2 * t4 + c;
          if (qr >= a.group) continue;
          if (g == 0) pm[qr] = make_float2(m[r][c] - kOwnBias<T>, sum);
#pragma unroll
          for (int k = 0; k < kSteps; k++) {
            po[qr * D + 16 * k + g] = o[r][k][c];
            po[qr * D + 16 * k + 8 + g] = o[r][k][c + 2];
          }
        }
      }
      fresh = true;
    }
    advance(cu, false);
  }
}

// ---------------------------------------------------------------------------
// out = sum over a row's parts of O 2^(m - M) / sum of l 2^(m - M); a warp per query row.
// A weight of 0 times a non-finite V at a masked position of the same tile is NaN, so a row
// that is not finite is computed again on its own, key by key, from its visible positions
// only (ordinary rows never take this path).
constexpr int kJoinWarps = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) attend_join_kernel(const PrefixArgs a, const Work w, const PrefixParts pp) {
  constexpr int EPL = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t row = blockIdx.x * kJoinWarps + warp;
  if (row >= a.n * a.nq) return;
  const uint32_t b = row / a.nq, hq = row % a.nq, h = hq / a.group, r = hq % a.group;
  grid_dep_wait();
  grid_dep_launch();
  // the row's parts: one per split of the shared prefix, then one per warp whose run touched
  // the pair (b, h)
  const uint32_t s0 = w.start[b], tiles = w.start[b + 1] - s0;
  const Deal d = *w.deal;
  const uint32_t t0 = s0 * a.nkv + h * tiles, y_tiles = d.y_runs * d.y;
  auto run_of = [&](uint32_t t) { return t < y_tiles ? t / d.y : d.y_runs + (t - y_tiles) / d.x; };
  const uint32_t w0 = tiles ? run_of(t0) : 0u, own = tiles ? run_of(t0 + tiles - 1) - w0 + 1 : 0u;
  const size_t rows = (size_t)a.n * a.group, at_prefix = (size_t)h * rows + (size_t)b * a.group + r;
  const size_t at_own = ((size_t)w0 + (size_t)b * a.nkv + h) * a.group + r;
  const uint32_t parts = d.splits + own;
  auto ml_of = [&](uint32_t p) {
    return p < d.splits ? pp.ml[at_prefix + (size_t)p * a.nkv * rows] : w.ml[at_own + (size_t)(p - d.splits) * a.group];
  };
  auto o_of = [&](uint32_t p) {
    return (p < d.splits ? pp.o + (at_prefix + (size_t)p * a.nkv * rows) * D
                          : w.o + (at_own + (size_t)(p - d.splits) * a.group) * D) + lane * EPL;
  };
  constexpr uint32_t kU = 4;  // parts whose loads are in flight together, the first before the maxima are known
  float v[kU][EPL];
  auto load = [&](uint32_t p0) {
#pragma unroll
    for (uint32_t u = 0; u < kU; u++) {
      if (p0 + u >= parts) break;
      const float *src = o_of(p0 + u);
      if constexpr (EPL == 2) {
        *reinterpret_cast<float2 *>(v[u]) = *reinterpret_cast<const float2 *>(src);
      } else {
#pragma unroll
        for (int e = 0; e < EPL; e += 4) *reinterpret_cast<float4 *>(&v[u][e]) = *reinterpret_cast<const float4 *>(src + e);
      }
    }
  };
  load(0);
  float top = -INFINITY;
  for (uint32_t p = lane; p < parts; p += 32) top = fmaxf(top, ml_of(p).x);
  top = warp_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float o[EPL], sum = 0.f;
#pragma unroll
  for (int e = 0; e < EPL; e++) o[e] = 0.f;
  for (uint32_t p0 = 0; p0 < parts; p0 += 32) {
    float f = 0.f;
    if (p0 + lane < parts) {
      const float2 x = ml_of(p0 + lane);
      f = exp2_approx(x.x - ref);
      sum = fmaf(x.y, f, sum);
    }
    for (uint32_t k = 0; k < 32 && p0 + k < parts; k += kU) {
      if (p0 + k) load(p0 + k);
#pragma unroll
      for (uint32_t u = 0; u < kU; u++) {
        const float fk = __shfl_sync(0xffffffffu, f, k + u);  // 0 past the last part
        if (fk == 0.f) continue;  // a part without a visible position has no O
#pragma unroll
        for (int e = 0; e < EPL; e++) o[e] = fmaf(v[u][e], fk, o[e]);
      }
    }
  }
  sum = warp_sum(sum);
  bool bad = !isfinite(sum);
#pragma unroll
  for (int e = 0; e < EPL; e++) {
    o[e] = sum == 0.f ? 0.f : o[e] / sum;
    bad |= !isfinite(o[e]);
  }
  if (__any_sync(0xffffffffu, bad)) {
    const T *q = static_cast<const T *>(a.q) + b * a.qs + hq * a.qh + lane * EPL;
    float qr[EPL], m = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; e++) qr[e] = to_f32(q[e]), o[e] = 0.f;
    uint32_t lo, hi;
    visible(a, b, lo, hi);
    for (uint32_t j = lo; j < hi; j++) {
      uint32_t in_page;
      const int32_t page = page_of(a, b, j, in_page);
      if (page < 0) continue;
      const long long at = page * a.page + (long long)in_page * a.token + h * a.head + lane * EPL;
      const T *k = static_cast<const T *>(a.k) + at, *v = static_cast<const T *>(a.v) + at;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; e++) s = fmaf(qr[e], to_f32(k[e]), s);
      s = warp_sum(s) * a.scale;
      if (s == -INFINITY) continue;
      const float m1 = fmaxf(m, s), c = expf(m - m1), p = expf(s - m1);
      sum = sum * c + p;
#pragma unroll
      for (int e = 0; e < EPL; e++) o[e] = fmaf(p, to_f32(v[e]), o[e] * c);
      m = m1;
    }
#pragma unroll
    for (int e = 0; e < EPL; e++) o[e] = sum == 0.f ? 0.f : o[e] / sum;
  }
  T *out = static_cast<T *>(a.out) + b * a.os + hq * a.oh + lane * EPL;
  uint32_t packed[EPL / 2];
#pragma unroll
  for (int e = 0; e < EPL / 2; e++) packed[e] = pack2(o[2 * e], o[2 * e + 1], static_cast<const T *>(nullptr));
  if constexpr (EPL == 8)
    *reinterpret_cast<uint4 *>(out) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
  else if constexpr (EPL == 4)
    *reinterpret_cast<uint2 *>(out) = make_uint2(packed[0], packed[1]);
  else
    *reinterpret_cast<uint32_t *>(out) = packed[0];
}

// The shared prefix has its own kernel when more than one stream can share it.
bool shares(const ch_prefix_attn_args *p) { return p->prefix_len > 0 && p->n_streams > 1; }

// As many splits as fit the SMs at once, at most one per key tile.
uint32_t max_splits(const ch_prefix_attn_args *p) {
  if (!shares(p)) return 0;
  const unsigned long long rows = (unsigned long long)p->n_streams * (p->n_q / p->n_kv);
  const unsigned long long per_split = (rows + kRows - 1) / kRows * p->n_kv;
  return (uint32_t)std::max(1ull, std::min<unsigned long long>((unsigned)num_sms() / per_split,
                                                               (p->prefix_len + kKeys - 1) / kKeys));
}
// workspace: w.start | w.deal | w.ml | w.o | the prefix's ml | o, each on 256 bytes (the parts of O
// are stored 32 bytes at a time); the caller's base is on 16 only, so there is room to align it
size_t aligned(size_t bytes) { return (bytes + 255) & ~(size_t)255; }
size_t carve(const ch_prefix_attn_args *p, uint8_t *base, Work *w, PrefixParts *pp) {
  base = reinterpret_cast<uint8_t *>(aligned(reinterpret_cast<uintptr_t>(base)));
  const uint32_t runs = (uint32_t)num_sms() * (p->head_dim == 256 ? Own<256>::kWarps : Own<128>::kWarps);
  static_assert(Own<64>::kWarps == Own<128>::kWarps, "runs");
  const size_t rows = ((size_t)runs + (size_t)p->n_streams * p->n_kv) * (p->n_q / p->n_kv);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t *r = base + at;
    at += aligned(bytes);
    return r;
  };
  w->start = reinterpret_cast<uint32_t *>(take(((size_t)p->n_streams + 1) * sizeof(uint32_t)));
  w->deal = reinterpret_cast<Deal *>(take(sizeof(Deal)));
  w->ml = reinterpret_cast<float2 *>(take(rows * sizeof(float2)));
  w->o = reinterpret_cast<float *>(take(rows * p->head_dim * sizeof(float)));
  pp->max_splits = max_splits(p);
  const size_t shared = (size_t)pp->max_splits * p->n_streams * p->n_q;
  pp->ml = reinterpret_cast<float2 *>(take(shared * sizeof(float2)));
  pp->o = reinterpret_cast<float *>(take(shared * p->head_dim * sizeof(float)));
  return at + 256 - 16;
}

// kernel<<<grid, block, smem, s>>>(args...), which may start before the kernel in front of it
// ends: both kernels here wait for that one before they read or write anything
template <typename K, typename... A>
cudaError_t start_kernel(K kernel, uint32_t grid, uint32_t block, size_t smem, cudaStream_t s, const A &...args) {
  cudaError_t e = ensure_smem_attr((const void *)kernel, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int D>
cudaError_t launch_t(PrefixArgs a, const Work &w, PrefixParts pp, cudaStream_t s) {
  alignas(64) CUtensorMap kmap, vmap;
  std::memset(&kmap, 0, sizeof(kmap));
  std::memset(&vmap, 0, sizeof(vmap));
  if (pp.max_splits) {
    const uint32_t ps = 1u << a.shift;
    // pools no tensor map can describe are read stream by stream
    if (pool_map(&kmap, a.k, a, D, std::min(ps, kKeys), false) != cudaSuccess ||
        pool_map(&vmap, a.v, a, D, std::min(ps, Tc<D>::kVKeys), true) != cudaSuccess)
      pp.max_splits = 0;
  }
  a.from = pp.max_splits ? a.prefix : 0;
  const size_t smem = 1024 + Own<D>::kOffStart + ((size_t)a.n + 1) * sizeof(uint32_t);
  const cudaError_t e = start_kernel(a.group <= 8 ? attend_kernel<T, D, 1> : attend_kernel<T, D, 2>, num_sms(),
                                     Own<D>::kThreads, smem, s, a, w, pp, kmap, vmap);
  if (e != cudaSuccess) return e;
  return start_kernel(attend_join_kernel<T, D>, (a.n * a.nq + kJoinWarps - 1) / kJoinWarps, kJoinWarps * 32, 0, s, a, w, pp);
}
template <typename T>
cudaError_t launch(const PrefixArgs &a, const Work &w, const PrefixParts &pp, uint32_t D, cudaStream_t s) {
  return D == 64 ? launch_t<T, 64>(a, w, pp, s) : D == 128 ? launch_t<T, 128>(a, w, pp, s) : launch_t<T, 256>(a, w, pp, s);
}

const char *check(const ch_prefix_attn_args *p) {
  if (!p) return "args is NULL";
  if (p->n_streams > kMaxStreams) return "at most 4096 streams";
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return "head_dim must be 64, 128 or 256";
  if (p->n_kv == 0 || p->n_q == 0 || p->n_q % p->n_kv || p->n_q / p->n_kv > 16)
    return "n_q must be n_kv times 1..16";
  if (p->n_q > 1024) return "at most 1024 q heads";
  if (p->page_size < 8 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
    return "page_size must be a power of two from 8 to 256";
  if (p->n_pages > 0x7FFFFFFFu || p->table_cols > 0x7FFFFFFFu || p->prefix_len > 0x7FFFFFFFu)
    return "a size is 2^31 or more";
  const unsigned long long reach = p->prefix_len + (unsigned long long)p->table_cols * p->page_size;
  if (reach >= 1ull << 32 || (reach / 16 + 1) * p->n_streams >= (1ull << 31) / p->n_kv)
    return "the positions of all streams and kv heads exceed 2^35";
  if (p->dtype != CH_F16 && p->dtype != CH_BF16) return "dtype must be CH_F16 or CH_BF16";
  return nullptr;
}

int prefix_attention(const ch_prefix_attn_args *p, void *workspace, size_t bytes, void *stream) {
  if (const char *why = check(p)) return set_last_error(CH_EINVAL, std::string("prefix_attention: ") + why);
  if (p->n_streams == 0) return CH_OK;
  if (!p->q || !p->out || !p->k_pool || !p->v_pool || !p->lens || (p->prefix_len && !p->prefix_table) ||
      (p->table_cols && !p->table))
    return set_last_error(CH_EINVAL, "prefix_attention: NULL argument");
  // (the stride of a dimension of one element is never used, and may be any number)
  const int64_t streams = p->n_streams > 1 ? p->q_stream_stride | p->out_stream_stride : 0;
  const int64_t heads = (p->n_q > 1 ? p->q_head_stride | p->out_head_stride : 0) | (p->n_kv > 1 ? p->head_stride : 0);
  if ((streams | heads | (p->n_pages > 1 ? p->page_stride : 0) | p->token_stride) & 7)
    return set_last_error(CH_EINVAL, "prefix_attention: strides must be multiples of 8 elements");
  if (((uintptr_t)p->q | (uintptr_t)p->out | (uintptr_t)p->k_pool | (uintptr_t)p->v_pool) & 15)
    return set_last_error(CH_EINVAL, "prefix_attention: q, out and the pools must be 16-byte aligned");
  const size_t need = ch_prefix_attention_workspace(p);
  if (bytes < need || (need && (!workspace || ((uintptr_t)workspace & 15))))
    return set_last_error(CH_EINVAL, "prefix_attention: workspace must be 16-byte aligned, of " +
                                         std::to_string(need) + " bytes");
  PrefixArgs a{};
  a.q = p->q;
  a.k = p->k_pool;
  a.v = p->v_pool;
  a.out = p->out;
  a.prefix_table = p->prefix_table;
  a.table = p->table;
  a.lens = p->lens;
  a.qs = p->q_stream_stride;
  a.qh = p->q_head_stride;
  a.os = p->out_stream_stride;
  a.oh = p->out_head_stride;
  a.page = p->page_stride;
  a.token = p->token_stride;
  a.head = p->head_stride;
  a.ts = p->table_stride;
  a.n = p->n_streams;
  a.nq = p->n_q;
  a.nkv = p->n_kv;
  a.group = p->n_q / p->n_kv;
  while ((1u << a.shift) < p->page_size) a.shift++;
  a.n_pages = p->n_pages;
  a.cols = p->table_cols;
  a.prefix = p->prefix_len;
  a.window = p->window;
  a.scale = p->scale;
  a.status = p->status;
  Work w;
  PrefixParts pp;
  carve(p, static_cast<uint8_t *>(workspace), &w, &pp);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      p->dtype == CH_F16 ? launch<__half>(a, w, pp, p->head_dim, s) : launch<__nv_bfloat16>(a, w, pp, p->head_dim, s);
  if (e != cudaSuccess) return set_last_error(CH_ECUDA, std::string("prefix_attention: ") + cudaGetErrorString(e));
  return CH_OK;
}
}  // namespace
}  // namespace ch

extern "C" size_t ch_prefix_attention_workspace(const ch_prefix_attn_args *args) {
  if (ch::check(args)) return 0;
  ch::Work w;
  ch::PrefixParts pp;
  return ch::carve(args, nullptr, &w, &pp);
}
extern "C" int ch_prefix_attention(const ch_prefix_attn_args *args, void *workspace, size_t workspace_bytes,
                                   void *stream) {
  try {
    return ch::prefix_attention(args, workspace, workspace_bytes, stream);
  } catch (...) {
    return CH_ENOMEM;
  }
}
