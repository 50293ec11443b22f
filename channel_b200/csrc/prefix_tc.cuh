// prefix_tc.cuh -- the shared prefix of ch_prefix_attention on the 5th-generation tensor
// cores: every shared K and V row is read once for all streams.
//
// The query rows of one kv head -- `group` per stream, row b * group + g -- are the M = 128
// rows of a tile (a batch of 64 streams with two q heads per kv head fills it); a unit is one
// row tile and a run of the prefix's 64-key tiles, and per key tile
//   S (128 x 64) = Q K^T,   P = 2^(scale log2(e) S - m),   O (128 x D) += P V.
// Q, S (two buffers), P (over its S) and O live in tensor memory (128 + 2 x 64 + 256 columns
// at D = 256; Q and P are the products' operand A), so that shared memory is one ring of K
// and V alone: 16 KB pieces by TMA from the pages (K: a box per page and 64 dims, V: a box
// per page; 128-byte swizzle) in the order the products take them: K_0, K_1, V_0, K_2, V_1,
// ...  A softmax thread owns a row: no shuffles.  O is rescaled only when a row's maximum has
// grown by more than 2^8 since its last scale; a row's sum is kept in f32 before P is rounded
// to the type of V, which is what the tensor cores take.  In f16 that loses weights below the
// type's least, so there m is taken 7 lower (P then reaches 2^15 at most): a weight is
// off by 2^-11 of itself or 2^-32 of the row's largest, and 32,768 small ones beside one large
// key by 2^-17 of the whole (unbiased, 2^-10).
//
// Bound: HBM.  A key tile of D = 256 is 64 KB, about 2,850 cycles of one SM's share of the
// bandwidth; its products take 1,024 and its exponentials (16 per SM and cycle) 512, both
// under the loads of the three tiles in the ring.
//
// Measured with 64 streams: 4,096 shared tokens 61 to 62 us for the whole call, 32,768 138 to 141 us
// (805 MB with the streams' own, 5.8 TB/s).  128-key tiles with Q in shared memory, which left no room
// for a third tile in the ring, took 76 us where this split first took 66; one copy warp needed
// 3,750 cycles a tile.
//
// Warps: 0, 6, 7 copies, 1 MMA issue, 2-5 softmax and epilogue (TMEM lanes 32 * (warp % 4)).
// Every wait is bounded; one that gives up sets the status word and the abort flag, the roles
// leave their loops, and the copies and products in flight are waited for (again with a limit)
// before the CTA goes on.  The rows of that unit get a sum of NaN, for which the join computes a
// row again on its own.
#pragma once
#include <cuda_bf16.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.cuh"
#include "tcgen05.cuh"

namespace ch {

struct PrefixArgs {
  const void *q, *k, *v;
  void *out;
  const int32_t *prefix_table, *table, *lens;
  long long qs, qh, os, oh;
  long long page, token, head, ts;
  uint32_t n, nq, nkv, group, shift, n_pages, cols, prefix, window;
  uint32_t from;  // first position read stream by stream
  float scale;
  uint32_t *status;
};

// positions stream b attends to: [lo, hi).  A length past what the table can hold is cut, but the
// window still ends where the stream does.  (prefix + table is below 2^32, as is prefix + length.)
CH_DEV void visible(const PrefixArgs &a, uint32_t b, uint32_t &lo, uint32_t &hi) {
  const uint32_t len = (uint32_t)max(a.lens[b], 0), end = a.prefix + len;
  hi = a.prefix + (uint32_t)min((unsigned long long)len, (unsigned long long)a.cols << a.shift);
  lo = a.window && end > a.window ? min(end - a.window, hi) : 0u;
}
// page and row inside it of position j of stream b; -1 when the page is not in the pool
CH_DEV int32_t page_of(const PrefixArgs &a, uint32_t b, uint32_t j, uint32_t &row) {
  const bool shared = j < a.prefix;
  const uint32_t i = shared ? j : j - a.prefix;
  row = i & ((1u << a.shift) - 1);
  const int32_t page = shared ? a.prefix_table[i >> a.shift] : a.table[b * a.ts + (i >> a.shift)];
  if (page < 0 || (uint32_t)page >= a.n_pages) {
    if (a.status) atomicOr(a.status, DEV_ERR_BAD_LIST);
    return -1;
  }
  return page;
}

// The shared prefix's parts in the caller's workspace: per split and kv head the n * group
// query rows (row b * group + g), unnormalised O, and the maximum (units of log2) and sum.
struct PrefixParts {
  float *o;             // [splits][n_kv][n * group][D]
  float2 *ml;           // [splits][n_kv][n * group]
  uint32_t max_splits;  // 0: the prefix is read stream by stream
};
namespace {
constexpr uint32_t kKeys = 64, kRows = 128;
constexpr int kTcThreads = 8 * 32, kSoft = 4 * 32;
constexpr uint32_t kTmemCols = 512, kQCol = 256, kSCol = 384;  // O: columns 0 .. D - 1; S: 384 and 448
constexpr int kMasks = 16;
template <typename T>
constexpr float kPrefixBias = std::is_same<T, __half>::value ? 7.f : 0.f;
constexpr float kGrow = 8.f;  // log2 of the growth of a maximum that O is not rescaled for

template <int D>
struct Tc {
  static constexpr uint32_t kPiece = D == 64 ? 8192 : 16384;
  static constexpr int kParts = kKeys * D * 2 / kPiece;  // pieces of a K tile, and of a V tile
  static constexpr int kDims = D / 64 / kParts;          // groups of 64 dims in a K piece
  static constexpr uint32_t kVKeys = kPiece / (2 * D);   // keys of a V piece
  static constexpr int kSlots = 13;
  static constexpr uint32_t kBytes = kSlots * kPiece;
  // The mask of tile i is written when K_{i-1}, first piece P (2i - 3) of the ring's order (P =
  // kParts), is on its way, for which piece P (2i - 3) - kSlots had to be taken.  The last V piece
  // up to there, place P (2j + 3) - 1, is of tile j = i - 3 - ceil((kSlots - 1) / 2P), so softmax is
  // done with tile j and may still be at the mask of tile j + 1: tiles j + 1 .. i need one each.
  static_assert(kMasks >= 3 + (kSlots + 2 * kParts - 2) / (2 * kParts), "masks in use at a time");
};

// instruction descriptor of kind::f16 with f32 sums: A K-major, B K-major or (mn) N-major
CH_DEV uint32_t idesc_of(uint32_t n, bool bf16, bool mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (mn ? 1u << 16 : 0u) | ((n >> 3) << 17) |
         ((kRows >> 4) << 24);
}
// V as the N-major operand B in the 128-byte swizzle: 64 dims x 8 keys are 1024 bytes; the
// next 8 keys lie `keys8` bytes on (stride offset), the next 64 dims `dims64` (leading offset)
CH_DEV uint64_t v_desc(uint32_t saddr, uint32_t dims64, uint32_t keys8) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(dims64 >> 4) << 16) | ((uint64_t)(keys8 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
struct TcBars {
  uint64_t full[13], empty[13], q_ready, s_full[2], p_ready[2], pv_done, done, mask_full[kMasks];
  uint32_t masks[kMasks][2], tmem_slot, abort_flag;
  uint32_t issued[13];  // 1 + the last piece on its way to a slot of the ring
};

// One unit: kv head h, row tile rt, key tiles [i0, i0 + nt) of the prefix, whose positions
// below zlo no stream sees.  Leaves the rows' parts at split `split`; false if it gave up, and
// then shared memory is not to be used again.  All threads of the CTA call it; sm
// (1024-byte aligned) is free before and after.  Each unit takes its tensor memory and gives it
// back, so the CTA keeps the permit to allocate: after giving that up it could not take any for
// its next unit.  (Taken once around all units, 32,768 shared tokens took 143 us instead of 138.)
template <typename T, int D>
CH_DEV bool prefix_unit(const PrefixArgs &a, const PrefixParts &w, const CUtensorMap &kmap, const CUtensorMap &vmap,
                        uint8_t *sm, TcBars &bars, uint32_t h, uint32_t rt, uint32_t split, uint32_t i0, uint32_t nt,
                        uint32_t zlo) {
  using C = Tc<D>;
  constexpr uint32_t kPiece = C::kPiece;
  const uint32_t ring = smem_u32(sm);
  uint64_t *full = bars.full, *empty = bars.empty, *s_full = bars.s_full, *p_ready = bars.p_ready,
           *mask_full = bars.mask_full;
  uint64_t &q_ready = bars.q_ready, &pv_done = bars.pv_done, &done = bars.done;
  auto &masks = bars.masks;
  volatile uint32_t &abort_flag = bars.abort_flag;
  // a V piece is boxes of vr keys, [D / 64][vr][64] each: 8 keys are 1024 bytes of a box, or
  // (pages of 8) a box of their own
  const uint32_t vr = min(1u << a.shift, C::kVKeys);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rows = a.n * a.group;

  if (tid == 0) {
    for (int s = 0; s < C::kSlots; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
    for (int s = 0; s < 2; s++) mbar_init(&s_full[s], 1), mbar_init(&p_ready[s], 4);
    for (int s = 0; s < kMasks; s++) mbar_init(&mask_full[s], 1);
    mbar_init(&q_ready, 4);
    mbar_init(&pv_done, 1);
    mbar_init(&done, 1);
    abort_flag = 0u;
    for (int s = 0; s < C::kSlots; s++) bars.issued[s] = 0u;
    fence_mbar_init();
  }
  if (warp == 1)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *(volatile uint32_t *)&bars.tmem_slot;

  // place in the ring's order of the first piece of K_i and of V_i
  auto k_seq = [&](uint32_t i) { return i ? C::kParts * (2 * i - 1) : 0u; };
  auto v_seq = [&](uint32_t i) { return C::kParts * (i + 1 < nt ? 2 * i + 2 : 2 * nt - 1); };

  if (warp == 0 || warp == 6 || (warp == 7 && C::kParts == 2)) {
    // ---- copies: warps 0 and 7 a half of each K tile, warp 6 V.  A box costs its warp about
    // 60 cycles to issue and a piece 300 to claim; one warp for all of it took 3,750 cycles a
    // tile of 16-token pages.  Lane l knows the page of keys [l * kr, (l + 1) * kr) ----
    const uint32_t ps = 1u << a.shift, kr = min(ps, kKeys), boxes = kKeys / kr;
    const bool is_v = warp == 6;
    auto look_up = [&](uint32_t i) {  // read a tile ahead, looked at when it is used
      const uint32_t j = (i0 + i) * kKeys + lane * kr;
      return i < nt && lane < (int)boxes && j < a.prefix ? a.prefix_table[j >> a.shift] : -1;
    };
    int32_t next = look_up(0);
    bool ok = true;
    for (uint32_t i = 0; i < nt && ok; i++) {
      const uint32_t j0 = (i0 + i) * kKeys;
      int32_t page = next;
      next = look_up(i + 1);
      const bool there = page >= 0 && (uint32_t)page < a.n_pages;
      if (!there) {
        if (a.status && lane < (int)boxes && j0 + lane * kr < a.prefix) atomicOr(a.status, DEV_ERR_BAD_LIST);
        page = (int32_t)a.n_pages;  // reads as zeros
      }
      if (warp == 0) {  // which keys are there, a lane per key of each half
        for (uint32_t half = 0; half < 2; half++) {
          const uint32_t key = half * 32 + lane;
          const bool in = __shfl_sync(0xffffffffu, there, key / kr);
          const uint32_t bits = __ballot_sync(0xffffffffu, in && j0 + key < a.prefix);
          if (lane == 0) masks[i % kMasks][half] = bits;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&mask_full[i % kMasks]);
      }
      for (uint32_t c = is_v ? 0 : warp / 7; c < (is_v ? C::kParts : warp / 7 + 1u) && ok; c++) {
        const uint32_t seq = (is_v ? v_seq(i) : k_seq(i)) + c, s = seq % C::kSlots;
        if (seq >= (uint32_t)C::kSlots) ok = tc_wait(&empty[s], ((seq / C::kSlots) - 1) & 1, &abort_flag, a.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[s], kPiece), bars.issued[s] = seq + 1;
        __syncwarp();
        if (is_v) {
          const uint32_t key = c * C::kVKeys + min((uint32_t)lane, C::kVKeys / vr - 1) * vr;
          const int32_t pg = __shfl_sync(0xffffffffu, page, key / kr);
          if (lane < (int)(C::kVKeys / vr))
            tma_load_5d(ring + s * kPiece + lane * vr * 2 * D, &vmap, 0, (int)((j0 + key) & (ps - 1)), 0, (int)h, pg,
                        &full[s]);
        } else {
          const uint32_t b = lane % boxes, g = lane / boxes;  // box, and its group of dims
          const int32_t pg = __shfl_sync(0xffffffffu, page, b);
          if (g < C::kDims)
            tma_load_4d(ring + s * kPiece + g * kKeys * 128 + b * kr * 128, &kmap, (c * C::kDims + g) * 64,
                        ps > kKeys ? (int)(j0 & (ps - 1)) : 0, (int)h, pg, &full[s]);
        }
      }
    }
  } else if (warp == 1) {
    // ---- products.  The warp walks the loop together and one elected lane issues: with the
    // branch on lane 0 around everything and the descriptors built per instruction, issue
    // (80 cycles an instruction) was slower than the products of N = 64 (49 cycles) ----
    const uint32_t issuer = elect_one();
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    const uint32_t s_idesc = idesc_of(kKeys, kBf16, false), o_idesc = idesc_of(D, kBf16, true);
    const uint32_t vs = vr == 8 ? 3 : vr == 16 ? 4 : vr == 32 ? 5 : 6;  // log2
    const uint64_t v_hi = v_desc(0, vr * 128, vr > 8 ? 1024u : 16u * D), k_hi = umma_desc_sw128(0);
    uint32_t slot = 0, phase = 0;
    bool ok = __all_sync(0xffffffffu, tc_wait(&q_ready, 0, &abort_flag, a.status));
    tc_fence_after();
    auto take = [&]() {  // waits for the next piece of the ring
      ok = ok && tc_wait(&full[slot], phase, &abort_flag, a.status);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      return (ring + slot * kPiece) >> 4;
    };
    auto pass = [&]() {
      if (++slot == (uint32_t)C::kSlots) slot = 0, phase ^= 1;
    };
    for (uint32_t i = 0; i <= nt && ok; i++) {
      if (i < nt) {
        // S_i lies where P_{i-2} lay
        if (i >= 2) ok = __all_sync(0xffffffffu, tc_wait(&pv_done, (i - 2) & 1, &abort_flag, a.status));
#pragma unroll
        for (int c = 0; c < C::kParts; c++) {
          const uint32_t at = take();
          if (!ok) break;
          if (issuer) {
            const uint32_t d = tmem + kSCol + (i & 1) * kKeys;
#pragma unroll
            for (int k = 0; k < 4 * C::kDims; k++)
              mma_ts(d, tmem + kQCol + (c * C::kDims * 4 + k) * 8, k_hi + (at + k / 4 * (kKeys * 8) + 2 * (k % 4)), s_idesc,
                     (c | k) != 0);
            commit(&empty[slot]);
            if (c + 1 == C::kParts) commit(&s_full[i & 1]);
          }
          __syncwarp();
          pass();
        }
      }
      if (i > 0 && ok) {
        const uint32_t j = i - 1;
        ok = __all_sync(0xffffffffu, tc_wait(&p_ready[j & 1], (j >> 1) & 1, &abort_flag, a.status));
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < C::kParts; c++) {
          const uint32_t at = take();
          if (!ok) break;
          if (issuer) {
            const uint32_t p = tmem + kSCol + (j & 1) * kKeys + c * (C::kVKeys / 2);
#pragma unroll
            for (uint32_t k = 0; k < C::kVKeys / 16; k++) {
              const uint32_t box = k * 16 >> vs, in = k * 16 & (vr - 1);
              mma_ts(tmem, p + k * 8, v_hi + (at + box * (vr * D / 8) + in * 8), o_idesc, (j | c | k) != 0);
            }
            commit(&empty[slot]);
            if (c + 1 == C::kParts) commit(&pv_done);
          }
          __syncwarp();
          pass();
        }
      }
    }
    if (issuer) commit(&done);  // every MMA issued (all of them, or those before an abort) is complete
  } else if (warp >= 2 && warp < 6) {
    // ---- softmax: thread = query row ----
    const uint32_t quad = warp & 3, row = quad * 32 + lane, row0 = rt * kRows;
    const uint32_t lanes = (quad * 32u) << 16;
    constexpr uint32_t kVecs = D / 8;  // 16-byte pieces of a row
    // this row of Q into tensor memory, 16 loads of 16 bytes in flight; a scale that is not
    // positive goes into it: below it is |scale|
    const uint32_t gr = row0 + row;
    const uint4 *q = gr < rows ? reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (gr / a.group) * a.qs +
                                                                 (h * a.group + gr % a.group) * a.qh)
                               : nullptr;
    const uint32_t q_keep = a.scale == 0.f ? 0u : 0xFFFFFFFFu, q_flip = a.scale < 0.f ? 0x80008000u : 0u;
    constexpr uint32_t kAt = kVecs < 16 ? kVecs : 16;
#pragma unroll 1
    for (uint32_t v0 = 0; v0 < kVecs; v0 += kAt) {
      uint4 x[kAt];
#pragma unroll
      for (uint32_t v = 0; v < kAt; v++) x[v] = q ? q[v0 + v] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (uint32_t v = 0; v < kAt; v += 8) {
        uint32_t r[32];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          r[4 * e] = (x[v + e].x & q_keep) ^ q_flip, r[4 * e + 1] = (x[v + e].y & q_keep) ^ q_flip;
          r[4 * e + 2] = (x[v + e].z & q_keep) ^ q_flip, r[4 * e + 3] = (x[v + e].w & q_keep) ^ q_flip;
        }
        tc_st32(tmem + kQCol + lanes + (v0 + v) * 4, r);
      }
    }
    tc_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&q_ready);

    uint32_t lo = 0;
    if (a.window && gr < rows) {
      uint32_t hi;
      visible(a, gr / a.group, lo, hi);
    }
    const float scale2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.44269504088896341f;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (uint32_t i = 0; i < nt; i++) {
      const uint32_t j0 = (i0 + i) * kKeys, scol = tmem + kSCol + (i & 1) * kKeys + lanes;
      ok = tc_wait(&s_full[i & 1], (i >> 1) & 1, &abort_flag, a.status) &&
           tc_wait(&mask_full[i % kMasks], (i / kMasks) & 1, &abort_flag, a.status);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      uint32_t s[2][32];
      tc_ld32(scol, s[0]);
      tc_ld32(scol + 32, s[1]);
      tc_wait_ld();
      uint32_t mask[2] = {masks[i % kMasks][0], masks[i % kMasks][1]};
      if (lo > j0) {  // hidden by the window
        const uint32_t hide = lo - j0;
        mask[0] &= hide >= 32 ? 0u : 0xFFFFFFFFu << hide;
        if (hide >= 32) mask[1] &= hide >= 64 ? 0u : 0xFFFFFFFFu << (hide - 32);
      }
      if (__any_sync(0xffffffffu, (mask[0] & mask[1]) != 0xFFFFFFFFu)) {
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (!((mask[c] >> e) & 1)) s[c][e] = 0xFF800000u;  // -inf
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 32; e++)
#pragma unroll
        for (int c = 0; c < 2; c++) top[(2 * e + c) & 3] = fmaxf(top[(2 * e + c) & 3], __uint_as_float(s[c][e]));
      const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale2;
      const bool grow = mx > m + kGrow || (m == -INFINITY && mx > -INFINITY);
      const float m1 = grow ? mx : m, ref = m1 == -INFINITY ? 0.f : m1;
      if (__any_sync(0xffffffffu, grow)) {
        const float keep = grow ? exp2_approx(m - ref) : 1.f;
        l *= keep;
        if (i > 0) {
          ok = tc_wait(&pv_done, (i - 1) & 1, &abort_flag, a.status);
          if (!__all_sync(0xffffffffu, ok)) break;
          tc_fence_after();
#pragma unroll 1
          for (uint32_t c = 0; c < D; c += 32) {
            uint32_t o[32];
            tc_ld32(tmem + lanes + c, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            tc_st32(tmem + lanes + c, o);
          }
        }
      }
      m = m1;
      const float low = ref - kPrefixBias<T>;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t p[32];
#pragma unroll
      for (int c = 0; c < 2; c++) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const float p0 = exp2_approx(fmaf(__uint_as_float(s[c][2 * e]), scale2, -low));
          const float p1 = exp2_approx(fmaf(__uint_as_float(s[c][2 * e + 1]), scale2, -low));
          sum[e & 1] += p0;
          sum[2 + (e & 1)] += p1;
          p[c * 16 + e] = pack2(p0, p1, static_cast<const T *>(nullptr));
        }
      }
      tc_st32(scol, p);
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tc_wait_st();
      // rows of V that no stream sees (past the prefix in its last page, before the first
      // visible position) are cleared: a weight of 0 must not meet stale bits
      const uint32_t z0 = zlo > j0 ? min(zlo - j0, kKeys) : 0u, z1 = a.prefix - j0 < kKeys ? a.prefix - j0 : kKeys;
      if (z0 > 0 || z1 < kKeys) {
        const uint32_t seq0 = v_seq(i);
        for (int c = 0; c < C::kParts; c++)
          ok = ok && tc_wait(&full[(seq0 + c) % C::kSlots], ((seq0 + c) / C::kSlots) & 1, &abort_flag, a.status);
        if (!__all_sync(0xffffffffu, ok)) break;
        const uint32_t n0 = z0, n1 = kKeys - z1;
        for (uint32_t x = tid - 64; x < (n0 + n1) * kVecs; x += kSoft) {
          const uint32_t z = x / kVecs, key = z < n0 ? z : z1 + (z - n0), v = x % kVecs;
          const uint32_t slot = (seq0 + key / C::kVKeys) % C::kSlots;
          const uint32_t in = key % C::kVKeys;
          *reinterpret_cast<uint4 *>(sm + slot * kPiece + in / vr * vr * 2 * D +
                                     ((v >> 3) * vr + in % vr) * 128 + (v & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[i & 1]);
    }
    // ---- this split's part ----
    ok = tc_wait(&done, 0, nullptr, a.status);
    tc_fence_after();
    ok = __all_sync(0xffffffffu, ok && !abort_flag);
    if (ok) {
      const size_t at = ((size_t)split * a.nkv + h) * rows + gr;
      if (gr < rows) w.ml[at] = make_float2(m - kPrefixBias<T>, l);
      {
        float *po = w.o + at * D;
#pragma unroll 1
        for (uint32_t c = 0; c < D; c += 32) {
          uint32_t o[32];
          tc_ld32(tmem + lanes + c, o);
          tc_wait_ld();
          if (gr < rows) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) st_global_32b(po + c + e, o + e);
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();  // every role done with tensor memory and the barriers
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
  // what is still on its way to shared memory or the barriers lands (normally long done): the
  // last copy into each slot and, unless a role gave up, the arrivals of the last products
  if (tid < C::kSlots && bars.issued[tid]) {
    const uint32_t parity = ((bars.issued[tid] - 1) / C::kSlots) & 1;
    if (!tc_wait(&full[tid], parity, nullptr, a.status) || (!abort_flag && !tc_wait(&empty[tid], parity, nullptr, a.status)))
      abort_flag = 1u;
  } else if (tid == 32 && !abort_flag && !tc_wait(&pv_done, (nt - 1) & 1, nullptr, a.status)) {
    abort_flag = 1u;
  }
  __syncthreads();
  if (abort_flag) return false;
  if (tid == 0) {  // the barriers' memory may be initialised again
    auto drop = [](uint64_t *bar) { asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory"); };
    for (int s = 0; s < C::kSlots; s++) drop(&full[s]), drop(&empty[s]);
    for (int s = 0; s < 2; s++) drop(&s_full[s]), drop(&p_ready[s]);
    for (int s = 0; s < kMasks; s++) drop(&mask_full[s]);
    drop(&q_ready), drop(&pv_done), drop(&done);
  }
  __syncthreads();
  return true;
}

// One layer's pool as a tensor of dim, token in the page, head and page (K: boxes of 64 dims
// of `rows` tokens), for V with the dims in groups of 64 (boxes of all dims); 128-byte swizzle.
cudaError_t pool_map(CUtensorMap *map, const void *pool, const PrefixArgs &a, uint32_t D, uint32_t rows, bool grouped) {
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn)
                                                                : nullptr;
  }();
  if (!encode) return cudaErrorNotSupported;
  // the stride of a dimension of one element is never used; torch may give any value there
  const cuuint64_t token = (cuuint64_t)a.token * 2;
  const cuuint64_t head = a.nkv > 1 ? (cuuint64_t)a.head * 2 : token, page = a.n_pages > 1 ? (cuuint64_t)a.page * 2 : token;
  const cuuint64_t dims4[4] = {D, 1ull << a.shift, a.nkv, a.n_pages}, strides4[3] = {token, head, page};
  const cuuint64_t dims5[5] = {64, 1ull << a.shift, D / 64, a.nkv, a.n_pages}, strides5[4] = {token, 128, head, page};
  const cuuint32_t box4[4] = {64, rows, 1, 1}, box5[5] = {64, rows, D / 64, 1, 1}, step[5] = {1, 1, 1, 1, 1};
  const CUresult r =
      encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, grouped ? 5 : 4, const_cast<void *>(pool), grouped ? dims5 : dims4,
             grouped ? strides5 : strides4, grouped ? box5 : box4, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorNotSupported;
}
}  // namespace

}  // namespace ch
