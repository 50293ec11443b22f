// prefix_tc.cuh -- the shared prefix of ch_prefix_attention on the 5th-generation tensor
// cores: every shared K and V row is read once for all streams.
//
// The query rows of one kv head -- `group` per stream, row b * group + g -- are the M = 128
// rows of a tile (a batch of 64 streams with two q heads per kv head fills it); a CTA takes
// one row tile and a run of the prefix's 128-key tiles, and per key tile
//   S (128 x 128) = Q K^T,   P = 2^(scale log2(e) S - m),   O (128 x D) += P V.
// Q stays in shared memory; K and V come by TMA from the pages (K: a box per page and 64
// dims, V: a box per page; 128-byte swizzle) through one ring of 16 KB pieces in the order the products take
// them: K_0, K_1, V_0, K_2, V_1, ...; S (two buffers), P (over its S, as the TMEM operand A)
// and O live in tensor memory (256 + 2 x 128 columns).  A softmax thread owns a row: no
// shuffles.  O is rescaled only when a row's maximum has grown by more than 2^8 since its
// last scale (P then stays below 2^8, exact in either type up to its rounding); a row's sum
// is kept in f32 before P is rounded.
//
// Bound: HBM.  A key tile of D = 256 is 128 KB, about 5,700 cycles of one SM's share of the
// bandwidth; its MMAs take 2,048 and its exponentials (16 per SM and cycle) 1,024, both
// under the next tile's loads.
//
// Warps: 0 copies, 1 MMA issue (lane 0), 2-5 softmax and epilogue (TMEM lanes 32 * (warp %
// 4)).  Every wait is bounded; one that gives up sets the status word and the abort flag,
// the roles leave their loops, and the MMA warp's last commit is waited for before tensor
// memory is released.
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

CH_DEV float to_f32(__half v) { return __half2float(v); }
CH_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// own tokens of stream b, limited to what its table can hold
CH_DEV uint32_t own_len(const PrefixArgs &a, uint32_t b) {
  const long long len = a.lens[b];
  return (uint32_t)min(max(len, 0ll), (long long)a.cols << a.shift);
}

CH_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
CH_DEV uint32_t pack2(float lo, float hi, const __half *) { return pack_half2(__float2half_rn(lo), __float2half_rn(hi)); }
CH_DEV uint32_t pack2(float lo, float hi, const __nv_bfloat16 *) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// positions stream b attends to: [lo, hi)
CH_DEV void visible(const PrefixArgs &a, uint32_t b, uint32_t &lo, uint32_t &hi) {
  hi = a.prefix + own_len(a, b);  // both below 2^31
  lo = a.window && hi > a.window ? hi - a.window : 0u;
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
constexpr uint32_t kKeys = 128, kRows = 128;
constexpr uint32_t kPiece = 16384;
constexpr int kTcThreads = 6 * 32, kSoft = 4 * 32;
constexpr uint32_t kTmemCols = 512, kSCol = 256;  // O: columns 0 .. D - 1; S: 256 and 384
constexpr int kMasks = 8;
constexpr float kGrow = 8.f;  // log2 of the growth of a maximum that O is not rescaled for

template <int D>
struct Tc {
  static constexpr int kParts = D / 64;  // pieces of a K tile (64 dims each) and of a V tile
  static constexpr uint32_t kVKeys = kPiece / (2 * D);  // keys of a V piece
  static constexpr int kSlots = D == 256 ? 9 : D == 128 ? 11 : 12;
  static constexpr uint32_t kOffRing = kRows * D * 2;
  static constexpr uint32_t kBytes = kOffRing + kSlots * kPiece;
};

CH_DEV void tma_load_5d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int u, int w, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
      "[%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(u), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
CH_DEV void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
// A from shared memory / from tensor memory
CH_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
CH_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
CH_DEV void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
CH_DEV void tc_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
CH_DEV void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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
CH_DEV void st_global_32b(float *p, const uint32_t *v) {  // 32 bytes, 32-byte aligned
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

struct TcBars {
  uint64_t full[12], empty[12], q_ready, s_full[2], p_ready[2], pv_done, done, mask_full[kMasks];
  uint32_t masks[kMasks][4], tmem_slot, abort_flag;
};

// One unit: kv head h, row tile rt, key tiles [i0, i0 + nt) of the prefix, whose positions
// below zlo no stream sees.  Leaves the rows' parts at split `split`.  All threads of the CTA
// call it; sm (1024-byte aligned) is free before and after.
template <typename T, int D>
CH_DEV void prefix_unit(const PrefixArgs &a, const PrefixParts &w, const CUtensorMap &kmap, const CUtensorMap &vmap,
                        uint8_t *sm, TcBars &bars, uint32_t h, uint32_t rt, uint32_t split, uint32_t i0, uint32_t nt,
                        uint32_t zlo) {
  using C = Tc<D>;
  const uint32_t sbase = smem_u32(sm), ring = sbase + C::kOffRing;
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
    for (int s = 0; s < 2; s++) mbar_init(&s_full[s], 1), mbar_init(&p_ready[s], kSoft);
    for (int s = 0; s < kMasks; s++) mbar_init(&mask_full[s], 1);
    mbar_init(&q_ready, kSoft);
    mbar_init(&pv_done, 1);
    mbar_init(&done, 1);
    abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *(volatile uint32_t *)&bars.tmem_slot;

  if (warp == 0) {
    // ---- copies.  Lane l of a tile holds the page of its keys [l * kr, (l + 1) * kr) ----
    const uint32_t ps = 1u << a.shift, kr = min(ps, kKeys), boxes = kKeys / kr;
    auto look_up = [&](uint32_t i) {
      const uint32_t j = i * kKeys + lane * kr;
      if (lane >= (int)boxes || j >= a.prefix) return -1;
      const int32_t page = a.prefix_table[j >> a.shift];
      if (page >= 0 && (uint32_t)page < a.n_pages) return page;
      if (a.status) atomicOr(a.status, DEV_ERR_BAD_LIST);
      return -1;
    };
    uint32_t seq = 0;
    bool ok = true;
    auto claim = [&]() {  // the next slot of the ring, its barrier armed
      const uint32_t s = seq % C::kSlots;
      if (seq >= (uint32_t)C::kSlots) ok = tc_wait(&empty[s], ((seq / C::kSlots) - 1) & 1, &abort_flag, a.status);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && lane == 0) mbar_arrive_expect_tx(&full[s], kPiece);
      __syncwarp();
      if (ok) seq++;
      return s;
    };
    // a page index past the pool reads as zeros
    int32_t page = look_up(i0), next = -1, prev = -1;
    for (uint32_t i = 0; i <= nt && ok; i++) {
      if (i < nt) {
        const uint32_t tile = i0 + i, j0 = tile * kKeys;
        next = i + 1 < nt ? look_up(tile + 1) : -1;
        // which keys are there: four per lane, put together to a word per eight lanes
        const int32_t mine = __shfl_sync(0xffffffffu, page, lane * 4 / kr);
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) bits |= (mine >= 0 && j0 + lane * 4 + e < a.prefix ? 1u : 0u) << e;
        bits <<= (lane & 7) * 4;
        bits |= __shfl_xor_sync(0xffffffffu, bits, 1);
        bits |= __shfl_xor_sync(0xffffffffu, bits, 2);
        bits |= __shfl_xor_sync(0xffffffffu, bits, 4);
        if ((lane & 7) == 0) masks[i % kMasks][lane >> 3] = bits;
        __syncwarp();
        if (lane == 0) mbar_arrive(&mask_full[i % kMasks]);
        for (int c = 0; c < C::kParts && ok; c++) {
          const uint32_t s = claim();
          if (ok && lane < (int)boxes)
            tma_load_4d(ring + s * kPiece + lane * kr * 128, &kmap, c * 64, ps > kKeys ? (int)(j0 & (ps - 1)) : 0, (int)h,
                        page >= 0 ? page : (int)a.n_pages, &full[s]);
        }
      }
      if (i > 0) {
        const uint32_t j0 = (i0 + i - 1) * kKeys;
        for (int c = 0; c < C::kParts && ok; c++) {
          const uint32_t s = claim();
          const uint32_t key = c * C::kVKeys + min((uint32_t)lane, C::kVKeys / vr - 1) * vr;
          const int32_t pg = __shfl_sync(0xffffffffu, prev, key / kr);
          if (ok && lane < (int)(C::kVKeys / vr))
            tma_load_5d(ring + s * kPiece + lane * vr * 2 * D, &vmap, 0, (int)((j0 + key) & (ps - 1)), 0, (int)h,
                        pg >= 0 ? pg : (int)a.n_pages, &full[s]);
        }
      }
      prev = page;
      page = next;
    }
    // the last copies land before the CTA may leave (normally long done)
    if (lane == 0)
      for (uint32_t j = seq > (uint32_t)C::kSlots ? seq - C::kSlots : 0; j < seq; j++)
        tc_wait(&full[j % C::kSlots], (j / C::kSlots) & 1, nullptr, a.status);
  } else if (warp == 1) {
    // ---- products ----
    if (lane == 0) {
      const uint32_t s_idesc = idesc_of(kKeys, std::is_same<T, __nv_bfloat16>::value, false);
      const uint32_t o_idesc = idesc_of(D, std::is_same<T, __nv_bfloat16>::value, true);
      uint32_t seq = 0;
      bool ok = tc_wait(&q_ready, 0, &abort_flag, a.status);
      auto take = [&]() {  // the next piece of the ring
        const uint32_t s = seq % C::kSlots;
        ok = ok && tc_wait(&full[s], (seq / C::kSlots) & 1, &abort_flag, a.status);
        tc_fence_after();
        seq++;
        return s;
      };
      for (uint32_t i = 0; i <= nt && ok; i++) {
        if (i < nt) {
          // S_i lies where P_{i-2} lay
          if (i >= 2) ok = tc_wait(&pv_done, (i - 2) & 1, &abort_flag, a.status);
          for (int c = 0; c < C::kParts && ok; c++) {
            const uint32_t s = take();
            if (!ok) break;
            const uint64_t qd = umma_desc_sw128(sbase + c * kRows * 128), kd = umma_desc_sw128(ring + s * kPiece);
#pragma unroll
            for (int k = 0; k < 4; k++)
              mma_ss(tmem + kSCol + (i & 1) * kKeys, qd + 2 * k, kd + 2 * k, s_idesc, (c | k) != 0);
            commit(&empty[s]);
          }
          if (ok) commit(&s_full[i & 1]);
        }
        if (i > 0 && ok) {
          const uint32_t j = i - 1;
          ok = tc_wait(&p_ready[j & 1], (j >> 1) & 1, &abort_flag, a.status);
          tc_fence_after();
          for (int c = 0; c < C::kParts && ok; c++) {
            const uint32_t s = take();
            if (!ok) break;
#pragma unroll
            for (uint32_t k = 0; k < C::kVKeys / 16; k++)
              mma_ts(tmem, tmem + kSCol + (j & 1) * kKeys + (c * C::kVKeys + k * 16) / 2,
                     v_desc(ring + s * kPiece + k * 16 / vr * vr * 2 * D + k * 16 % vr * 128, vr * 128,
                            vr > 8 ? 1024u : 16u * D),
                     o_idesc, (j | c | k) != 0);
            commit(&empty[s]);
          }
          if (ok) commit(&pv_done);
        }
      }
      commit(&done);  // every MMA issued (all of them, or those before an abort) is complete
    }
  } else if (warp < 6) {
    // ---- softmax: thread = query row ----
    const uint32_t quad = warp & 3, row = quad * 32 + lane, row0 = rt * kRows;
    const uint32_t lanes = (quad * 32u) << 16;
    constexpr uint32_t kVecs = D / 8;  // 16-byte pieces of a row
    // the warp's 32 rows of Q, all copies in flight together; lane l knows row l's place
    const uint32_t gr = row0 + row;
    const T *mine = gr < rows ? static_cast<const T *>(a.q) + (gr / a.group) * a.qs + (h * a.group + gr % a.group) * a.qh
                              : nullptr;
#pragma unroll 8
    for (uint32_t u = 0; u < kVecs; u++) {
      const uint32_t x = u * 32 + lane, v = x % kVecs, r = x / kVecs;
      const T *src = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), r));
      uint8_t *dst = sm + (v >> 3) * kRows * 128 + (quad * 32 + r) * 128 + (((v & 7) ^ (r & 7)) << 4);
      if (src)
        cp_async16(dst, src + v * 8);
      else
        *reinterpret_cast<uint4 *>(dst) = make_uint4(0, 0, 0, 0);
    }
    cp_async_wait_all();
    if (!(a.scale > 0.f)) {  // a scale that is not positive goes into Q: below it is |scale|
      __syncwarp();
      for (uint32_t u = 0; u < kVecs; u++) {
        const uint32_t x = u * 32 + lane, v = x % kVecs, r = x / kVecs;
        uint4 *q = reinterpret_cast<uint4 *>(sm + (v >> 3) * kRows * 128 + (quad * 32 + r) * 128 + ((v & 7) << 4));
        const uint32_t keep = a.scale < 0.f ? 0xFFFFFFFFu : 0u, flip = a.scale < 0.f ? 0x80008000u : 0u;
        *q = make_uint4((q->x & keep) ^ flip, (q->y & keep) ^ flip, (q->z & keep) ^ flip, (q->w & keep) ^ flip);
      }
    }
    fence_proxy_async();
    mbar_arrive(&q_ready);

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
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; c++) tc_ld32(scol + c * 32, s[c]);
      tc_wait_ld();
      uint32_t mask[4];
#pragma unroll
      for (int c = 0; c < 4; c++) mask[c] = masks[i % kMasks][c];
      if (lo > j0) {  // hidden by the window
        const uint32_t hide = lo - j0;
#pragma unroll
        for (int c = 0; c < 4; c++)
          if (hide >= 32u * c) mask[c] &= hide >= 32u * (c + 1) ? 0u : 0xFFFFFFFFu << (hide - 32u * c);
      }
      if (__any_sync(0xffffffffu, (mask[0] & mask[1] & mask[2] & mask[3]) != 0xFFFFFFFFu)) {
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (!((mask[c] >> e) & 1)) s[c][e] = 0xFF800000u;  // -inf
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 32; e++)
#pragma unroll
        for (int c = 0; c < 4; c++) top[c] = fmaxf(top[c], __uint_as_float(s[c][e]));
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
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        uint32_t p[32];
#pragma unroll
        for (int e = 0; e < 32; e++) {
          const uint32_t b0 = s[c + (e >> 4)][(2 * e) & 31], b1 = s[c + (e >> 4)][(2 * e + 1) & 31];
          const float p0 = exp2_approx(fmaf(__uint_as_float(b0), scale2, -ref));
          const float p1 = exp2_approx(fmaf(__uint_as_float(b1), scale2, -ref));
          sum[e & 1] += p0;
          sum[2 + (e & 1)] += p1;
          p[e] = pack2(p0, p1, static_cast<const T *>(nullptr));
        }
        tc_st32(scol + c * 16, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tc_wait_st();
      // rows of V that no stream sees (past the prefix in its last page, before the first
      // visible position) are cleared: a weight of 0 must not meet stale bits
      const uint32_t z0 = zlo > j0 ? min(zlo - j0, kKeys) : 0u, z1 = a.prefix - j0 < kKeys ? a.prefix - j0 : kKeys;
      if (z0 > 0 || z1 < kKeys) {
        const uint32_t seq0 = C::kParts * (i + 1 < nt ? 2 * i + 2 : 2 * nt - 1);
        for (int c = 0; c < C::kParts; c++)
          ok = ok && tc_wait(&full[(seq0 + c) % C::kSlots], ((seq0 + c) / C::kSlots) & 1, &abort_flag, a.status);
        if (!__all_sync(0xffffffffu, ok)) break;
        const uint32_t n0 = z0, n1 = kKeys - z1;
        for (uint32_t x = tid - 64; x < (n0 + n1) * kVecs; x += kSoft) {
          const uint32_t z = x / kVecs, key = z < n0 ? z : z1 + (z - n0), v = x % kVecs;
          const uint32_t slot = (seq0 + key / C::kVKeys) % C::kSlots;
          const uint32_t in = key % C::kVKeys;
          *reinterpret_cast<uint4 *>(sm + C::kOffRing + slot * kPiece + in / vr * vr * 2 * D +
                                     ((v >> 3) * vr + in % vr) * 128 + (v & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
      }
      tc_fence_before();
      mbar_arrive(&p_ready[i & 1]);
    }
    // ---- this split's part ----
    ok = tc_wait(&done, 0, nullptr, a.status);
    tc_fence_after();
    ok = __all_sync(0xffffffffu, ok && !abort_flag);
    if (ok) {
      const size_t at = ((size_t)split * a.nkv + h) * rows + gr;
      if (gr < rows) w.ml[at] = make_float2(m, l);
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
  if (tid == 0) {  // the barriers' memory may be initialised again
    auto drop = [](uint64_t *bar) { asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory"); };
    for (int s = 0; s < C::kSlots; s++) drop(&full[s]), drop(&empty[s]);
    for (int s = 0; s < 2; s++) drop(&s_full[s]), drop(&p_ready[s]);
    for (int s = 0; s < kMasks; s++) drop(&mask_full[s]);
    drop(&q_ready), drop(&pv_done), drop(&done);
  }
  __syncthreads();
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
