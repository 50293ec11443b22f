// chunk_tc.cuh -- ch_chunk_attention on the 5th-generation tensor cores.
//
// A unit is one kv head of one stream and the query rows of 2 x floor(128 / group) of its new
// tokens, row = token * group + q head: the M = 256 rows of a CTA pair (a cluster of two, rows 0 to
// 127 in the first).  Its keys are the 128-key tiles of the prefix, of the cached tokens and of the
// new ones that any of its rows sees, and per tile
//   S (256 x 128) = Q K^T,   P = 2^(scale log2(e) S - m),   O (256 x D) += P V
// with cta_group::2 products: each CTA loads half of the tile's keys for the first and half of the
// dims of V for the second, so a byte of K or V that reaches shared memory serves 256 rows.
// O (D columns), and S in two buffers with P over it, lie in tensor memory; Q and a ring of K and V
// tiles in shared memory, in the order the products take them: K_0, K_1, V_0, K_2, V_1, ...
//
// Two softmax threads own a row, 64 keys of a tile each: S of the tile after the next waits for the
// product of this P (it lies over P), so the way from S to P is to be short.  (A thread for each row,
// taking every other tile: 16,384 tokens 1.99 ms, so 1.79.)  O is rescaled only when a row's maximum
// has grown by more than 2^8 since its last scale; a row's sum is kept in f32 before P is rounded to
// the type of V, which is what the tensor cores take (in f16 P is 2^7 larger, so that small weights
// beside a large one do not fall below the type's range).
//
// All tiles of all units, laid end to end with a unit's start counted as some tiles, are cut
// into equal runs, one for each pair; a unit that is cut leaves (O, m, l) of each of its parts in the
// workspace, and chunk_join_kernel, already resident, adds them.
//
// Warps: 0 copies Q and K, 1 copies V, 2 issues the products (in the second CTA: tells the first that
// its copies have landed; in both it clears what of Q and V is to be zeros), 3 walks the units and looks pages up, 4 to 11 softmax and results (TMEM
// lanes 32 * (warp % 4); 8 to 11 the second half of the keys, and of O's columns).  Every wait is
// bounded; one that gives up sets the status word and the abort flag, the roles leave their loops,
// and what is in flight, the last copy into each slot among it, is waited for (again with a limit).
//
// A row that sees a value that is not finite, or whose tiles hold one, may come out NaN: rows that are not
// finite are settled by the join kernel (chunk_mend), which waits for nobody.
//
// Measured, at full clocks, of the products' 1,637 TFLOP/s: a prompt of 16,384 tokens, 16 q heads of
// 256 dims on 8, f16, 1,684 us (1,306 TFLOP/s; 1,937 us again and again, when the 1,000 W limit holds
// the clocks at 1,150 MHz); 64 prompts of 16 to 2,048 tokens in a window of 1,024, bf16, 788 us (820);
// 8,192 tokens, 32 q heads on 8, bf16: of 128 dims 622 us (885), of 64 dims 569 (483; half of the second
// product is zeros).  A tile's products take 2,048 cycles of 256 dims and 1,024 of 128, its way from S to
// P 2,450: below 256 dims, and where units are short, the softmax threads are what bounds it.
#pragma once
#include <cudaTypedefs.h>

#include <type_traits>

#include "chunk_attn.cuh"

namespace ch {
namespace {
constexpr uint32_t kKeys = 128, kRows = 128;  // keys of a tile; rows of a CTA
constexpr int kSoftWarps = 8, kTcThreads = (4 + kSoftWarps) * 32;
constexpr uint32_t kTmemCols = 512, kSCol = 256;  // O: columns 0 .. DV - 1; S: 256 and 384
// what a unit's start costs, in tiles (256-dim heads: 64 prompts 796 us with 3, 809 with 4, 814 with 6; 128-dim
// heads: 21 chunks 793 us with 2, 782 with 3, 788 with 5)
constexpr uint32_t kUnitCost = 3;
constexpr uint32_t kItems = 2;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kGrow = 8.f;  // log2 of the growth of a maximum that O is not rescaled for
template <typename T>
constexpr float kBias = std::is_same<T, __half>::value ? 7.f : 0.f;

template <int D>
struct Tc {
  static constexpr int kGroups = D / 64;             // groups of 64 dims
  static constexpr uint32_t kDv = D < 128 ? 128 : D;  // columns of O: 64 dims a CTA at least
  static constexpr int kVGroups = kDv / 128;         // groups of 64 dims in a CTA's half of V
  static constexpr uint32_t kQ = kRows * D * 2;
  static constexpr uint32_t kK = kKeys / 2 * D * 2, kV = kKeys * kDv;  // bytes of a CTA's half tile
  static constexpr uint32_t kPiece = kK > kV ? kK : kV;
  static constexpr int kSlots = D == 256 ? 5 : 11;
  static constexpr uint32_t kRecs = D == 256 ? 4 : 6;
  static constexpr uint32_t kMisc = kQ + kSlots * kPiece;
};

struct Item {  // a run of one unit's tiles
  ChunkStream s;
  uint32_t b, h, tok0, tok1;       // stream, kv head, the unit's new tokens [tok0, tok1)
  uint32_t p0, np, c0, nc, n0;     // first tile of each segment and how many tiles the first two have
  uint32_t k0, nt;                 // first tile of the run among the unit's, and how many
  uint32_t part;                   // 0: the whole unit; 1 + slot of its part in the workspace
};
struct Rec {  // a tile
  uint32_t seg, key0;  // segment (+ 4: every row of the unit sees every key of the tile), first key
  uint32_t z0, z1;     // keys [z0, z1) of the tile may be seen
  uint32_t mask[4];            // which keys are there
  uint32_t page[16];           // of every min(page size, 128) keys
};
template <int D>
struct TcShared {
  static constexpr int kSlots = Tc<D>::kSlots;
  static constexpr uint32_t kRecs = Tc<D>::kRecs;
  uint64_t full[kSlots], empty[kSlots], q_here, q_full, q_empty, s_full[2], p_ready[2], pv_done, o_full, o_free, done;
  alignas(16) Rec recs[kRecs];
  uint64_t item_full[kItems], item_empty[kItems], rec_full[kRecs], rec_empty[kRecs];
  Item items[kItems];
  // of the V tile in a slot: keys of a box; how many rows ahead of its keys and behind them are to be zeros (bits
  // 8 and 12 on); first and last 16 keys of use (bytes 2 and 3)
  uint32_t v_info[kSlots];
  uint32_t tmem_slot, abort_flag;
  uint64_t wait_ns;
  uint32_t dead[kSoftWarps];  // a wait of the warp gave up
  uint32_t fills[kSlots], q_loads;  // copies into a slot, and of Q, that were issued
  uint32_t bad[2];            // first item, and the one behind the last, with a row for chunk_mend
  float half[2][kRows];       // what the two threads of a row tell each other
};

// A unit cut between pairs: parts of it in the workspace, for the join (0: none).  Part slot 2 w is
// the end or the middle of a unit in pair w's run, 2 w + 1 the beginning of one.
struct Cut {
  uint32_t b, h, tok0, tok1, parts;
  uint32_t run_b, run_h, run_tok;  // the first unit of the pair's run
};
struct ChunkWork {
  Cut *cut;    // [pairs], by the pair that begins the unit
  uint2 *bad;  // [pairs][2 CTAs]: TcShared::bad
  float *o;    // [2 * pairs] parts of 256 rows (part_at)
  float2 *ml;  // [2 * pairs][256]: maximum (log2), sum
  uint32_t pairs;
};

// place of column c (a multiple of 8) of a row in a part of O: [D / 8][256][8], so that a warp stores
// 32 rows' 32 bytes in one piece
template <int D>
CH_DEV size_t part_at(uint32_t slot, uint32_t row, uint32_t c) {
  return (((size_t)slot * (D / 8) + c / 8) * (2 * kRows) + row) * 8 + c % 8;
}

// tiles of the unit of tokens [tok0, tok1)
struct Tiles {
  uint32_t p0, np, c0, nc, n0, nn;
  CH_DEV uint32_t all() const { return np + nc + nn; }
};
CH_DEV Tiles tiles_of(const ChunkArgs &a, const ChunkStream &s, uint32_t tok0, uint32_t tok1) {
  const ChunkLow lo = chunk_low(a, s, s.before + (a.parents ? 0u : tok0));
  auto tiles = [](uint32_t from, uint32_t to, uint32_t &first) {
    first = from / kKeys;
    return to > from ? (to + kKeys - 1) / kKeys - first : 0u;
  };
  Tiles t;
  t.np = tiles(lo.prefix, a.prefix, t.p0);
  t.nc = tiles(lo.cached, s.cached, t.c0);
  t.nn = tiles(lo.fresh, tok1, t.n0);
  return t;
}

CH_DEV void mma2_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
CH_DEV void mma2_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// arrive on `bar` in both CTAs once every product issued so far is complete
CH_DEV void commit2(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((unsigned short)3)
      : "memory");
}
// Arrive on the first CTA's barrier.  What it announces is in tensor memory (tcgen05.wait, fence) or
// was written by copies, so it takes no release of the cluster: that waits for every access of the
// thread in flight (16,384 tokens took 2.6 ms with it, 2.0 without).  The zeros that threads of the second
// CTA write into Q and V are announced by mbar_arrive_cluster, and waited for by an acquire of the cluster.
CH_DEV void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// instruction descriptor of kind::f16 with f32 sums, M = 256: A K-major, B K-major or (mn) N-major
CH_DEV uint32_t idesc2(uint32_t n, bool bf16, bool mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((2 * kRows >> 4) << 24);
}
// V as the N-major operand B in the 128-byte swizzle: 64 dims x 8 keys are 1024 bytes; the
// next 8 keys lie `keys8` bytes on (stride offset), the next 64 dims `dims64` (leading offset)
CH_DEV uint64_t v_desc(uint32_t saddr, uint32_t dims64, uint32_t keys8) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(dims64 >> 4) << 16) | ((uint64_t)(keys8 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// bits [lo, hi) of a word, for numbers that may lie outside 0..32
CH_DEV uint32_t bits_of(int lo, int hi) {
  lo = max(lo, 0), hi = min(hi, 32);
  if (hi <= lo) return 0u;
  return (hi == 32 ? 0xFFFFFFFFu : (1u << hi) - 1u) & ~((1u << lo) - 1u);
}

// barrier `id` of 64 threads, the two warps of 32 rows; pair_any: whether `p` holds in one of them
CH_DEV void pair_sync(uint32_t id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
CH_DEV bool pair_any(uint32_t id, bool p) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, 64, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)p), "r"(id)
      : "memory");
  return r != 0;
}
template <typename T, int D>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTcThreads, 1)
    chunk_tc_kernel(const __grid_constant__ ChunkArgs a, const ChunkWork w, const __grid_constant__ CUtensorMap qmap,
                    const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const __grid_constant__ CUtensorMap kpmap, const __grid_constant__ CUtensorMap vpmap) {
  using C = Tc<D>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t sm[];
  TcShared<D> &sh = *reinterpret_cast<TcShared<D> *>(sm + C::kMisc);
  constexpr uint32_t kRecs = C::kRecs;
  const uint32_t ring = smem_u32(sm) + C::kQ;
  volatile uint32_t *abort = &sh.abort_flag;
  // The limit of a wait is a parameter, or looked up in shared memory once the wait is not over at once: the
  // loops' speed hangs on the code around them (8,192 tokens, 64-dim heads 569 us with the first, 690 with
  // the second; 128 dims 671 and 621, 256 dims 430 and 414).
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if constexpr (D == 64) return tc_wait(bar, parity, abort, a.status, false, a.wait_ns);
    if (mbar_try_wait(bar, parity)) return true;
    return tc_wait(bar, parity, abort, a.status, false, *(volatile uint64_t *)&sh.wait_ns);
  };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), pair = blockIdx.x >> 1;
  const uint32_t tpt = kRows / a.group;  // tokens of a CTA

  if (tid == 0) {
    const uint32_t ctas = rank == 0 ? 2 : 1;  // the first CTA waits for the copies of both
    for (int s = 0; s < C::kSlots; s++) mbar_init(&sh.full[s], ctas), mbar_init(&sh.empty[s], 1), sh.fills[s] = 0u;
    mbar_init(&sh.q_here, 1), mbar_init(&sh.q_full, 1), mbar_init(&sh.q_empty, 1);
    for (int s = 0; s < 2; s++) mbar_init(&sh.s_full[s], 1), mbar_init(&sh.p_ready[s], 2 * kSoftWarps);
    mbar_init(&sh.pv_done, 1), mbar_init(&sh.o_full, 1), mbar_init(&sh.o_free, 2 * kSoftWarps), mbar_init(&sh.done, 1);
    for (int s = 0; s < kSoftWarps; s++) sh.dead[s] = 0u;
    sh.bad[0] = ~0u, sh.bad[1] = 0u;
    for (uint32_t s = 0; s < kItems; s++) mbar_init(&sh.item_full[s], 1), mbar_init(&sh.item_empty[s], 3 + kSoftWarps);
    for (uint32_t s = 0; s < kRecs; s++) mbar_init(&sh.rec_full[s], 1), mbar_init(&sh.rec_empty[s], 2 + kSoftWarps);
    sh.abort_flag = 0u, sh.q_loads = 0u, sh.wait_ns = a.wait_ns;
    fence_mbar_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }

  grid_dep_wait();  // the kernel in front may still be running
  // ---- what all units cost, and where this pair's run starts: the same sums in every CTA ----
  unsigned long long *sums = reinterpret_cast<unsigned long long *>(sm);  // (before the first copy)
  uint32_t *begin = reinterpret_cast<uint32_t *>(sm + 8 * (kTcThreads / 32));
  // a thread takes a stream or several; a warp one, where there are enough (with both this and the start
  // of the run found by a warp's lanes together, 16,384 tokens of 16 q heads on one kv head take 1,530 us;
  // unit after unit by one thread 1,670)
  const bool by_warp = a.n <= kTcThreads / 32;
  const uint32_t per = (a.n + kTcThreads - 1) / kTcThreads;
  const uint32_t b0 = by_warp ? min(a.n, (uint32_t)warp) : min(a.n, tid * per), b1 = min(a.n, b0 + per);
  auto stream_cost = [&](uint32_t b, uint32_t u, uint32_t step) {  // of one kv head, of units u, u + step, ...
    const ChunkStream s = chunk_stream(a, b);
    unsigned long long c = 0;
    for (uint32_t t = u * 2 * tpt; t < s.count; t += step * 2 * tpt)
      c += kUnitCost + tiles_of(a, s, t, min(s.count, t + 2 * tpt)).all();
    return c;
  };
  unsigned long long mine = 0, cost = 0;  // cost: of the thread's last stream
  if (by_warp) {
    if (b0 < b1) cost = stream_cost(b0, lane, 32);
#pragma unroll
    for (int o = 16; o; o >>= 1) cost += __shfl_xor_sync(0xffffffffu, cost, o);
    if (lane == 0) mine = cost * a.nkv;
  } else {
    for (uint32_t b = b0; b < b1; b++) mine += (cost = stream_cost(b, 0, 1)) * a.nkv;
  }
  unsigned long long at = mine, total = 0;  // at: cost of the streams before this thread's
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += u;
  }
  if (lane == 31) sums[warp] = at;
  if (tid == 0) *begin = a.n;
  if (blockIdx.x == 0) chunk_report(a);
  __syncthreads();
  at -= mine;
  for (int i = 0; i < kTcThreads / 32; i++) {
    if (i < warp) at += sums[i];
    total += sums[i];
  }
  const unsigned long long run = (total + w.pairs - 1) / w.pairs;
  const unsigned long long first = run * pair, last = min(first + run, total);
  __syncthreads();
  unsigned long long *found = sums;  // where the stream of the run's start begins, and its cost
  if (first < last && at <= first && first < at + mine) {
    uint32_t b = b0;
    if (per > 1)
      for (; at + (cost = stream_cost(b, 0, 1)) * a.nkv <= first; b++) at += cost * a.nkv;
    *begin = b;
    found[0] = at, found[1] = cost;
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();  // barriers initialised and tensor memory taken in both CTAs
  tc_fence_after();
  grid_dep_launch();
  const uint32_t tmem = *(volatile uint32_t *)&sh.tmem_slot;
  const uint32_t run_b = *begin;
  const unsigned long long run_at = found[0], run_cost = found[1];
  fence_proxy_async();
  __syncthreads();  // (read before the first copy)

  if (warp == 3) {
    // ---- units and tiles of the run ----
    Cut cut{};
    uint32_t n_items = 0, n_recs = 0;
    bool ok = true;
    unsigned long long x = run_at;  // start of the unit looked at
    for (uint32_t b = run_b; b < a.n && x < last && ok; b++) {
      const ChunkStream s = chunk_stream(a, b);
      uint32_t h = 0, t0 = 0;
      if (b == run_b) {  // the run starts in it; units that end before are left out, 32 at a time
        h = (uint32_t)((first - x) / run_cost);
        x += h * run_cost;
        for (uint32_t out = 32; out == 32 && t0 < s.count;) {
          const uint32_t t = t0 + lane * 2 * tpt;
          const uint32_t c = t < s.count ? kUnitCost + tiles_of(a, s, t, min(s.count, t + 2 * tpt)).all() : 0u;
          uint32_t end = c;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += u;
          }
          out = __popc(__ballot_sync(0xffffffffu, c && x + end <= first));
          if (out) x += __shfl_sync(0xffffffffu, end, out - 1);
          t0 += out * 2 * tpt;
        }
      }
      for (; h < a.nkv && x < last && ok; h++, t0 = 0) {
        for (uint32_t t = t0; t < s.count && x < last && ok; t += 2 * tpt) {
          const uint32_t tok1 = min(s.count, t + 2 * tpt);
          const Tiles u = tiles_of(a, s, t, tok1);
          const uint32_t all = u.all();
          const unsigned long long k_at = x + kUnitCost;  // place of its first tile
          const uint32_t k0 = first > k_at ? (uint32_t)min(first - k_at, (unsigned long long)all) : 0u;
          const uint32_t k1 = last > k_at ? (uint32_t)min(last - k_at, (unsigned long long)all) : 0u;
          x = k_at + all;
          if (k1 <= k0) continue;
          const uint32_t slot = n_items % kItems;
          if (n_items >= kItems) ok = wait(&sh.item_empty[slot], (n_items / kItems - 1) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          Item it{s, b, h, t, tok1, u.p0, u.np, u.c0, u.nc, u.n0, k0, k1 - k0, 0u};
          if (k0 > 0)
            it.part = 1 + 2 * pair;
          else if (k1 < all) {
            it.part = 2 + 2 * pair;
            cut.b = b, cut.h = h, cut.tok0 = t, cut.tok1 = tok1, cut.parts = 1u + (uint32_t)((x - 1) / run) - pair;
          }
          if (n_items == 0) cut.run_b = b, cut.run_h = h, cut.run_tok = t;
          if (lane == 0) {
            sh.items[slot] = it;
            mbar_arrive(&sh.item_full[slot]);
          }
          __syncwarp();
          n_items++;
          // its tiles; a page is looked up one tile before it is used
          const ChunkLow lo = chunk_low(a, s, s.before + (a.parents ? 0u : t));
          const ChunkLow high = a.parents && a.window ? ChunkLow{~0u, ~0u, ~0u} : chunk_low(a, s, s.before + tok1 - 1);
          const uint32_t pk = min(1u << a.shift, kKeys), pages = kKeys / pk;
          auto seg_of = [&](uint32_t k, uint32_t &key0) {
            if (k < u.np) {
              key0 = (u.p0 + k) * kKeys;
              return 0u;
            }
            if (k < u.np + u.nc) {
              key0 = (u.c0 + k - u.np) * kKeys;
              return 1u;
            }
            key0 = (u.n0 + k - u.np - u.nc) * kKeys;
            return 2u;
          };
          auto end_of = [&](uint32_t seg) { return seg == 0 ? a.prefix : seg == 1 ? s.cached : tok1; };
          auto low_of = [&](uint32_t seg) { return seg == 0 ? lo.prefix : seg == 1 ? lo.cached : lo.fresh; };
          // this lane's page of a tile: one that the unit's rows see something of (those ahead of a window may be gone)
          auto in_use = [&](uint32_t seg, uint32_t key0) {
            const uint32_t j = key0 + lane * pk;
            return seg < 2 && lane < (int)pages && j < end_of(seg) && j + pk > low_of(seg);
          };
          auto look_up = [&](uint32_t k) {
            uint32_t key0;
            const uint32_t seg = seg_of(k, key0), j = key0 + lane * pk;
            if (!in_use(seg, key0)) return -1;
            return seg == 0 ? a.prefix_table[j >> a.shift] : a.table[b * a.ts + (j >> a.shift)];
          };
          int32_t next = look_up(k0);
          for (uint32_t k = k0; k < k1; k++) {
            uint32_t key0;
            const uint32_t seg = seg_of(k, key0), end = end_of(seg);
            const uint32_t low = low_of(seg);
            const int32_t page = next;
            if (k + 1 < k1) next = look_up(k + 1);
            const uint32_t r = n_recs % kRecs;
            if (n_recs >= kRecs) ok = wait(&sh.rec_empty[r], (n_recs / kRecs - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const bool there = seg == 2 || (page >= 0 && (uint32_t)page < a.n_pages);
            if (!there && in_use(seg, key0) && a.status) atomicOr(a.status, DEV_ERR_BAD_LIST);
            // (the last token sees from high.* on, the first one up to itself)
            const bool all_in = seg < 2 ? key0 + kKeys <= end : !a.parents && key0 + kKeys <= t + 1;
            const bool all_see = all_in && (seg == 0 ? high.prefix : seg == 1 ? high.cached : high.fresh) <= key0 &&
                                 __all_sync(0xffffffffu, there || lane >= (int)pages);
            Rec &rec = sh.recs[r];
            if (lane < 16) rec.page[lane] = there ? (uint32_t)page : a.n_pages;  // past the pool: reads as zeros
#pragma unroll
            for (int c4 = 0; c4 < 4; c4++) {
              const uint32_t key = c4 * 32 + lane;
              const bool in = __shfl_sync(0xffffffffu, there, key / pk);
              const uint32_t bits = __ballot_sync(0xffffffffu, in && key0 + key < end);
              if (lane == 0) rec.mask[c4] = bits;
            }
            if (lane == 0) {
              rec.seg = seg + (all_see ? 4 : 0), rec.key0 = key0;
              rec.z0 = low > key0 ? low - key0 : 0u;
              rec.z1 = min(end - key0, kKeys);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.rec_full[r]);
            n_recs++;
          }
        }
      }
    }
    // the end: an item without tiles
    if (ok) {
      const uint32_t slot = n_items % kItems;
      if (n_items >= kItems) ok = wait(&sh.item_empty[slot], (n_items / kItems - 1) & 1);
      if (__all_sync(0xffffffffu, ok) && lane == 0) {
        sh.items[slot].nt = 0;
        mbar_arrive(&sh.item_full[slot]);
      }
    }
    if (rank == 0 && lane == 0) w.cut[pair] = cut;
  } else {
    // every other role walks the items
    uint32_t n = 0;
    Item it;
    auto next_item = [&]() {  // false: the run is over, or a wait gave up
      const uint32_t slot = n % kItems;
      const bool ok = __all_sync(0xffffffffu, wait(&sh.item_full[slot], (n / kItems) & 1));
      if (!ok) return false;
      it = sh.items[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.item_empty[slot]);
      n++;
      return it.nt != 0;
    };
    // place in the ring's order of K_i and of V_i of the item whose first piece has place `base`
    auto k_seq = [&](uint32_t i) { return i ? 2 * i - 1 : 0u; };
    auto v_seq = [&](uint32_t i) { return i + 1 < it.nt ? 2 * i + 2 : 2 * it.nt - 1; };
    uint32_t base = 0, recs = 0;
    // The rows of Q behind the unit's last are zeros: products of zeros take less power, and where few
    // rows are of use the clocks follow from it (64 trees of 16 nodes, again and again: 324 us, so 280).
    uint32_t zero_from = kRows;  // rows from here on are zeros already
    auto clear_q = [&]() {       // by the warp that tells that Q is here
      const uint32_t tok = min(it.tok0 + rank * tpt, it.tok1), used = min(it.tok1 - tok, tpt) * a.group;
      if (used) zero_from = min(max(zero_from, tpt * a.group), kRows);  // the copy has written the others
      if (used >= zero_from) return;
      for (int g = 0; g < C::kGroups; g++)
        for (uint32_t x = used * 8 + lane; x < zero_from * 8; x += 32)
          *reinterpret_cast<uint4 *>(sm + g * kRows * 128 + x * 16) = make_uint4(0, 0, 0, 0);
      zero_from = used;
      fence_proxy_async();
      __syncwarp();
    };

    // Rows of V that no row of the unit sees but are in the product, up to 15 ahead of its keys and
    // behind them, are zeros: a weight of 0 must not meet stale bits.  (By the same warp, ahead of its wait
    // for P: by the softmax warps it was on the way from S to P.)
    auto clear_v = [&](uint32_t slot, uint32_t info) {
      const uint32_t vr = info & 0xFF, y0 = info >> 8 & 15, y1 = info >> 12 & 15, z0 = (info >> 16 & 0xFF) * 16, z1 = (info >> 24) * 16 - y1;
      constexpr uint32_t kVecs = C::kDv / 16;  // 16-byte pieces of a key's dims
      for (uint32_t x = lane; x < (y0 + y1) * kVecs; x += 32) {
        const uint32_t y = x / kVecs, v = x % kVecs, key = y < y0 ? z0 + y : z1 + (y - y0);
        *reinterpret_cast<uint4 *>(sm + C::kQ + slot * C::kPiece + key / vr * vr * C::kDv + ((v >> 3) * vr + key % vr) * 128 +
                                   (v & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async();
      __syncwarp();
    };

    if (warp == 0 || warp == 1) {
      // ---- copies of K (this CTA's 64 keys of a tile) and Q, and of V (its half of the dims) ----
      const bool is_v = warp == 1;
      const uint32_t ps = 1u << a.shift, pk = min(ps, kKeys), kb = min(ps, kKeys / 2);
      uint32_t loaded_q = 0;
      bool ok = true;
      auto load_q = [&](uint32_t row0) {
        if (lane == 0) {
          if (it.tok0 + rank * tpt < it.tok1) {
            mbar_arrive_expect_tx(&sh.q_here, C::kGroups * tpt * a.group * 128);
            for (int g = 0; g < C::kGroups; g++)
              tma_load_3d(sm + g * kRows * 128, &qmap, g * 64, (int)(it.h * a.group), (int)(row0 + it.tok0 + rank * tpt), &sh.q_here);
          } else {  // no row of this CTA's
            mbar_arrive(&sh.q_here);
          }
        }
        loaded_q++;
        __syncwarp();
      };
      for (uint32_t k = 0; ok && next_item(); k++) {
        const uint32_t row0 = it.s.first;
        if (!is_v && k == 0) load_q(row0);
        for (uint32_t i = 0; i < it.nt && ok; i++, recs++) {
          const uint32_t r = recs % kRecs;
          ok = wait(&sh.rec_full[r], (recs / kRecs) & 1);
          const uint32_t seq = base + (is_v ? v_seq(i) : k_seq(i)), s = seq % C::kSlots;
          if (ok && seq >= (uint32_t)C::kSlots) ok = wait(&sh.empty[s], (seq / C::kSlots - 1) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const Rec &rec = sh.recs[r];
          const uint32_t seg = rec.seg & 3, key0 = rec.key0, dst = ring + s * C::kPiece;
          if (lane == 0) {
            if (is_v)
              sh.v_info[s] = (seg == 2 ? kKeys : pk) | (rec.z0 & 15) << 8 | (-rec.z1 & 15) << 12 | rec.z0 / 16 << 16 | (rec.z1 + 15) / 16 << 24;
            sh.fills[s] = seq / C::kSlots + 1;
            mbar_arrive_expect_tx(&sh.full[s], is_v ? C::kV : C::kK);
          }
          __syncwarp();
          if (is_v) {
            if (seg == 2) {
              if (lane == 0) tma_load_4d(dst, &vmap, 0, (int)(row0 + key0), (int)(rank * C::kVGroups), (int)it.h, &sh.full[s]);
            } else if (lane < (int)(kKeys / pk)) {
              tma_load_5d(dst + lane * pk * C::kDv, &vpmap, 0, (int)((key0 + lane * pk) & (ps - 1)), (int)(rank * C::kVGroups),
                          (int)it.h, (int)rec.page[lane], &sh.full[s]);
            }
          } else {
            const uint32_t half = rank * (kKeys / 2);
            if (seg == 2) {
              if (lane == 0) tma_load_4d(dst, &kmap, 0, (int)(row0 + key0 + half), 0, (int)it.h, &sh.full[s]);
            } else {
              const uint32_t boxes = kKeys / 2 / kb, bx = lane % boxes, g = lane / boxes;
              const uint32_t key = half + bx * kb;
              if (g < (boxes == 1 ? 1u : (uint32_t)C::kGroups))
                tma_load_5d(dst + g * (kKeys / 2 * 128) + bx * kb * 128, &kpmap, 0, (int)((key0 + key) & (ps - 1)), (int)g,
                            (int)it.h, (int)rec.page[key / pk], &sh.full[s]);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.rec_empty[r]);
          // Q of a later item behind its first K, which finds room before Q does
          if (!is_v && i == 0 && k > 0) {
            ok = __all_sync(0xffffffffu, wait(&sh.q_empty, (k - 1) & 1));
            if (!ok) break;
            load_q(row0);
          }
        }
        base += 2 * it.nt;
      }
      if (!is_v && lane == 0) sh.q_loads = loaded_q;
    } else if (warp == 2 && rank == 1) {
      // ---- this CTA's copies have landed: tell the first CTA ----
      const uint32_t full0 = map_shared(smem_u32(sh.full), 0), q_full0 = map_shared(smem_u32(&sh.q_full), 0);
      bool ok = true;
      for (uint32_t k = 0; ok && next_item(); k++) {
        ok = __all_sync(0xffffffffu, wait(&sh.q_here, k & 1));
        if (ok) clear_q();
        if (ok && lane == 0) mbar_arrive_cluster(q_full0);
        for (uint32_t i = 0; ok && i < 2 * it.nt; i++, base++) {
          const uint32_t slot = base % C::kSlots;
          ok = __all_sync(0xffffffffu, wait(&sh.full[slot], (base / C::kSlots) & 1));
          if (!ok) break;
          const bool is_v = i + 1 == 2 * it.nt || (i > 0 && i % 2 == 0);
          const uint32_t info = is_v ? *(volatile uint32_t *)&sh.v_info[slot] : 0u;
          if (info & 0xFF00) clear_v(slot, info);
          if (lane == 0) {
            if (info & 0xFF00) mbar_arrive_cluster(full0 + slot * 8);
            else arrive_remote(full0 + slot * 8);
          }
        }
      }
      __syncwarp();
    } else if (warp == 2) {
      // ---- products: the warp walks the loop together and one elected lane issues ----
      const uint32_t issuer = elect_one();
      const uint32_t s_idesc = idesc2(kKeys, kBf16, false), o_idesc = idesc2(C::kDv, kBf16, true);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(sm)), k_hi = umma_desc_sw128(0);
      uint32_t g0 = 0, slot = 0, phase = 0;
      uint32_t v_rows = 0, v_at[kKeys / 16];  // how V lies in a slot: keys of a box, and where each 16 keys begin
      uint64_t v_hi = 0;
      bool ok = true;
      auto take = [&]() {  // waits for the next piece of the ring, in both CTAs
        ok = __all_sync(0xffffffffu, ok && wait(&sh.full[slot], phase));
        tc_fence_after();
        return (ring + slot * C::kPiece) >> 4;
      };
      auto pass = [&]() {
        if (issuer) commit2(&sh.empty[slot]);
        __syncwarp();
        if (++slot == (uint32_t)C::kSlots) slot = 0, phase ^= 1;
      };
      for (uint32_t k = 0; ok && next_item(); k++) {
        ok = __all_sync(0xffffffffu, wait(&sh.q_here, k & 1));
        if (ok) clear_q();
        ok = __all_sync(0xffffffffu, ok && wait(&sh.q_full, k & 1));
        if (ok) (void)mbar_try_wait_cluster(&sh.q_full, k & 1);  // (it is over: acquires the second CTA's zeros)
        for (uint32_t i = 0; i <= it.nt && ok; i++) {
          const uint32_t g = g0 + i;
          if (i < it.nt) {
            // S_g lies where P_{g-2} lay, whose product was issued before: the tensor cores take the
            // products of a thread in order (waiting for it here left them idle 500 cycles a tile)
            const uint32_t from = take();
            if (!ok) break;
            if (issuer) {
              const uint32_t d = tmem + kSCol + (g & 1) * kKeys;
#pragma unroll
              for (int c = 0; c < D / 16; c++)
                mma2_ss(d, q_desc + c / 4 * (kRows * 8) + 2 * (c % 4), k_hi + (from + c / 4 * (kKeys / 2 * 8) + 2 * (c % 4)), s_idesc,
                        c != 0);
              commit2(&sh.s_full[g & 1]);
              if (i + 1 == it.nt) commit2(&sh.q_empty);
            }
            pass();
          }
          if (i > 0 && ok) {
            const uint32_t gj = g - 1;
            const uint32_t from = take();
            const uint32_t info = *(volatile uint32_t *)&sh.v_info[slot], c0 = info >> 16 & 0xFF, c1 = info >> 24;
            if (ok && (info & 0xFF00)) {
              (void)mbar_try_wait_cluster(&sh.full[slot], phase);  // (it is over: acquires the second CTA's zeros)
              clear_v(slot, info);
            }
            if (const uint32_t vr = info & 0xFF; vr != v_rows) {
              v_rows = vr;
              v_hi = v_desc(0, vr * 128, vr > 8 ? 1024u : 8u * C::kDv);
#pragma unroll
              for (uint32_t c = 0; c < kKeys / 16; c++) v_at[c] = c * 16 / vr * (vr * C::kDv / 16) + c * 16 % vr * 8;
            }
            if (ok && i == 1 && k > 0) ok = wait(&sh.o_free, (k - 1) & 1);
            ok = __all_sync(0xffffffffu, ok && wait(&sh.p_ready[gj & 1], (gj >> 1) & 1));
            tc_fence_after();
            if (!ok) break;
            if (issuer) {
              const uint32_t p = tmem + kSCol + (gj & 1) * kKeys;
              if (info >> 16 == (kKeys / 16) << 8) {
#pragma unroll
                for (uint32_t c = 0; c < kKeys / 16; c++) mma2_ts(tmem, p + c * 8, v_hi + (from + v_at[c]), o_idesc, (i - 1) | c);
              } else {  // keys that no row sees are left out, 16 at a time
#pragma unroll
                for (uint32_t c = 0; c < kKeys / 16; c++)
                  if (c >= c0 && c < c1) mma2_ts(tmem, p + c * 8, v_hi + (from + v_at[c]), o_idesc, (i - 1) | (c - c0));
              }
              commit2(&sh.pv_done);
              if (i == it.nt) commit2(&sh.o_full);
            }
            pass();
          }
        }
        g0 += it.nt;
      }
      if (issuer) commit2(&sh.done);  // every product issued is complete, and its arrivals are made
      __syncwarp();
    } else {
      // ---- softmax: two threads, half 0 and 1 of the keys, for a query row ----
      const uint32_t quad = warp & 3, row = quad * 32 + lane, lanes = (quad * 32u) << 16, half = warp >= 8, bar = 1 + quad;
      const uint32_t p_ready = map_shared(smem_u32(sh.p_ready), 0), o_free = map_shared(smem_u32(&sh.o_free), 0);
      const float scale2 = a.scale * kLog2e;  // (positive and finite)
      const uint64_t scale22 = pair_of(scale2, scale2);
      const uint32_t token = row / a.group, qg = row % a.group;
      // A row's two warps wait for each other by barriers without a limit, so they leave together: one
      // whose wait gave up goes on to the next barrier and says so there.
      volatile uint32_t *dead = sh.dead;
      uint32_t g = 0, items = 0;
      bool ok = true;
      for (;; items++) {
        const bool got = next_item();
        if (pair_any(bar, !got)) break;
        const ChunkStream st = it.s;
        const uint32_t i = it.tok0 + rank * tpt + token;  // this row's token
        const bool valid = token < tpt && i < it.tok1;
        const bool any = __any_sync(0xffffffffu, valid);
        const uint32_t depth = valid && a.parents && a.window ? chunk_depth(a, st.first, i) : 0u;
        const ChunkLow lo = chunk_low(a, st, st.before + (a.parents ? depth : i));
        float m = valid ? -INFINITY : INFINITY, l = 0.f;  // (other rows: weights of 0, see clear_q)
        for (uint32_t t = 0; t < it.nt; t++, g++, recs++) {
          const uint32_t scol = tmem + kSCol + (g & 1) * kKeys + lanes;
          ok = ok && wait(&sh.s_full[g & 1], (g >> 1) & 1);
          __syncwarp();
          tc_fence_after();
          uint32_t s[2][32];
          tc_ld32(scol + half * 64, s[0]);
          tc_ld32(scol + half * 64 + 32, s[1]);
          // the tile's record (K was copied by it, so it is there)
          const Rec &rec = sh.recs[recs % kRecs];
          const uint2 head = *reinterpret_cast<const uint2 *>(&rec);
          const uint32_t seg = head.x & 3, key0 = head.y;
          const bool masked = any && !(head.x & 4);
          uint32_t mask[2] = {~0u, ~0u};  // which of this thread's keys the row sees
          if (masked) {
            mask[0] = rec.mask[half * 2], mask[1] = rec.mask[half * 2 + 1];
            const uint32_t at = key0 + half * 64;
            if (seg == 2 && a.parents) {
              if (valid && half == 0) chunk_report_parent(a, st.first, i);
              uint32_t own[2] = {0u, 0u};
              int32_t j = valid ? (int32_t)i : -1;
              for (uint32_t d = depth; j >= (int32_t)at && (!a.window || d >= lo.fresh); d--, j = chunk_parent(a, st.first, (uint32_t)j)) {
                const uint32_t x = (uint32_t)j - at;
#pragma unroll
                for (int c = 0; c < 2; c++) own[c] |= x / 32 == (uint32_t)c ? 1u << (x & 31) : 0u;
              }
              mask[0] &= own[0], mask[1] &= own[1];
            } else {
              const uint32_t from = seg == 0 ? lo.prefix : seg == 1 ? lo.cached : lo.fresh;
              const int k0 = from > at ? (int)min(from - at, 64u) : 0;
              const int k1 = seg < 2 ? 64 : i < at ? 0 : (int)min(i - at + 1, 64u);
              mask[0] &= bits_of(k0, k1), mask[1] &= bits_of(k0 - 32, k1 - 32);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.rec_empty[recs % kRecs]);
          tc_wait_ld();
          float mx = -INFINITY;
          if (any) {
            if (masked) {
#pragma unroll
              for (int c = 0; c < 2; c++)
#pragma unroll
                for (int e = 0; e < 32; e++)
                  if (!((mask[c] >> e) & 1)) s[c][e] = 0xFF800000u;  // -inf
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; e += 2)
#pragma unroll
              for (int c = 0; c < 2; c++)
                top[(e + c) & 3] = max3_nan(top[(e + c) & 3], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
            mx = max3_nan(max3_nan(top[0], top[1], top[2]), top[3], top[3]) * scale2;
          }
          // (a NaN grows whatever there is, and its sum stays NaN; a tile without a visible key leaves all as it is)
          auto grows = [&]() { return !(mx <= m + kGrow) && mx != -INFINITY; };
          // P of the second half lies over S of the first: both have read S behind this barrier
          tc_fence_before();
          if (!ok) dead[warp - 4] = 1u;
          const bool some = pair_any(bar, !ok || grows());
          tc_fence_after();
          if (some) {  // a row's maximum has grown: the two halves agree on it
            sh.half[half][row] = mx;
            pair_sync(bar);
            mx = max3_nan(mx, sh.half[half ^ 1][row], sh.half[half ^ 1][row]);
            ok = !(dead[quad] | dead[4 + quad]);
            pair_sync(bar);
            if (!ok) break;
            const bool grow = grows();
            // (with a maximum of +inf the result is NaN, as inf - inf would be: see chunk_mend)
            const float m1 = grow ? mx : m, keep = grow ? exp2_approx(m - m1) : 1.f;
            m = m1;
            l *= keep;
            if (t > 0) {
              // O is rescaled behind the product of the tile before.  (A barrier can only be asked for the phase
              // that follows one known to be over, while the one after that cannot end: S of this tile came
              // behind the product before that one, and the next product waits for this P.)
              ok = __all_sync(0xffffffffu, wait(&sh.pv_done, (g - 1) & 1));
              tc_fence_after();
#pragma unroll 1
              for (uint32_t c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
                uint32_t o[32];
                tc_ld32(tmem + lanes + c, o);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tc_st32(tmem + lanes + c, o);
              }
            }
          }
          if (any) {
            const float low = kBias<T> - (m == -INFINITY ? 0.f : m);
            const uint64_t low2 = pair_of(low, low);
            uint64_t sum[2] = {0ull, 0ull};
            uint32_t p[32];
#pragma unroll
            for (int e = 0; e < 32; e++) {
              const uint64_t x = fma2(pair_of(__uint_as_float(s[e / 16][2 * (e % 16)]), __uint_as_float(s[e / 16][2 * (e % 16) + 1])),
                                      scale22, low2);
              float p0, p1;
              halves(x, p0, p1);
              p0 = exp2_approx(p0), p1 = exp2_approx(p1);
              sum[e & 1] = add2(sum[e & 1], pair_of(p0, p1));
              p[e] = pack2(p0, p1, static_cast<const T *>(nullptr));
            }
            tc_st32(scol + half * 32, p);
            float l0, l1;
            halves(add2(sum[0], sum[1]), l0, l1);
            l += l0 + l1;
            tc_wait_st();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_remote(p_ready + (g & 1) * 8);
        }
        if (!ok && (dead[quad] | dead[4 + quad])) break;  // (both warps left the loop above)
        // ---- the result, or this part of it ----
        ok = __all_sync(0xffffffffu, ok && wait(&sh.o_full, items & 1));
        tc_fence_after();
        bool bad = false;
        sh.half[half][row] = l;
        if (pair_any(bar, !ok)) break;
        l = m == -INFINITY ? 0.f : l + sh.half[half ^ 1][row];  // the sums of both halves
        if (any && it.part) {
          const size_t at_row = (size_t)(it.part - 1) * (2 * kRows) + rank * kRows + row;
          if (valid && half == 0) w.ml[at_row] = make_float2(m - kBias<T>, l);
#pragma unroll 1
          for (uint32_t c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
            uint32_t o[32];
            tc_ld32(tmem + lanes + c, o);
            tc_wait_ld();
            if (valid) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) st_global_32b(w.o + part_at<D>(it.part - 1, rank * kRows + row, c + e), o + e);
            }
          }
        } else if (any) {
          // four lanes write 64 bytes of a row (with a lane to a row the stores took 7,000 cycles a unit)
          T *out = static_cast<T *>(a.out) + (long long)(st.first + i) * a.os + (it.h * a.group + qg) * a.oh;
          if (!valid) out = nullptr;
          T *rows[4];
#pragma unroll
          for (int r = 0; r < 4; r++) rows[r] = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, (unsigned long long)out, (lane & 28) + r));
          const float inv = m == INFINITY ? NAN : l == 0.f ? 0.f : 1.f / l;
          float most = 0.f;
#pragma unroll 1
          for (uint32_t c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
            uint32_t o[32], y[4][4];
            tc_ld32(tmem + lanes + c, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; e++) {
              const float x0 = __uint_as_float(o[2 * e]) * inv, x1 = __uint_as_float(o[2 * e + 1]) * inv;
              most = max3_nan(most, fabsf(x0), fabsf(x1));
              y[e / 4][e % 4] = pack2(x0, x1, static_cast<const T *>(nullptr));
            }
            // 4 x 4 pieces of 16 bytes turned over: y[r] becomes this lane's quarter of row r
#pragma unroll
            for (int step = 1; step <= 2; step++) {
              const bool odd = lane & step;
#pragma unroll
              for (int q = 0; q < 2; q++) {
                const int p = step == 1 ? 2 * q : q;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                  const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? y[p][e] : y[p + step][e], step);
                  if (odd) y[p][e] = got; else y[p + step][e] = got;
                }
              }
            }
#pragma unroll
            for (int r = 0; r < 4; r++)
              if (rows[r]) *reinterpret_cast<uint4 *>(rows[r] + c + (lane & 3) * 8) = make_uint4(y[r][0], y[r][1], y[r][2], y[r][3]);
          }
          // not finite beside a sum that is, or a maximum that is infinite in the power of 2 only: chunk_mend
          bad = valid && suspect(most, static_cast<const T *>(nullptr)) && (!isnan(l) || m == INFINITY);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_remote(o_free);
        // (by the join kernel: here it would keep the other roles waiting)
        if (__any_sync(0xffffffffu, bad) && lane == 0) atomicMin(&sh.bad[0], items), atomicMax(&sh.bad[1], items + 1);
      }
    }
  }
  __syncwarp();
  // every arrival that a product makes has been made, in both CTAs, and tensor memory is at rest
  tc_wait(&sh.done, 0, nullptr, a.status);
  __syncthreads();
  if (*abort) {  // and so are copies that no product has waited for (the second CTA may not have told of its own)
    if (tid < C::kSlots && sh.fills[tid]) tc_wait(&sh.full[tid], (sh.fills[tid] - 1) & 1, nullptr, a.status, false, kWaitNs / 20);
    if (tid == 32 && sh.q_loads) tc_wait(&sh.q_here, (sh.q_loads - 1) & 1, nullptr, a.status, false, kWaitNs / 20);
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  if (tid == 0) w.bad[blockIdx.x] = make_uint2(sh.bad[0], sh.bad[1]);
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ---------------------------------------------------------------------------
// out = sum over a row's parts of O 2^(m - M) / sum of l 2^(m - M).  A CTA takes 32 rows of a cut unit,
// a thread 16 columns of one: a warp reads a part's rows as they lie, and all loads of a unit's first
// parts are in flight at once; 20 to 28 bytes spill at 64 registers.  (A warp per row, one row after the other, took 11.6 us behind the
// main kernel of 64 trees of 16 nodes, this 7.0; of 21 chunks 15.2 and 7.9.)
constexpr uint32_t kJoinRows = 32, kJoinCols = 16;  // (a lane to a row)
template <int D>
constexpr uint32_t kJoinWarps = D / kJoinCols;
template <int D>
constexpr uint32_t kJoinThreads = 32 * kJoinWarps<D>;
// A CTA's rows that are not finite and need a second look (chunk_mend), a warp each: `again` of the pair's cut
// unit, and those of its whole ones.  The kernel waits for nobody here, however long a row takes.
template <typename T, int D>
__device__ __noinline__ void chunk_mend_rows(const ChunkArgs &a, const ChunkWork &w, uint32_t again) {
  const uint32_t warp = threadIdx.x >> 5, row0 = blockIdx.x * kJoinRows, rank = row0 / kRows, tpt = kRows / a.group;
  const Cut &cut = w.cut[blockIdx.y];
  ChunkKey<T> hint{nullptr, nullptr};
  auto mend = [&](const ChunkStream &s, uint32_t b, uint32_t h, uint32_t t, uint32_t x) {  // row x of the unit at token t
    const uint32_t at = (row0 + x) % kRows, i = t + rank * tpt + at / a.group;
    if (at / a.group < tpt && i < min(s.count, t + 2 * tpt)) chunk_mend<T, D>(a, s, b, i, h * a.group + at % a.group, hint);
  };
  if (again) {
    const ChunkStream s = chunk_stream(a, cut.b);
    for (uint32_t x = warp; x < kJoinRows; x += kJoinWarps<D>)
      if (again >> x & 1) mend(s, cut.b, cut.h, cut.tok0, x);
  }
  const uint2 items = w.bad[2 * blockIdx.y + rank];
  if (items.x >= items.y) return;
  hint = ChunkKey<T>{nullptr, nullptr};  // (of later tokens than these)
  uint32_t b = cut.run_b, h = cut.run_h, t = cut.run_tok;
  ChunkStream s = chunk_stream(a, b);
  for (uint32_t n = 0; n < items.y; n++) {
    for (uint32_t x = warp; n >= items.x && x < kJoinRows; x += kJoinWarps<D>) mend(s, b, h, t, x);
    t += 2 * tpt;
    if (t < s.count) continue;
    t = 0;
    hint = ChunkKey<T>{nullptr, nullptr};
    if (++h < a.nkv) continue;
    h = 0;
    do {
      if (++b >= a.n) return;
      s = chunk_stream(a, b);
    } while (!s.count);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads<D>, 1024 / kJoinThreads<D>)
    chunk_join_kernel(const __grid_constant__ ChunkArgs a, const ChunkWork w) {
  constexpr uint32_t kU = 2;  // parts whose loads are in flight together
  __shared__ uint32_t bad_rows;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pair = blockIdx.y;
  const uint32_t row = blockIdx.x * kJoinRows + lane, col = warp * kJoinCols;
  if (threadIdx.x == 0) bad_rows = 0;
  grid_dep_wait();
  grid_dep_launch();
  const Cut cut = w.cut[pair];
  const uint32_t tpt = kRows / a.group;
  const uint32_t rank = row / kRows, token = row % kRows / a.group;
  const uint32_t i = cut.tok0 + rank * tpt + token, hq = cut.h * a.group + row % kRows % a.group;
  const bool valid = cut.parts && token < tpt && i < cut.tok1;
  const uint2 items = w.bad[2 * pair + rank];
  if (!__any_sync(0xffffffffu, valid) && items.x >= items.y) return;  // (the same in all warps)
  // the beginning of the unit in slot 2 pair + 1, the rest in slots 2 (pair + 1), 2 (pair + 2), ...
  auto slot = [&](uint32_t p) { return 2 * (pair + p) + (p == 0); };
  float v[kU][kJoinCols];
  auto load = [&](uint32_t p0) {
#pragma unroll
    for (uint32_t u = 0; u < kU; u++)
      if (p0 + u < cut.parts) {
#pragma unroll
        for (uint32_t e = 0; e < kJoinCols; e += 4)
          *reinterpret_cast<float4 *>(&v[u][e]) =
              *reinterpret_cast<const float4 *>(w.o + part_at<D>(slot(p0 + u), row, col + e / 8 * 8) + e % 8);
      }
  };
  auto ml_of = [&](uint32_t p) { return w.ml[(size_t)slot(p) * (2 * kRows) + row]; };
  const ChunkStream st = chunk_stream(a, cut.b);
  float o[kJoinCols], sum = 0.f;
#pragma unroll
  for (uint32_t e = 0; e < kJoinCols; e++) o[e] = 0.f;
  bool bad = false;
  if (valid) {
    load(0);
    float top = -INFINITY;
#pragma unroll 4
    for (uint32_t p = 0; p < cut.parts; p++) top = fmaxf(top, ml_of(p).x);
    const float ref = top == -INFINITY ? 0.f : top;
    for (uint32_t p0 = 0; p0 < cut.parts; p0 += kU) {
      if (p0) load(p0);
#pragma unroll
      for (uint32_t u = 0; u < kU; u++) {
        if (p0 + u >= cut.parts) break;
        const float2 ml = ml_of(p0 + u);
        if (ml.x == -INFINITY) continue;  // a part without a visible position has no O
        const float f = exp2_approx(ml.x - ref);  // (0 of a part that is not finite is NaN)
        sum = fmaf(ml.y, f, sum);
#pragma unroll
        for (uint32_t e = 0; e < kJoinCols; e++) o[e] = fmaf(v[u][e], f, o[e]);
      }
    }
#pragma unroll
    for (uint32_t e = 0; e < kJoinCols; e++) {
      o[e] = sum == 0.f ? 0.f : o[e] / sum;
      bad |= suspect(fabsf(o[e]), static_cast<const T *>(nullptr));
    }
    bad = bad && (!isnan(sum) || top == INFINITY);
    T *out = static_cast<T *>(a.out) + (long long)(st.first + i) * a.os + hq * a.oh + col;
#pragma unroll
    for (uint32_t e = 0; e < kJoinCols; e += 8)
      *reinterpret_cast<uint4 *>(out + e) =
          make_uint4(pack2(o[e], o[e + 1], static_cast<const T *>(nullptr)), pack2(o[e + 2], o[e + 3], static_cast<const T *>(nullptr)),
                     pack2(o[e + 4], o[e + 5], static_cast<const T *>(nullptr)),
                     pack2(o[e + 6], o[e + 7], static_cast<const T *>(nullptr)));
  }
  const uint32_t mine = __ballot_sync(0xffffffffu, bad);
  __syncthreads();
  if (mine && lane == 0) atomicOr(&bad_rows, mine);
  __syncthreads();
  if (bad_rows || items.x < items.y) chunk_mend_rows<T, D>(a, w, bad_rows);
}

// ---------------------------------------------------------------------------
// Host: tensor maps.  Token, head and page strides of dimensions of one element are never used and
// may be any number, so they are replaced.
struct MapDims {
  uint32_t rank;
  cuuint64_t dims[5], strides[4];  // elements; bytes from the second dimension on
  cuuint32_t box[5];
};
inline cudaError_t encode_map(CUtensorMap *map, const void *base, const MapDims &d) {
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn)
                                                                : nullptr;
  }();
  if (!encode) return cudaErrorNotSupported;
  const cuuint32_t step[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, d.rank, const_cast<void *>(base), d.dims, d.strides, d.box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorNotSupported;
}
inline cuuint64_t stride_or(uint32_t n, long long elements, cuuint64_t other) {
  return n > 1 ? (cuuint64_t)elements * 2 : other;
}
}  // namespace
}  // namespace ch
