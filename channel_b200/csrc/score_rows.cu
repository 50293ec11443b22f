// score_rows.cu -- log-probability, entropy, rank and top alternatives of given tokens, from whole
// rows of logits (ch_score_rows).
//
// With x the (capped) logits of a row, m their maximum, S = sum e^(x - m), T = sum (x - m) e^(x - m):
//   log p_t = x_t - m - log S,   entropy = -sum p log p = log S - T / S.
// One pass over the row, cut into equal parts for the CTAs of a cluster: a thread keeps its own
// running m, S and T (rescaled when its m grows; sums of all threads in 64 bits)
// and the count of logits in front of the given one.  The alternatives need no second pass: a warp
// keeps the largest logit of each block of 256, and the k largest logits of a part (equal ones by
// index) lie in the k blocks with the largest maxima (equal ones by index): if a block is not among
// them, k blocks each hold a logit that comes before all of its own.  Those blocks are read again for
// what reaches the k-th maximum, mostly little more than k logits, which are ranked by comparing all
// with all; where it is too much (equal logits), the blocks are taken apart the same way, first into
// a lane's 8 logits, then one by one.  The parts' sorted lists are merged in the cluster's first CTA.
#include <cuda_bf16.h>

#include <algorithm>
#include <cstring>
#include <string>

#include "../../include/channel_cuda.h"
#include "common.cuh"
#include "kernels.cuh"

namespace ch {
int set_last_error(int code, const std::string &msg);

namespace {
constexpr uint32_t kMaxVocab = 262144, kMaxTop = 64;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kBlock = 256, kLane = 8;  // logits of a block, and of a lane in it
constexpr uint32_t kMaxBlocks = kMaxVocab / kBlock, kMaxParts = 16, kNear = 512;
#ifndef X_WANT
#define X_WANT 12
#define X_LEAST 8
#endif
constexpr uint32_t kParts = 8, kWant = X_WANT, kLeast = X_LEAST;
constexpr float kLog2e = 1.44269504088896341f;

struct ScoreArgs {
  const void *logits;
  const int32_t *targets;
  float *logprobs, *entropy, *top_logprobs;
  int32_t *ranks, *top_ids;
  long long stride;
  uint32_t n, vocab, top, parts;
  float cap, lowest;  // logits at or below `lowest` are masked
  uint32_t *status;
};

CH_DEV float value(float v) { return v; }
CH_DEV float value(__half v) { return __half2float(v); }
CH_DEV float value(__nv_bfloat16 v) { return __bfloat162float(v); }

// a logit as the order sees it: masked ones and NaN are -inf, both zeros are one
CH_DEV float clean(float x, float lowest) { return x > lowest ? x + 0.f : -INFINITY; }
// floats in the order of unsigned numbers; -inf is the smallest that occurs
CH_DEV uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
CH_DEV float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u); }

// logits [i, i + 8) of a row, -inf past its end
template <typename T>
CH_DEV void load8(const T *row, uint32_t i, uint32_t vocab, bool vec, float (&x)[kLane]) {
  if (vec && i + kLane <= vocab) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < (int)kLane / kPer; c++) {
      const uint4 u = *reinterpret_cast<const uint4 *>(row + i + c * kPer);
      const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
      for (int e = 0; e < kPer; e++) x[c * kPer + e] = value(t[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < (int)kLane; e++) x[e] = i + e < vocab ? value(row[i + e]) : -INFINITY;
  }
}

CH_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh(y) for |y| <= 0.6: y + y u q(u), u = y^2, q of degree 3 with the least relative error of the
// whole, 2^-23.5
constexpr float kNearZero = 0.6f;
CH_DEV uint64_t tanh_small(uint64_t y) {
  const uint64_t u = mul2(y, y);
  uint64_t q = fma2(u, pair_of(0.015612633898854256f, 0.015612633898854256f), pair_of(-0.05221180617809296f, -0.05221180617809296f));
  q = fma2(q, u, pair_of(0.13313116133213043f, 0.13313116133213043f));
  q = fma2(q, u, pair_of(-0.33332598209381104f, -0.33332598209381104f));
  return fma2(mul2(y, u), q, y);
}
// and elsewhere, 1 - 2 / (1 + e^2y): off by some 2^-23, of at least 0.53
CH_DEV float tanh_large(float y) { return 1.f - __fdividef(2.f, 1.f + ex2(y * (2.f * kLog2e))); }

// running maximum, sum of e^(x - m) and of (x - m) e^(x - m).  In the sums +inf stands for f32's
// largest value: tokens of +inf share the weight, and m tells that there are some.
struct Sums {
  float m;
  uint32_t before;  // logits in front of the given one
  double s, t;
};
constexpr float kMax = 3.402823466e38f;
CH_DEV Sums join(const Sums &a, const Sums &b) {
  Sums r{fmaxf(a.m, b.m), a.before + b.before, 0., 0.};
  for (const Sums *x : {&a, &b}) {
    if (x->m == -INFINITY) continue;
    const float d = fminf(x->m, kMax) - fminf(r.m, kMax);
    const double f = expf(d);
    if (f == 0.) continue;
    r.s += x->s * f;
    r.t += (x->t + d * x->s) * f;
  }
  return r;
}

struct Shared {
  uint32_t best[kMaxBlocks];  // a block's largest logit, ordered
  uint32_t list[kMaxTop], n_list, n_over, counts[2][kWarps], warp_at[kWarps];
  uint32_t near_key[kNear], near_id[kNear];  // logits that may be alternatives
  uint32_t lanes[kMaxTop * 32];
  Sums warps[kWarps];
  // of the cluster's parts, in the first CTA
  Sums part[kMaxParts];
  uint32_t n_part[kMaxParts], key[kMaxParts][kMaxTop], id[kMaxParts][kMaxTop];
};

// a number that want of the CTA's keys (PER a thread; 0: none) reach, or more of them if the want-th
// largest is not alone; want keys at least
template <int PER>
CH_DEV uint32_t kth_largest(const uint32_t (&key)[PER], uint32_t want, Shared &sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // bits above the first one in which keys differ are the same in all
  uint32_t any = 0, all = ~0u;
#pragma unroll
  for (int e = 0; e < PER; e++)
    if (key[e]) any |= key[e], all &= key[e];
  any = __reduce_or_sync(0xffffffffu, any), all = __reduce_and_sync(0xffffffffu, all);
  if (lane == 0) sh.counts[0][warp] = any, sh.counts[1][warp] = all;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; w++) any |= sh.counts[0][w], all &= sh.counts[1][w];
  const int top = 32 - __clz(any ^ all);  // bits that differ
  uint32_t k = top == 32 ? 0u : all >> top << top;
  __syncthreads();
  for (int bit = top - 1; bit >= 0; bit--) {
    const uint32_t edge = k | 1u << bit;
    uint32_t n = 0;
    if constexpr (PER == 1) {
      n = __syncthreads_count(key[0] >= edge);
    } else {
      uint32_t mine = 0;
#pragma unroll
      for (int e = 0; e < PER; e++) mine += key[e] >= edge;
      mine = __reduce_add_sync(0xffffffffu, mine);
      if (lane == 0) sh.counts[bit & 1][warp] = mine;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; w++) n += sh.counts[bit & 1][w];
    }
    if (n >= want) k = edge;
    if (n == want) break;
  }
  __syncthreads();
  return k;
}
// want keys of the CTA's (PER a thread, in index order by thread), the largest and of equal ones the
// first: take(e) for each; returns a number that they reach and no other key does, or equal ones only
template <int PER, typename F>
CH_DEV uint32_t choose(const uint32_t (&key)[PER], uint32_t want, Shared &sh, F take) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t edge = kth_largest(key, want, sh);
  // keys of `edge` itself are taken as far as there is room: more than that only if they are the want-th
  uint32_t over = 0, same = 0;
#pragma unroll
  for (int e = 0; e < PER; e++) over += key[e] > edge, same += key[e] == edge;
  if (threadIdx.x == 0) sh.n_over = 0;
  uint32_t inc = same;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) sh.warp_at[warp] = inc;
  __syncthreads();
  over = __reduce_add_sync(0xffffffffu, over);
  if (lane == 0) atomicAdd(&sh.n_over, over);
  uint32_t rank = inc - same;
  for (int w = 0; w < warp; w++) rank += sh.warp_at[w];
  __syncthreads();
  const uint32_t room = want - sh.n_over;
#pragma unroll
  for (int e = 0; e < PER; e++) {
    if (key[e] > edge) take(e);
    if (key[e] == edge && rank++ < room) take(e);
  }
  __syncthreads();
  return edge;
}
// a list of n distinct numbers (n <= kMaxTop) into rising order
CH_DEV void sort_list(uint32_t *list, uint32_t n) {
  uint32_t mine = 0, place = 0;
  if (threadIdx.x < n) {
    mine = list[threadIdx.x];
    for (uint32_t j = 0; j < n; j++) place += list[j] < mine;
  }
  __syncthreads();
  if (threadIdx.x < n) list[place] = mine;
  __syncthreads();
}

// writes to the first CTA's copy of a shared variable
template <typename V>
CH_DEV void to_first(V *local, V v) {
  static_assert(sizeof(V) % 4 == 0, "words");
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(local)));
  uint32_t w[sizeof(V) / 4];
  memcpy(w, &v, sizeof(V));
#pragma unroll
  for (uint32_t k = 0; k < sizeof(V) / 4; k++)
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at + 4 * k), "r"(w[k]) : "memory");
}

template <typename T, bool CAP>
__global__ void __launch_bounds__(kThreads, 4) score_rows_kernel(const ScoreArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // waited for ahead of stores to the first CTA
  const T *row = static_cast<const T *>(a.logits) + r * a.stride;
  const bool vec = ((uintptr_t)row & 15) == 0;
  const uint32_t all_blocks = (a.vocab + kBlock - 1) / kBlock, per_part = (all_blocks + a.parts - 1) / a.parts;
  const uint32_t first = min(part * per_part, all_blocks), blocks = min(per_part, all_blocks - first);
  const int32_t target = a.targets[r];
  const bool asked = target >= 0 && (uint32_t)target < a.vocab;
  if (tid == 0 && part == 0 && target >= 0 && !asked && a.status) atomicOr(a.status, DEV_ERR_BAD_SLOT);
  const float given = asked ? clean(value(row[target]), a.lowest) : INFINITY;
  // in front of the target are larger logits, and equal ones of a lower index: in blocks before its own
  // what is above `least`, in those behind it what is above `given`
  const float least = asked && given > -INFINITY ? nextafterf(given, -INFINITY) : INFINITY;
  const uint32_t own_block = asked ? (uint32_t)target / kBlock : 0u;

  // ---- the pass ----
  // logits below `small` (capped: where the polynomial holds) are neither masked nor infinite nor NaN,
  // and differ from any m by a finite number
  const float inv_cap = CAP ? 1.f / a.cap : 0.f, small = fminf(CAP ? a.cap * kNearZero : 1e30f, -a.lowest);
  const uint64_t cap2 = pair_of(a.cap, a.cap), inv2 = pair_of(inv_cap, inv_cap), log2e2 = pair_of(kLog2e, kLog2e);
  float m = -INFINITY, s = 0.f, t = 0.f;
  uint32_t before = 0;
  bool infinite = false;
  constexpr int kU = 4;  // blocks whose loads are in flight together
  auto block = [&](uint32_t b, float (&x)[kLane]) {
    const uint32_t i = (first + b) * kBlock + lane * kLane;
    const float top = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), fmaxf(x[6], x[7]));
    const uint32_t most = __reduce_max_sync(0xffffffffu, ordered(clean(top, a.lowest)));
    if (lane == 0) sh.best[b] = most;
    if (asked && (first + b == own_block || given == -INFINITY)) {
#pragma unroll
      for (int e = 0; e < (int)kLane; e++) {
        const float y = clean(x[e], a.lowest);
        before += (y > given || (y == given && i + e < (uint32_t)target)) && i + e < a.vocab;
      }
    } else {
      const float edge = first + b < own_block ? least : given;
      if (top > edge) {
#pragma unroll
        for (int e = 0; e < (int)kLane; e++) before += x[e] > edge;
      }
    }
    // the largest magnitude, NaN if there is one
    const float far = max3_nan(max3_nan(fabsf(x[0]), fabsf(x[1]), fabsf(x[2])), max3_nan(fabsf(x[3]), fabsf(x[4]), fabsf(x[5])),
                               max3_nan(fabsf(x[6]), fabsf(x[7]), 0.f));
    auto raise = [&](float m1) {  // m1: largest of the lane's
      if (!(m1 > m)) return;
      const float d = m - m1, f = ex2(d * kLog2e);
      t = f == 0.f ? 0.f : (t + d * s) * f;
      s = f == 0.f ? 0.f : s * f;
      m = m1;
    };
    if (__any_sync(0xffffffffu, !(far < small))) {  // one by one
      float z[kLane], most_z = -INFINITY;
#pragma unroll
      for (int e = 0; e < (int)kLane; e++) {
        z[e] = -INFINITY;
        if (!(x[e] > a.lowest)) continue;
        if (CAP) {
          const float w = x[e] * inv_cap;
          float lo, hi;
          halves(tanh_small(pair_of(w, w)), lo, hi);
          z[e] = a.cap * (fabsf(w) < kNearZero ? lo : tanh_large(w));
        } else {
          infinite |= x[e] == INFINITY;
          z[e] = fminf(x[e], kMax);
        }
        most_z = fmaxf(most_z, z[e]);
      }
      raise(most_z);
#pragma unroll
      for (int e = 0; e < (int)kLane; e++) {
        const float d = z[e] - m, w = z[e] == -INFINITY ? 0.f : ex2(d * kLog2e);
        s += w;
        if (w != 0.f) t = fmaf(d, w, t);  // (0 times -inf would be NaN)
      }
      return;
    }
    uint64_t y[kLane / 2];
    float most_y = top;
#pragma unroll
    for (int e = 0; e < (int)kLane / 2; e++) {
      y[e] = pair_of(x[2 * e], x[2 * e + 1]);
      if (CAP) y[e] = mul2(tanh_small(mul2(y[e], inv2)), cap2);
    }
    if (CAP) {  // (the polynomial rises, but roundings of neighbours may not)
      float z[kLane];
#pragma unroll
      for (int e = 0; e < (int)kLane / 2; e++) halves(y[e], z[2 * e], z[2 * e + 1]);
      most_y = max3(max3(z[0], z[1], z[2]), max3(z[3], z[4], z[5]), fmaxf(z[6], z[7]));
    }
    raise(most_y);
    const uint64_t low = pair_of(-m, -m);
    uint64_t s2 = 0ull, t2 = 0ull;
#pragma unroll
    for (int e = 0; e < (int)kLane / 2; e++) {
      const uint64_t d = add2(y[e], low);
      float w0, w1;
      halves(mul2(d, log2e2), w0, w1);
      const uint64_t w = pair_of(ex2(w0), ex2(w1));
      s2 = add2(s2, w);
      t2 = fma2(d, w, t2);
    }
    float lo, hi;
    halves(s2, lo, hi), s += lo + hi;
    halves(t2, lo, hi), t += lo + hi;
  };
  uint32_t b = warp;
  for (; b + (kU - 1) * kWarps < blocks; b += kU * kWarps) {
    float x[kU][kLane];
#pragma unroll
    for (int u = 0; u < kU; u++) load8(row, (first + b + u * kWarps) * kBlock + lane * kLane, a.vocab, vec, x[u]);
#pragma unroll
    for (int u = 0; u < kU; u++) block(b + u * kWarps, x[u]);
  }
  for (; b < blocks; b += kWarps) {
    float x[kLane];
    load8(row, (first + b) * kBlock + lane * kLane, a.vocab, vec, x);
    block(b, x);
  }

  // ---- the part's sums ----
  Sums mine{infinite ? INFINITY : m, before, s, t};
#pragma unroll
  for (int o = 16; o; o >>= 1)
    mine = join(mine, Sums{__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.before, o),
                           __shfl_xor_sync(0xffffffffu, mine.s, o), __shfl_xor_sync(0xffffffffu, mine.t, o)});
  if (lane == 0) sh.warps[warp] = mine;
  __syncthreads();

  // ---- the part's alternatives, sorted ----
  const uint32_t n_blocks = min(a.top, blocks);
  uint32_t n = 0;
  if (n_blocks) {
    if (tid == 0) sh.n_list = 0;
    uint32_t edge;
    auto take_block = [&](uint32_t b) { sh.list[atomicAdd(&sh.n_list, 1u)] = b; };
    if (blocks <= kThreads) {
      const uint32_t key[1] = {(uint32_t)tid < blocks ? sh.best[tid] : 0u};
      edge = choose(key, n_blocks, sh, [&](int) { take_block(tid); });
    } else {
      constexpr int kPer = kMaxBlocks / kThreads;
      uint32_t key[kPer];
#pragma unroll
      for (int e = 0; e < kPer; e++) key[e] = tid * kPer + e < blocks ? sh.best[tid * kPer + e] : 0u;
      edge = choose(key, n_blocks, sh, [&](int e) { take_block(tid * kPer + e); });
    }
    sort_list(sh.list, n_blocks);  // equal keys go by index
    if (tid == 0) sh.n_list = 0;
    if (n_blocks < a.top) edge = 0;  // fewer blocks than alternatives: any logit may be one
    __syncthreads();
    // the logits of those blocks that reach the last one's maximum
    for (uint32_t c = warp; c < n_blocks; c += kWarps) {
      const uint32_t i = (first + sh.list[c]) * kBlock + lane * kLane;
      float x[kLane];
      load8(row, i, a.vocab, vec, x);
      uint32_t best = 0;
#pragma unroll
      for (int e = 0; e < (int)kLane; e++) {
        const uint32_t k = i + e < a.vocab ? ordered(clean(x[e], a.lowest)) : 0u;
        best = max(best, k);
        if (k >= edge && k) {
          const uint32_t at = atomicAdd(&sh.n_list, 1u);
          if (at < kNear) sh.near_key[at] = k, sh.near_id[at] = i + e;
        }
      }
      sh.lanes[c * 32 + lane] = best;
    }
    __syncthreads();
    n = sh.n_list;
    __syncthreads();
    if (n > kNear) {  // too many near ones: the first k lanes of 8 logits hold the alternatives
      constexpr int kPer = kMaxTop * 32 / kThreads;
      uint32_t lanes[kPer];
#pragma unroll
      for (int e = 0; e < kPer; e++) lanes[e] = tid * kPer + e < n_blocks * 32 ? sh.lanes[tid * kPer + e] : 0u;
      if (tid == 0) sh.n_list = 0;
      __syncthreads();
      choose(lanes, min(a.top, n_blocks * 32), sh, [&](int e) { sh.near_id[atomicAdd(&sh.n_list, 1u)] = tid * kPer + e; });
      // (every block but the row's last has 32 lanes, and n_blocks * 32 > kNear / 8 here)
      uint32_t l[2], k[2] = {0u, 0u};
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const uint32_t x = tid + u * kThreads;
        l[u] = x < a.top * kLane ? sh.near_id[x / kLane] : 0u;
        l[u] = (first + sh.list[l[u] / 32]) * kBlock + (l[u] % 32) * kLane + x % kLane;
        if (x < a.top * kLane && l[u] < a.vocab) k[u] = ordered(clean(value(row[l[u]]), a.lowest));
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 2; u++) sh.near_key[tid + u * kThreads] = k[u], sh.near_id[tid + u * kThreads] = l[u];
      n = min(a.top * kLane, kNear);
      __syncthreads();
    }
  }
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the first CTA has started
  if (tid == 0) {
    Sums all = sh.warps[0];
    for (int w = 1; w < kWarps; w++) all = join(all, sh.warps[w]);
    to_first(&sh.part[part], all);
    to_first(&sh.n_part[part], min(a.top, min(n, blocks * kBlock)));
  }
  for (uint32_t x = tid; x < n; x += kThreads) {
    const uint32_t k = sh.near_key[x], i = sh.near_id[x];
    if (!k) continue;  // past the row's end
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; j++) rank += sh.near_key[j] > k || (sh.near_key[j] == k && sh.near_id[j] < i);
    if (rank < a.top) to_first(&sh.key[part][rank], k), to_first(&sh.id[part][rank], i);
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (part) return;

  // ---- the row ----
  Sums all = sh.part[0];
  for (uint32_t p = 1; p < a.parts; p++) all = join(all, sh.part[p]);
  const bool any = all.m > -INFINITY;
  const double log_s = any ? log(all.s) : 0.;
  auto logprob = [&](float x) {
    if (x == -INFINITY || (x < INFINITY && all.m == INFINITY)) return -INFINITY;
    const float y = CAP ? a.cap * tanhf(x / a.cap) : fminf(x, kMax);
    return (float)((double)y - fminf(all.m, kMax) - log_s);
  };
  if (tid == 0) {
    a.logprobs[r] = asked ? logprob(given) : 0.f;
    a.entropy[r] = any ? (float)(log_s - all.t / all.s) : 0.f;
    a.ranks[r] = asked ? (int32_t)all.before + 1 : 0;
  }
  for (uint32_t x = tid; x < a.parts * a.top; x += kThreads) {
    const uint32_t p = x / a.top, e = x % a.top;
    if (e >= sh.n_part[p]) continue;
    const uint32_t k = sh.key[p][e];
    uint32_t rank = e;
    for (uint32_t q = 0; q < a.parts; q++) {  // ids rise with the part, so equal logits go by it
      if (q == p) continue;
      uint32_t lo = 0, hi = sh.n_part[q];  // how many of part q's list come before
      while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (q < p ? sh.key[q][mid] >= k : sh.key[q][mid] > k) lo = mid + 1; else hi = mid;
      }
      rank += lo;
    }
    if (rank < a.top) {
      const size_t at = (size_t)r * a.top + rank;
      a.top_ids[at] = (int32_t)sh.id[p][e];
      a.top_logprobs[at] = logprob(from_ordered(k));
    }
  }
}

template <typename T, bool CAP>
cudaError_t launch_t(const ScoreArgs &a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.n * a.parts);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, score_rows_kernel<T, CAP>, a);
}
template <typename T>
cudaError_t launch(const ScoreArgs &a, cudaStream_t s) {
  return a.cap != 0.f ? launch_t<T, true>(a, s) : launch_t<T, false>(a, s);
}

int score_rows(const ch_score_args *p, void *stream) {
  if (!p) return set_last_error(CH_EINVAL, "score_rows: args is NULL");
  if (p->n_rows == 0) return CH_OK;
  if (p->vocab == 0 || p->vocab > kMaxVocab)
    return set_last_error(CH_EINVAL, "score_rows: vocab must be 1.." + std::to_string(kMaxVocab));
  if (p->top > kMaxTop || p->top > p->vocab)
    return set_last_error(CH_EINVAL, "score_rows: top must be at most " + std::to_string(kMaxTop) + " and vocab");
  if (p->n_rows > 0x0FFFFFFFu) return set_last_error(CH_EINVAL, "score_rows: n_rows must be below 2^28");
  if (!p->logits || !p->targets || !p->logprobs || !p->entropy || !p->ranks || (p->top && (!p->top_ids || !p->top_logprobs)))
    return set_last_error(CH_EINVAL, "score_rows: NULL argument");
  if (!(p->softcap == 0.f || (p->softcap >= 1e-30f && p->softcap <= 1e30f)))
    return set_last_error(CH_EINVAL, "score_rows: softcap must be 0 or from 1e-30 to 1e30");
  ScoreArgs a{};
  a.logits = p->logits;
  a.targets = p->targets;
  a.logprobs = p->logprobs;
  a.entropy = p->entropy;
  a.top_logprobs = p->top_logprobs;
  a.ranks = p->ranks;
  a.top_ids = p->top_ids;
  a.stride = p->row_stride;
  a.n = p->n_rows;
  a.vocab = p->vocab;
  a.top = p->top;
  // parts of a row, each for a CTA of its cluster
  a.parts = 1;
  const uint32_t blocks = (p->vocab + kBlock - 1) / kBlock;
  while (a.parts < kParts && (unsigned long long)p->n_rows * a.parts < kWant * num_sms() && blocks >= 2 * a.parts * std::max(kLeast, p->top))
    a.parts *= 2;
  a.cap = p->softcap;
  a.status = p->status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (p->dtype == CH_F32) {
    a.lowest = -3.402823466e38f;
    e = launch<float>(a, s);
  } else if (p->dtype == CH_F16) {
    a.lowest = -65504.f;
    e = launch<__half>(a, s);
  } else if (p->dtype == CH_BF16) {
    a.lowest = -3.38953139e38f;
    e = launch<__nv_bfloat16>(a, s);
  } else {
    return set_last_error(CH_EINVAL, "score_rows: dtype must be CH_F32, CH_F16 or CH_BF16");
  }
  if (e != cudaSuccess) return set_last_error(CH_ECUDA, std::string("score_rows: ") + cudaGetErrorString(e));
  return CH_OK;
}
}  // namespace
}  // namespace ch

extern "C" int ch_score_rows(const ch_score_args *args, void *stream) {
  try {
    return ch::score_rows(args, stream);
  } catch (...) {
    return CH_ENOMEM;
  }
}
