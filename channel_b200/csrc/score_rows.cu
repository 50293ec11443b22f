// score_rows.cu -- log-probability, entropy, rank and top alternatives of given tokens, from whole
// rows of logits (ch_score_rows).
//
// With x the (capped) logits of a row, m their maximum, S = sum e^(x - m), T = sum (x - m) e^(x - m):
//   log p_t = x_t - m - log S,   entropy = -sum p log p = log S - T / S.
// One pass over the row, cut into equal parts for the CTAs of a cluster: a thread keeps its own
// running m, S and T (rescaled when its m grows; f32, as are the sums of a warp's lanes, and those of the
// warps and parts in 64 bits) and the count of logits in front of the given one.  The alternatives need no second pass: a warp
// keeps the largest logit of each block of 512, and the k largest logits of a part (equal ones by
// index) lie in the k blocks with the largest maxima (equal ones by index): if a block is not among
// them, k blocks each hold a logit that comes before all of its own.  Those blocks are read again for
// what reaches the k-th maximum, mostly little more than k logits, which are ranked by comparing all
// with all; where it is too much (equal logits), the blocks are taken apart the same way, first into
// a lane's 8 logits, then one by one.  The parts' sorted lists are merged in the cluster's first CTA.
//
// Bound: the pass by HBM (a block of 512 f32 logits takes an SM 77 cycles, its share of the bandwidth 85),
// the rest by latency: the blocks read again come behind what the other CTAs stream.  512 rows of 262,144
// capped f32 logits 117 us (537 MB, 4.6 TB/s), 777 rows of 100,003 bf16 61 us, one row 17 us a call;
// without the cap 512 f32 rows 87 us (6.2 TB/s).
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
constexpr uint32_t kBlock = 512, kLane = 8, kRuns = 2;  // logits of a block, and of a lane in each half of it
constexpr uint32_t kMaxBlocks = kMaxVocab / kBlock, kMaxParts = 16, kNear = 512;
constexpr uint32_t kParts = 8;
// What a part costs beside its blocks (first loads, the cluster; reading again for the alternatives), in
// blocks.  512 capped f32 rows of 262,144 with 5 alternatives take 123, 109, 125 and 155 us in 1, 2, 4
// and 8 parts; 777 16-bit rows of 100,003 with 20 alternatives 60, 71, 102 and 185; one row 47, 30, 22, 20.
constexpr uint32_t kPartCost = 90, kTopCost = 7;
constexpr float kLog2e = 1.44269504088896341f;

// CTAs on an SM: the polynomial of the cap wants 80 registers (24 to 28 bytes spill; without it, at 64
// registers, 64 to 76 bytes)
constexpr int ctas_of(bool cap) { return cap ? 3 : 4; }

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

// logits [i, i + 8) of a row as they lie in memory, -inf past its end
template <typename T>
struct Raw {
  static constexpr int kPer = 16 / sizeof(T), kVecs = kLane / kPer;
  uint4 v[kVecs];
};
CH_DEV uint32_t minus_inf(const float *) { return 0xFF800000u; }
CH_DEV uint32_t minus_inf(const __half *) { return 0xFC00u; }
CH_DEV uint32_t minus_inf(const __nv_bfloat16 *) { return 0xFF80u; }
template <typename T>
CH_DEV void load8(const T *row, uint32_t i, uint32_t vocab, bool vec, Raw<T> &x) {
  if (vec && i + kLane <= vocab) {
#pragma unroll
    for (int c = 0; c < Raw<T>::kVecs; c++) x.v[c] = __ldcs(reinterpret_cast<const uint4 *>(row + i) + c);
  } else {
    constexpr int kIn = 4 / sizeof(T);  // logits of a word
    uint32_t w[kLane / kIn];
#pragma unroll
    for (int k = 0; k < (int)kLane / kIn; k++) {
      w[k] = 0;
#pragma unroll
      for (int e = 0; e < kIn; e++) {
        const uint32_t at = i + k * kIn + e;
        uint32_t bits = minus_inf(row);
        if (at < vocab) {
          if constexpr (sizeof(T) == 4) bits = reinterpret_cast<const uint32_t *>(row)[at];
          else bits = reinterpret_cast<const uint16_t *>(row)[at];
        }
        w[k] |= bits << (16 * e);
      }
    }
#pragma unroll
    for (int c = 0; c < Raw<T>::kVecs; c++) x.v[c] = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
  }
}
CH_DEV void values(const Raw<float> &r, float *x) {
#pragma unroll
  for (int c = 0; c < 2; c++)
    x[4 * c] = __uint_as_float(r.v[c].x), x[4 * c + 1] = __uint_as_float(r.v[c].y), x[4 * c + 2] = __uint_as_float(r.v[c].z),
          x[4 * c + 3] = __uint_as_float(r.v[c].w);
}
CH_DEV void values(const Raw<__nv_bfloat16> &r, float *x) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
  for (int k = 0; k < 4; k++) x[2 * k] = __uint_as_float(w[k] << 16), x[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
}
CH_DEV void values(const Raw<__half> &r, float *x) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
    x[2 * k] = f.x, x[2 * k + 1] = f.y;
  }
}

CH_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The cap.  tanh(y) = y + y u q(u), u = y^2, for |y| <= 0.6, with q of degree 3 and the least relative
// error of the whole, 2^-23.5; so cap tanh(x / cap) = x + x v r(v), v = x^2, with the coefficients of q
// over powers of cap^2 in r.  Elsewhere 1 - 2 / (1 + e^2y), off by some 2^-23 of at least 0.53.
constexpr float kNearZero = 0.6f;
struct Cap {
  float cap, inv;
  uint64_t c[4];
  CH_DEV explicit Cap(float at) : cap(at), inv(1.f / at) {
    const float u = inv * inv, q[4] = {-0.33332598209381104f, 0.13313116133213043f, -0.05221180617809296f, 0.015612633898854256f};
    float f = u;
#pragma unroll
    for (int k = 0; k < 4; k++, f *= u) c[k] = pair_of(q[k] * f, q[k] * f);
  }
  CH_DEV uint64_t small(uint64_t x) const {
    const uint64_t v = mul2(x, x);
    return fma2(mul2(x, v), fma2(fma2(fma2(c[3], v, c[2]), v, c[1]), v, c[0]), x);
  }
  CH_DEV float any(float x) const {
    const float y = x * inv;
    float lo, hi;
    halves(small(pair_of(x, x)), lo, hi);
    // (outside, the powers of cap^2 above may not be numbers of f32)
    if (cap < 1e-4f || cap > 1e4f) lo = fabsf(y) < 1e-3f ? fmaf(x * y, y * -0.33333333f, x) : cap * tanhf(y);
    return fabsf(y) < kNearZero ? lo : cap * (1.f - __fdividef(2.f, 1.f + ex2(y * (2.f * kLog2e))));
  }
};

// maximum, sum of e^(x - m) and of (x - m) e^(x - m)
struct Sums {
  float m;
  uint32_t before;  // logits in front of the given one
  double s, t;
};
CH_DEV Sums join(const Sums &a, const Sums &b) {
  Sums r{fmaxf(a.m, b.m), a.before + b.before, 0., 0.};
  for (const Sums *x : {&a, &b}) {
    const float d = x->m == r.m ? 0.f : x->m - r.m;
    const double f = expf(d);
    if (f == 0.) continue;
    r.s += x->s * f;
    r.t += (x->t + d * x->s) * f;
  }
  return r;
}

// of the lanes' (the same in all)
CH_DEV Sums join_lanes(Sums x, int lanes) {
  for (int o = lanes / 2; o; o >>= 1)
    x = join(x, Sums{__shfl_xor_sync(0xffffffffu, x.m, o), __shfl_xor_sync(0xffffffffu, x.before, o),
                     __shfl_xor_sync(0xffffffffu, x.s, o), __shfl_xor_sync(0xffffffffu, x.t, o)});
  return x;
}

struct Shared {
  uint32_t best[kMaxBlocks];  // a block's largest logit, ordered
  Sums joined;
  uint32_t list[kMaxTop], n_list, n_over, counts[2][kWarps], warp_at[kWarps];
  uint64_t near[kNear];  // logits that may be alternatives: their order, equal ones by falling index
  uint32_t lanes[kMaxTop * kRuns * 32];
  Sums warps[kWarps];
  // of the cluster's parts, in the first CTA
  Sums part[kMaxParts];
  uint32_t n_part[kMaxParts], key[kMaxParts][kMaxTop], id[kMaxParts][kMaxTop];
};

// a number that want of the CTA's keys (PER a thread; 0: none) reach, or more of them if the want-th
// largest is not alone (exact: it is); want keys at least
template <int PER>
CH_DEV uint32_t kth_largest(const uint32_t (&key)[PER], uint32_t want, Shared &sh, bool &exact) {
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
  exact = false;
  for (int bit = top - 1; bit >= 0 && !exact; bit--) {
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
    exact = n == want;
  }
  return k;
}
// want keys of the CTA's (PER a thread, in index order by thread), the largest and of equal ones the
// first: take(e) for each; returns a number that they reach and no other key does, or equal ones only
template <int PER, typename F>
CH_DEV uint32_t choose(const uint32_t (&key)[PER], uint32_t want, Shared &sh, F take) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bool exact;
  const uint32_t edge = kth_largest(key, want, sh, exact);
  if (exact) {
#pragma unroll
    for (int e = 0; e < PER; e++)
      if (key[e] >= edge) take(e);
    __syncthreads();
    return edge;
  }
  __syncthreads();
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
__global__ void __launch_bounds__(kThreads, ctas_of(CAP)) score_rows_kernel(const ScoreArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t r = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // waited for ahead of stores to the first CTA
  const T *row = static_cast<const T *>(a.logits) + r * a.stride;
  const bool vec = ((uintptr_t)row & 15) == 0;
  const uint32_t all_blocks = (a.vocab + kBlock - 1) / kBlock, per_part = (all_blocks + a.parts - 1) / a.parts;
  const uint32_t first = min(part * per_part, all_blocks), blocks = min(per_part, all_blocks - first);
  // in front of the target are larger logits, and equal ones of a lower index: in blocks before its own
  // what is above `least`, in those behind it what is above `given`
  bool asked = false;
  uint32_t at = 0, own_block = 0;
  float given = INFINITY, least = INFINITY;

  // ---- the pass ----
  const Cap cap(CAP ? a.cap : 1.f);
  // below `small` in magnitude the polynomial holds, and nothing is masked
  const float small = !CAP || a.cap < 1e-4f || a.cap > 1e4f ? 0.f : fminf(a.cap * kNearZero, -a.lowest);
  const uint64_t log2e2 = pair_of(kLog2e, kLog2e);
  float m = -INFINITY, s = 0.f, t = 0.f;
  uint32_t before = 0, infinite = 0;
  constexpr int kN = kLane * kRuns;
  auto raise = [&](float m1) {  // m1: largest of the lane's
    if (!(m1 > m)) return;
    const float d = m - m1, f = ex2(d * kLog2e);
    t = f == 0.f ? 0.f : (t + d * s) * f;
    s = f == 0.f ? 0.f : s * f;
    m = m1;
  };
  auto most_of = [](const float (&x)[kN]) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = max3(max3(x[4 * e], x[4 * e + 1], x[4 * e + 2]), x[4 * e + 3], -INFINITY);
    return max3(max3(y[0], y[1], y[2]), y[3], -INFINITY);
  };
  auto block = [&](uint32_t b, float (&x)[kN]) {
    auto index = [&](int e) { return (first + b) * kBlock + (e / kLane) * (kBlock / kRuns) + lane * kLane + e % kLane; };
    const float top = most_of(x);
    const uint32_t most = __reduce_max_sync(0xffffffffu, ordered(clean(top, a.lowest)));
    if (lane == 0) sh.best[b] = most;
    if (first + b == own_block || given == -INFINITY) {
      if (asked) {
#pragma unroll
        for (int e = 0; e < kN; e++) {
          const float y = clean(x[e], a.lowest);
          before += (y > given || (y == given && index(e) < at)) && index(e) < a.vocab;
        }
      }
    } else {
      const float edge = first + b < own_block ? least : given;
      if (top > edge) {
#pragma unroll
        for (int e = 0; e < kN; e++) before += x[e] > edge;
      }
    }
    uint64_t y[kN / 2];
    if constexpr (CAP) {
      float far = 0.f;  // the largest magnitude, NaN if there is one
#pragma unroll
      for (int e = 0; e < kN; e += 2) far = max3_nan(far, fabsf(x[e]), fabsf(x[e + 1]));
      if (__any_sync(0xffffffffu, !(far < small))) {  // one by one
        float most_z = -INFINITY;
#pragma unroll
        for (int e = 0; e < kN; e++) {
          x[e] = x[e] > a.lowest ? cap.any(x[e]) : -INFINITY;
          most_z = fmaxf(most_z, x[e]);
        }
        raise(most_z);
#pragma unroll
        for (int e = 0; e < kN; e++) {
          const float d = x[e] - m, w = x[e] == -INFINITY ? 0.f : ex2(d * kLog2e);
          s += w;
          if (w != 0.f) t = fmaf(d, w, t);  // (0 times -inf would be NaN)
        }
        return;
      }
#pragma unroll
      for (int e = 0; e < kN / 2; e++) {
        y[e] = cap.small(pair_of(x[2 * e], x[2 * e + 1]));
        halves(y[e], x[2 * e], x[2 * e + 1]);
      }
      raise(most_of(x));  // (the polynomial rises, but roundings of neighbours may not)
    } else {
      if (top == INFINITY) {  // the others then weigh nothing
#pragma unroll
        for (int e = 0; e < kN; e++) infinite += x[e] == INFINITY;
      }
      raise(top);
#pragma unroll
      for (int e = 0; e < kN / 2; e++) y[e] = pair_of(x[2 * e], x[2 * e + 1]);
    }
    const uint64_t low = pair_of(-m, -m);
    uint64_t s2 = 0ull, t2 = 0ull;
#pragma unroll
    for (int e = 0; e < kN / 2; e++) {
      uint64_t d = add2(y[e], low);
      float w0, w1;
      if constexpr (!CAP) {  // masked ones and NaN: a weight of 0, and a product of 0 with it
        halves(d, w0, w1);
        d = pair_of(fmaxf(w0, -1e30f), fmaxf(w1, -1e30f));
      }
      halves(mul2(d, log2e2), w0, w1);
      const uint64_t w = pair_of(ex2(w0), ex2(w1));
      s2 = add2(s2, w);
      t2 = fma2(d, w, t2);
    }
    float lo, hi;
    halves(s2, lo, hi), s += lo + hi;
    halves(t2, lo, hi), t += lo + hi;
  };
  // a warp's next block is on its way while this one is added (two at a time: 777 16-bit rows 67.5 us, so
  // 61; 512 capped 16-bit rows of 262,144 116 us, so 105: twice the code)
  Raw<T> next[kRuns];
  auto fetch = [&](uint32_t b) {
    if (b < blocks) {
#pragma unroll
      for (int c = 0; c < (int)kRuns; c++)
        load8(row, (first + b) * kBlock + c * (kBlock / kRuns) + lane * kLane, a.vocab, vec, next[c]);
    }
  };
  fetch(warp);
  // (behind the first loads: the target's logit takes two more on end)
  const int32_t target = a.targets[r];
  asked = target >= 0 && (uint32_t)target < a.vocab;
  if (tid == 0 && part == 0 && target >= 0 && !asked && a.status) atomicOr(a.status, DEV_ERR_BAD_SLOT);
  at = asked ? (uint32_t)target : 0u;
  own_block = at / kBlock;
  given = asked ? clean(value(row[at]), a.lowest) : INFINITY;
  least = asked && given > -INFINITY ? nextafterf(given, -INFINITY) : INFINITY;
  for (uint32_t b = warp; b < blocks; b += kWarps) {
    float x[kN];
#pragma unroll
    for (int c = 0; c < (int)kRuns; c++) values(next[c], x + c * kLane);
    fetch(b + kWarps);
    block(b, x);
  }

  // ---- the part's sums ----
  if (infinite) m = INFINITY, s = (float)infinite, t = 0.f;  // tokens of +inf share the weight
  if (!(m > a.lowest) && !CAP) m = -INFINITY, s = t = 0.f;    // masked ones only
  before = __reduce_add_sync(0xffffffffu, before);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o), t2 = __shfl_xor_sync(0xffffffffu, t, o);
    const float top = fmaxf(m, m2);
    // (equal maxima, infinite ones too, need no factor; far ones have none)
    const float d1 = m == top ? 0.f : fmaxf(m - top, -1e30f), d2 = m2 == top ? 0.f : fmaxf(m2 - top, -1e30f);
    const float f1 = ex2(d1 * kLog2e), f2 = ex2(d2 * kLog2e);
    t = (f1 == 0.f ? 0.f : (t + d1 * s) * f1) + (f2 == 0.f ? 0.f : (t2 + d2 * s2) * f2);
    s = s * f1 + s2 * f2;
    m = top;
  }
  const Sums mine{m, before, s, t};
  if (lane == 0) sh.warps[warp] = mine;
  __syncthreads();

  // ---- the part's sums joined, and its alternatives, sorted ----
  const uint32_t n_blocks = min(a.top, blocks);
  uint32_t n = 0;
  if (warp == 1) {
    const Sums all = join_lanes(sh.warps[lane % kWarps], kWarps);
    if (lane == 0) sh.joined = all;
  }
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
    if (tid == 0) sh.n_list = 0;
    if (n_blocks < a.top) edge = 0;  // fewer blocks than alternatives: any logit may be one
    __syncthreads();
    // the edge as a logit; with masked ones among the chosen every logit may be one
    const bool plain = edge > ordered(-INFINITY);
    const float near_from = plain ? from_ordered(edge) : -INFINITY;
    // the logits of those blocks that reach the last one's maximum; a few loads in flight together
    auto start_of = [&](uint32_t c) { return (first + sh.list[c / kRuns]) * kBlock + c % kRuns * (kBlock / kRuns) + lane * kLane; };
    constexpr int kG = sizeof(T) == 4 ? 2 : 4;
    for (uint32_t c0 = warp; c0 < n_blocks * kRuns; c0 += kG * kWarps) {
      Raw<T> raw[kG];
#pragma unroll
      for (int u = 0; u < kG; u++)
        if (c0 + u * kWarps < n_blocks * kRuns) load8(row, start_of(c0 + u * kWarps), a.vocab, vec, raw[u]);
#pragma unroll
      for (int u = 0; u < kG; u++) {
        if (c0 + u * kWarps >= n_blocks * kRuns) break;
        const uint32_t i = start_of(c0 + u * kWarps);
        float x[kLane];
        values(raw[u], x);
        const float top = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), fmaxf(x[6], x[7]));
        if (plain && !(top >= near_from)) continue;
#pragma unroll
        for (int e = 0; e < (int)kLane; e++) {
          if ((plain ? x[e] >= near_from : true) && i + e < a.vocab) {
            const uint32_t near = atomicAdd(&sh.n_list, 1u);
            if (near < kNear) sh.near[near] = (uint64_t)ordered(clean(x[e], a.lowest)) << 32 | (uint32_t)~(i + e);
          }
        }
      }
    }
    __syncthreads();
    n = sh.n_list;
    __syncthreads();
    if (n > kNear) {  // too many near ones: the first k lanes of 8 logits hold the alternatives
      sort_list(sh.list, n_blocks);  // equal keys go by index
      for (uint32_t c = warp; c < n_blocks * kRuns; c += kWarps) {
        Raw<T> raw;
        float x[kLane];
        load8(row, start_of(c), a.vocab, vec, raw);
        values(raw, x);
        uint32_t best = 0;
#pragma unroll
        for (int e = 0; e < (int)kLane; e++) best = max(best, start_of(c) + e < a.vocab ? ordered(clean(x[e], a.lowest)) : 0u);
        sh.lanes[c * 32 + lane] = best;
      }
      __syncthreads();
      constexpr int kPer = kMaxTop * kRuns * 32 / kThreads;
      uint32_t lanes[kPer];
#pragma unroll
      for (int e = 0; e < kPer; e++) lanes[e] = tid * kPer + e < n_blocks * kRuns * 32 ? sh.lanes[tid * kPer + e] : 0u;
      if (tid == 0) sh.n_list = 0;
      __syncthreads();
      choose(lanes, a.top, sh, [&](int e) { sh.near[atomicAdd(&sh.n_list, 1u)] = tid * kPer + e; });
      // (more than kNear logits lie in more lanes than there are alternatives)
      uint64_t k[2] = {0ull, 0ull};  // (a block's lanes of both halves are in index order)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const uint32_t x = tid + u * kThreads;
        if (x >= a.top * kLane) continue;
        const uint32_t l = (uint32_t)sh.near[x / kLane];
        const uint32_t i = (first + sh.list[l / (kRuns * 32)]) * kBlock + l % (kRuns * 32) * kLane + x % kLane;
        if (i < a.vocab) k[u] = (uint64_t)ordered(clean(value(row[i]), a.lowest)) << 32 | (uint32_t)~i;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 2; u++) sh.near[tid + u * kThreads] = k[u];
      n = min(a.top * kLane, kNear);
      __syncthreads();
    }
  }
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the first CTA has started
  if (tid == kThreads - 1) {
    to_first(&sh.part[part], sh.joined);
    to_first(&sh.n_part[part], min(a.top, min(n, blocks * kBlock)));
  }
  for (uint32_t x = warp; x < n; x += kWarps) {  // a warp ranks one after the other
    const uint64_t k = sh.near[x];
    if (!k) continue;  // past the row's end
    uint32_t rank = 0;
    for (uint32_t j = lane; j < n; j += 32) rank += sh.near[j] > k;
    rank = __reduce_add_sync(0xffffffffu, rank);
    if (rank < a.top && lane == 0) to_first(&sh.key[part][rank], (uint32_t)(k >> 32)), to_first(&sh.id[part][rank], ~(uint32_t)k);
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (part) return;

  // ---- the row ----
  int lanes = 1;
  while (lanes < (int)a.parts) lanes *= 2;
  const Sums all = join_lanes(lane % lanes < (int)a.parts ? sh.part[lane % lanes] : Sums{-INFINITY, 0u, 0., 0.}, lanes);
  const bool any = all.m > -INFINITY;
  const double log_s = any ? log(all.s) : 0.;
  auto logprob = [&](float x) {
    if (x == -INFINITY || (x < INFINITY && all.m == INFINITY)) return -INFINITY;
    if (!CAP && x == INFINITY) return (float)-log_s;
    // the cap as the pass computed it, so that the maximum's is m itself; a block takes the polynomial and `any`
    // does not where x is a rounding away from the border, so not above 0 all the same
    const float y = CAP ? cap.any(x) : x;
    return (float)fmin((double)y - all.m - log_s, 0.);
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
  const uint32_t blocks = (p->vocab + kBlock - 1) / kBlock, slots = num_sms() * ctas_of(p->softcap != 0.f);
  unsigned long long least = ~0ull;
  for (uint32_t parts = 1; parts <= kParts && (parts == 1 || blocks >= parts * std::max(4u, p->top)); parts *= 2) {
    const unsigned long long waves = ((unsigned long long)p->n_rows * parts + slots - 1) / slots;
    const unsigned long long cost = waves * ((blocks + parts - 1) / parts + kPartCost + kTopCost * p->top);
    if (cost < least) least = cost, a.parts = parts;
  }
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
