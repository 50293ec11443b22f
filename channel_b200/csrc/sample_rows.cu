// sample_rows.cu -- one token per row of logits (temperature, min-p, top-k, top-p) from
// given uniform numbers; the multi-stream counterpart of the one-row sampler over 64
// candidates (sampler.cu), over the whole vocabulary.
//
// Mathematics.  With m the row's largest (soft-capped) logit, token i has the weight
//   e_i = exp((x_i - m) / T) in f32,   w_i = floor(2^44 e_i) as an integer.
// Everything after the exponential is integer arithmetic, so sums do not depend on the
// order of additions: any split over threads, CTAs and atomics gives the same token.
// 2^18 tokens of weight at most 2^44 sum to at most 2^62.  The tokens are ordered by
// (e descending, index ascending); min-p, top-k and top-p each keep a first part of that
// order, and the draw takes the first kept token, in index order, at which the running sum
// of kept weights exceeds floor(u sum).
//
// Split.  A cluster of C CTAs takes one row, each CTA a contiguous part of at most 16,384
// tokens that it reads once from global memory and keeps in shared memory; everything
// after that touches shared memory only.
//
// Few candidates (the usual case).  min-p bounds the weights that can stay from below, and
// top-k the logits: the k-th largest of the threads' own maxima (32 tokens each) is at most
// the row's k-th largest logit.  The tokens above such a bound -- lowered by more than the
// rounding of the soft cap, the division and the exponential can reorder -- are gathered
// into one CTA, at most 2,048 of them, sorted there by (e, index) and cut.  With top-p alone
// the 512 largest are gathered, and the sum of all weights says whether the cut lies among
// them.
//
// Otherwise e_cut comes from a radix selection over the bits of e (non-negative floats
// order like their bits; 2^-44 <= e <= 1 spans 1409 bins of 2^18 ulps, then 2048 of 2^7, then
// 128), by counts for top-k and by sums of w for top-p, and
//   { i : e_i > e_cut  or  (e_i = e_cut and i <= i_cut) }
// is what stays.  The histograms of a round are added over distributed shared memory (CTA r
// adds every CTA's bins of part r and gives the sums to all), two cluster barriers a round.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <string>

#include "../../include/channel_cuda.h"
#include "common.cuh"
#include "kernels.cuh"

namespace cg = cooperative_groups;

namespace ch {
int set_last_error(int code, const std::string &msg);

namespace {
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr uint32_t kSlice = 16384, kMaxCluster = 16;
constexpr uint32_t kMaxVocab = kSlice * kMaxCluster;
constexpr uint32_t kKeyLow = 0x29800000u;  // bits of 2^-44: the least e of non-zero weight
constexpr uint32_t kKeyOne = 0x3F800000u;  // bits of 1
constexpr uint32_t kBins = 2048;
constexpr float kOne = 17592186044416.0f;  // 2^44

struct RowsArgs {
  const void *logits;
  long long row_stride;
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t *top_k;
  int32_t *tokens, *kept;
  float *logprobs;
  uint32_t vocab, per;  // tokens per CTA
  float softcap;
};

constexpr uint32_t kList = 2048;    // candidates one CTA sorts
constexpr uint32_t kMaxima = 1024;  // bins of the threads' maxima
constexpr int32_t kMostK = 1024;    // largest top-k that goes by the maxima
constexpr uint32_t kNucleus = 512;  // tokens gathered for top-p alone

struct Shared {
  union {
    struct {
      unsigned long long hist[kBins], tot[kBins];
    };
    struct {
      unsigned long long list[kList];  // candidates
      uint32_t maxima[kMaxima], all_maxima[kMaxima];
    };
  };
  unsigned long long xch[2][kMaxCluster][2];  // what every CTA gives to all, two sets in turn
  unsigned long long warp_a[kWarps];
  uint32_t warp_b[kWarps];
  unsigned long long found[3];  // bin, sum above it, its sum
  uint32_t cut_idx, n_list, again, pick;
  alignas(16) float e[kSlice + 8];
};

CH_DEV float load1(const float *p) { return *p; }
CH_DEV float load1(const __half *p) { return __half2float(*p); }
CH_DEV float load1(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
CH_DEV float lowest_of(const float *) { return -3.402823466e38f; }
CH_DEV float lowest_of(const __half *) { return -65504.f; }
CH_DEV float lowest_of(const __nv_bfloat16 *) { return __uint_as_float(0xFF7F0000u); }
CH_DEV void unpack16(const uint4 &r, float (&f)[4], const float *) {
  f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y), f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
}
CH_DEV void unpack16(const uint4 &r, float (&f)[8], const __half *) {
  const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
    f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}
CH_DEV void unpack16(const uint4 &r, float (&f)[8], const __nv_bfloat16 *) {
  const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; i++) f[2 * i] = __uint_as_float(u[i] << 16), f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
}
CH_DEV unsigned long long weight_of(float e) { return (unsigned long long)(e * kOne); }
CH_DEV unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Cut {  // kept: key > key_, or key == key_ and idx <= idx_
  uint32_t key, idx;
  CH_DEV bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= idx); }
};

// gives (a, b) of this CTA to every CTA of the cluster; after the barrier inside,
// s->xch[set][rank] holds every CTA's pair
CH_DEV void exchange(Shared *s, cg::cluster_group &cl, uint32_t C, uint32_t rank, int set, unsigned long long a,
                     unsigned long long b) {
  if (threadIdx.x < C) {
    unsigned long long *to = cl.map_shared_rank(&s->xch[set][rank][0], threadIdx.x);
    to[0] = a;
    to[1] = b;
  }
  cl.sync();
}

// bin of s->tot[0, nb) (from the highest) with sum above < target <= sum above + its own;
// s->found = {bin, sum above, its sum}; bin = nb when the bins hold less than target.
// *all gets the sum of all bins.
CH_DEV void find_bin(Shared *s, uint32_t nb, unsigned long long target) {
  constexpr int kPer = kBins / kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long v[kPer], mine = 0;
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    const uint32_t at = threadIdx.x * kPer + j;
    v[j] = at < nb ? s->tot[nb - 1 - at] : 0;
    mine += v[j];
  }
  unsigned long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) s->warp_a[warp] = inc;
  if (threadIdx.x == 0) s->found[0] = nb;
  __syncthreads();
  unsigned long long above = inc - mine;
  for (int w = 0; w < warp; w++) above += s->warp_a[w];
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    if (above < target && target <= above + v[j]) {
      s->found[0] = nb - 1 - (threadIdx.x * kPer + j);
      s->found[1] = above;
      s->found[2] = v[j];
    }
    above += v[j];
  }
  __syncthreads();
}

// bins [b0, b1) of every CTA's `mine` added up into every CTA's `all`; C (a power of two)
// neighbouring threads share a bin, so that the remote reads are in flight together
template <typename V>
CH_DEV void gather_bins(cg::cluster_group &cl, uint32_t C, V *mine, V *all, uint32_t b0, uint32_t b1) {
  const uint32_t c = threadIdx.x & (C - 1);
  for (uint32_t b = b0 + threadIdx.x / C; b < ((b1 - b0 + 31) & ~31u) + b0; b += kThreads / C) {
    V sum = b < b1 ? *cl.map_shared_rank(&mine[b], c) : V(0);
    for (uint32_t o = 1; o < C; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (b < b1) *cl.map_shared_rank(&all[b], c) = sum;
  }
}

// Narrows `cut` to the first part of the order that holds `target` tokens (COUNT) or,
// with target = 0, the weight ceil(p * sum).
template <bool COUNT>
CH_DEV Cut select(Shared *s, cg::cluster_group &cl, uint32_t C, uint32_t rank, const float *e, uint32_t n,
                  uint32_t base, Cut cut, unsigned long long target, double p, int &set) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t prefix = 0;
  for (int round = 0; round < 3; round++) {
    const uint32_t nb = round == 0 ? ((kKeyOne - kKeyLow) >> 18) + 1 : round == 1 ? 2048 : 128;
    const uint32_t shift = round == 0 ? 18 : round == 1 ? 7 : 0;
    for (uint32_t i = threadIdx.x; i < nb; i += kThreads) s->hist[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t key = __float_as_uint(e[i]);
      if (key == 0 || !cut.keeps(key, base + i)) continue;
      uint32_t bin;
      if (round == 0) {
        bin = (key - kKeyLow) >> 18;
      } else {
        if ((key >> (round == 1 ? 18 : 7)) != prefix) continue;
        bin = (key >> shift) & (nb - 1);
      }
      atomicAdd(&s->hist[bin], COUNT ? 1ull : weight_of(e[i]));
    }
    cl.sync();  // every CTA's bins are complete
    const uint32_t part = (nb + C - 1) / C, b0 = min(nb, rank * part), b1 = min(nb, b0 + part);
    gather_bins(cl, C, s->hist, s->tot, b0, b1);
    cl.sync();  // every CTA has every sum, and is done with every CTA's bins
    if (!COUNT && round == 0) {  // what top-p asks for, from the sum of all weights
      unsigned long long sum = 0;
      for (uint32_t i = threadIdx.x; i < nb; i += kThreads) sum += s->tot[i];
      sum = warp_sum64(sum);
      if (lane == 0) s->warp_a[warp] = sum;
      __syncthreads();
      sum = 0;
      for (int w = 0; w < kWarps; w++) sum += s->warp_a[w];
      __syncthreads();
      const unsigned long long need = (unsigned long long)ceil(p * (double)sum);
      target = need < 1 ? 1 : need;
    }
    find_bin(s, nb, target);
    const uint32_t bin = (uint32_t)s->found[0];
    const unsigned long long above = s->found[1], in_bin = s->found[2];
    if (bin >= nb) return cut;  // fewer tokens than asked for: all stay
    prefix = round == 0 ? bin + (kKeyLow >> 18) : (prefix << (round == 1 ? 11 : 7)) | bin;
    const uint32_t low = prefix << shift;  // the bin's lowest key
    target -= above;
    // the whole bin stays when all its tokens are asked for; by weight, when it holds one token
    const bool whole = COUNT ? target == in_bin : in_bin < 2 * weight_of(__uint_as_float(low));
    if (whole) {
      if (low > cut.key) cut = Cut{low, 0xFFFFFFFFu};
      return cut;
    }
    if (round == 2) {  // one key: the `take` lowest indices of it stay
      const unsigned long long w = COUNT ? 1 : weight_of(__uint_as_float(low));
      const unsigned long long take = (target + w - 1) / w;
      if (take == in_bin / w) {
        if (low > cut.key) cut = Cut{low, 0xFFFFFFFFu};
        return cut;
      }
      // tokens of this key per warp part (a warp owns a contiguous part of the slice)
      const uint32_t seg = ((n + kThreads - 1) / kThreads) * 32, w0 = min(n, warp * seg), w1 = min(n, w0 + seg);
      uint32_t cnt = 0;
      for (uint32_t i = w0 + lane; i < w1; i += 32) {
        const uint32_t key = __float_as_uint(e[i]);
        cnt += key == low && cut.keeps(key, base + i);
      }
      cnt = __reduce_add_sync(0xffffffffu, cnt);
      if (lane == 0) s->warp_b[warp] = cnt;
      __syncthreads();
      uint32_t mine = 0, before = 0;
      for (int k = 0; k < kWarps; k++) {
        if (k < warp) before += s->warp_b[k];
        mine += s->warp_b[k];
      }
      exchange(s, cl, C, rank, set, mine, 0);
      for (uint32_t c = 0; c < rank; c++) before += (uint32_t)s->xch[set][c][0];
      set ^= 1;
      if (before < take && take <= before + cnt) {  // this warp's part holds the last one that stays
        uint32_t left = (uint32_t)take - before;
        for (uint32_t i0 = w0; i0 < w1; i0 += 32) {
          const uint32_t i = i0 + lane, key = i < w1 ? __float_as_uint(e[i]) : 0u;
          const uint32_t hit = __ballot_sync(0xffffffffu, key == low && cut.keeps(key, base + i));
          const uint32_t c = __popc(hit);
          if (left <= c) {
            const int at = __fns(hit, 0, left);
            if (lane < (int)C) *cl.map_shared_rank(&s->cut_idx, lane) = base + i0 + at;
            break;
          }
          left -= c;
        }
      }
      cl.sync();
      return Cut{low, s->cut_idx};
    }
  }
  return cut;
}

// Descending order of a[0, n), padded to a power of two with zeros (no key is 0).  Threads of
// a warp own 64 neighbouring keys, so that short strides need no CTA barrier.
CH_DEV void sort_down(unsigned long long *a, uint32_t n) {
  uint32_t size = 64;
  while (size < n) size <<= 1;
  for (uint32_t i = n + threadIdx.x; i < size; i += kThreads) a[i] = 0;
  __syncthreads();
  for (uint32_t k = 2; k <= size; k <<= 1) {
    for (uint32_t j = k >> 1; j > 0; j >>= 1) {
      for (uint32_t p = threadIdx.x; p < size / 2; p += kThreads) {
        const uint32_t lo = 2 * p - (p & (j - 1)), hi = lo + j;
        const unsigned long long x = a[lo], y = a[hi];
        if ((x < y) == ((lo & k) == 0)) a[lo] = y, a[hi] = x;
      }
      if (j > 32) __syncthreads(); else __syncwarp();
    }
    __syncthreads();
  }
}

// Inclusive sums over the CTA of v (4 neighbouring values per thread); s->warp_a is used.
CH_DEV void scan4(Shared *s, const unsigned long long (&v)[4], unsigned long long (&inc)[4]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  inc[0] = v[0];
#pragma unroll
  for (int j = 1; j < 4; j++) inc[j] = inc[j - 1] + v[j];
  unsigned long long run = inc[3];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += u;
  }
  __syncthreads();
  if (lane == 31) s->warp_a[warp] = run;
  __syncthreads();
  unsigned long long before = run - inc[3];
  for (int w = 0; w < warp; w++) before += s->warp_a[w];
#pragma unroll
  for (int j = 0; j < 4; j++) inc[j] += before;
  __syncthreads();
}

// What one row asks for
struct Row {
  float temp, inv, top_p, min_p, cap, lowest, u;
  int32_t top_k;
  bool quick;  // q_of may divide by multiplication

  // (a logit of -inf or the type's lowest value masks its token and stays as it is)
  CH_DEV float capped(float v) const { return cap > 0.f && v > lowest ? tanhf(__fdiv_rn(v, cap)) * cap : v; }
  // (x - m) / T, correctly rounded.  quick: with r = 1 / T correctly rounded and q = d r, the
  // quotient is q + (d - q T) r, each step one FMA (P. Markstein, IBM J. Res. Dev. 34, 1990);
  // d and T are far from the ends of the range there, and where d / T is below -64 only the
  // sign of the answer matters.
  CH_DEV float q_of(float x, float m) const {
    const float d = x - m;
    if (!quick) return __fdiv_rn(d, temp);
    const float q = d * inv;
    return __fmaf_rn(__fmaf_rn(-temp, q, d), inv, q);
  }
  // e, or 0 where the weight is 0 or min-p drops the token
  CH_DEV float weigh(float x, float m) const {
    float w = 1.0f;
    if (x != m) {
      const float d = x - m;
      if (!(d >= -64.f * temp)) return 0.f;  // far below 2^-44
      w = expf(q_of(x, m));
    }
    if (!(w >= __uint_as_float(kKeyLow)) || (min_p > 0.f && w < min_p && w != 1.0f)) w = 0.f;
    return w;
  }
  // A logit below which no capped one exceeds c: the cap's inverse, lowered until the cap
  // itself says so
  CH_DEV float below(float c) const {
    if (!(cap > 0.f)) return c;
    const float y = __fdiv_rn(c, cap);
    if (!(y > -0.9999f)) return -INFINITY;
    float v = cap * atanhf(fminf(y, 0.9999998f)), step = (fabsf(v) + cap) * 1e-6f;
    for (int i = 0; i < 40; i++) {
      if (capped(v) <= c - cap * 5e-7f) return v;
      v -= step;
      step *= 2.f;
    }
    return -INFINITY;
  }
  // by how much a capped logit has to be lower for its e to be lower too, whatever the
  // roundings of the cap (3 ulp), the difference, the division (31 2^-23) and exp (2 ulp)
  CH_DEV float slack(float m) const { return temp * 1.6e-5f + (cap > 0.f ? cap : fabsf(m)) * 1e-6f; }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const RowsArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared *s = reinterpret_cast<Shared *>(smem_raw);
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t C = cl.num_blocks(), rank = cl.block_rank(), row = blockIdx.x / C;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t base = min(a.vocab, rank * a.per), n = min(a.vocab - base, a.per);
  const T *x = static_cast<const T *>(a.logits) + (long long)row * a.row_stride + base;
  int set = 0;
  for (uint32_t i = threadIdx.x; i < kMaxima; i += kThreads) s->maxima[i] = 0;
  if (threadIdx.x == 0) s->n_list = 0;

  // ---- the logits, once from global memory; 16-byte loads between a ragged head and tail.
  // Element i lies at e[i], with e shifted so that 16-byte loads meet 16-byte stores. ----
  constexpr uint32_t E = 16 / sizeof(T);
  const uint32_t off = (uint32_t)(((uintptr_t)x / sizeof(T)) % E);
  const uint32_t head = min(n, (E - off) % E), vecs = (n - head) / E;
  float *e = s->e + (off & 3u);
  float own = -INFINITY;  // the thread's maximum
  auto put = [&](float v) {
    v = v == v ? v : -INFINITY;  // NaN counts as masked
    own = fmaxf(own, v);
    return v;
  };
  for (uint32_t i = threadIdx.x; i < head; i += kThreads) e[i] = put(load1(x + i));
  const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
#pragma unroll 4
  for (uint32_t j = threadIdx.x; j < vecs; j += kThreads) {
    const uint4 r = xv[j];
    float f[E];
    unpack16(r, f, x);
#pragma unroll
    for (uint32_t k = 0; k < E; k++) f[k] = put(f[k]);
#pragma unroll
    for (uint32_t k = 0; k < E; k += 4)
      *reinterpret_cast<float4 *>(e + head + j * E + k) = make_float4(f[k], f[k + 1], f[k + 2], f[k + 3]);
  }
  for (uint32_t i = head + vecs * E + threadIdx.x; i < n; i += kThreads) e[i] = put(load1(x + i));
  Row r;
  r.temp = a.temperature ? a.temperature[row] : 1.0f;
  r.top_p = a.top_p ? a.top_p[row] : 1.0f;
  r.min_p = a.min_p ? a.min_p[row] : 0.f;
  r.top_k = a.top_k ? a.top_k[row] : 0;
  r.u = a.uniform[row];
  r.cap = a.softcap;
  r.lowest = lowest_of(x);
  r.inv = __frcp_rn(r.temp);
  r.quick = r.temp > 1e-15f && r.temp < 1e15f && (__float_as_uint(r.temp) & 0x7FFFFFu) != 0x7FFFFFu;
  if (r.top_k <= 0 || (uint32_t)r.top_k >= a.vocab) r.top_k = 0;

  // ---- the largest logit m, and the least of the threads' maxima ----
  float m = warp_max(own), least = own > -INFINITY ? own : INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  if (lane == 0) s->warp_a[warp] = (unsigned long long)__float_as_uint(m) << 32 | __float_as_uint(least);
  __syncthreads();
  for (int w = 0; w < kWarps; w++) {
    m = fmaxf(m, __uint_as_float((uint32_t)(s->warp_a[w] >> 32)));
    least = fminf(least, __uint_as_float((uint32_t)s->warp_a[w]));
  }
  exchange(s, cl, C, rank, set, __float_as_uint(m), __float_as_uint(least));
  for (uint32_t c = 0; c < C; c++) {
    m = fmaxf(m, __uint_as_float((uint32_t)s->xch[set][c][0]));
    least = fminf(least, __uint_as_float((uint32_t)s->xch[set][c][1]));
  }
  set ^= 1;

  if (m == -INFINITY) {  // nothing to choose from
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
      if (a.kept) a.kept[row] = 0;
    }
    return;
  }
  const float mc = r.capped(m);  // the largest capped logit, up to the cap's rounding

  if (!(r.temp > 0.f)) {  // greedy: the lowest index of the largest capped logit
    const float low = r.cap > 0.f ? r.below(mc - r.cap * 1e-6f) : m;
    unsigned long long best = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      if (!(e[i] >= low)) continue;
      const uint32_t bits = __float_as_uint(r.capped(e[i])), key = bits >> 31 ? ~bits : bits | 0x80000000u;
      best = max(best, (unsigned long long)key << 32 | (uint32_t)~(base + i));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) s->warp_a[warp] = best;
    __syncthreads();
    for (int w = 0; w < kWarps; w++) best = max(best, s->warp_a[w]);
    exchange(s, cl, C, rank, set, best, 0);
    for (uint32_t c = 0; c < C; c++) best = max(best, s->xch[set][c][0]);
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = (int32_t)~(uint32_t)best;
      if (a.logprobs) a.logprobs[row] = 0.f;
      if (a.kept) a.kept[row] = 1;
    }
    return;
  }

  // ---- few candidates: a bound `low` on the logits that can stay ----
  const bool by_k = r.top_k > 0 && r.top_k <= kMostK, by_p = !(r.min_p > 0.f) && r.top_k == 0 && r.top_p < 1.f;
  if (m < INFINITY && (a.vocab <= kList || by_k || by_p || r.min_p > 0.f)) {
    float low = -INFINITY;
    if (r.min_p > 0.f) low = r.below(mc + r.temp * (logf(fminf(r.min_p, 1.f)) - 1e-5f) - r.slack(mc));
    // with top-p alone, as many as the threads' maxima can bound well
    const uint32_t nucleus = min(kNucleus, C * kThreads / 4);
    if (a.vocab > kList && (by_k || by_p)) {
      const uint32_t want = by_k ? r.top_k : nucleus;
      // the bin of the want-th largest of the threads' maxima
      const float per_bin = least < m ? (kMaxima - 1) / (m - least) : 0.f;
      if (own > -INFINITY) atomicAdd(&s->maxima[min(kMaxima - 1, (uint32_t)((m - own) * per_bin))], 1u);
      cl.sync();
      const uint32_t part = kMaxima / C;
      gather_bins(cl, C, s->maxima, s->all_maxima, rank * part, (rank + 1) * part);
      cl.sync();
      uint32_t v[2] = {s->all_maxima[2 * threadIdx.x], s->all_maxima[2 * threadIdx.x + 1]}, run = v[0] + v[1];
      static_assert(kMaxima == 2 * kThreads, "two bins per thread");
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += u;
      }
      if (lane == 31) s->warp_b[warp] = run;
      if (threadIdx.x == 0) s->pick = kMaxima;
      __syncthreads();
      uint32_t before = run - v[0] - v[1];
      for (int w = 0; w < warp; w++) before += s->warp_b[w];
      if (before < want && want <= before + v[0]) s->pick = 2 * threadIdx.x;
      if (before + v[0] < want && want <= before + v[0] + v[1]) s->pick = 2 * threadIdx.x + 1;
      __syncthreads();
      // at least `want` tokens are not below the bin's lower end
      if (s->pick < kMaxima - 1 && per_bin > 0.f) {
        const float end = m - (s->pick + 1) / per_bin, t0 = end - (fabsf(end) + fabsf(m)) * 1e-6f;
        low = fmaxf(low, r.below(r.capped(t0) - r.slack(mc)));
      }
    }
    // candidates into the first CTA's list, in any order
    Shared *to = cl.map_shared_rank(s, 0);
    unsigned long long mass = 0;  // of all tokens, where top-p alone asks for it
    const bool all_mass = by_p && a.vocab > kList;
    // (with a cap the largest capped logit is only known up to its rounding: the sum of all
    // weights needs it exactly)
    float top = mc;
    if (all_mass && r.cap > 0.f) {
      const float near = r.below(mc - r.cap * 1e-6f);
      for (uint32_t i = threadIdx.x; i < n; i += kThreads)
        if (e[i] >= near) top = fmaxf(top, r.capped(e[i]));
      top = warp_max(top);
      __syncthreads();
      if (lane == 0) s->warp_b[warp] = __float_as_uint(top);
      __syncthreads();
      for (int w = 0; w < kWarps; w++) top = fmaxf(top, __uint_as_float(s->warp_b[w]));
      exchange(s, cl, C, rank, set, __float_as_uint(top), 0);
      for (uint32_t c = 0; c < C; c++) top = fmaxf(top, __uint_as_float((uint32_t)s->xch[set][c][0]));
      set ^= 1;
    }
    for (uint32_t i0 = warp * 32; i0 < n; i0 += kThreads) {
      const uint32_t i = i0 + lane;
      const float v = i < n ? e[i] : -INFINITY;
      if (all_mass) mass += weight_of(r.weigh(r.capped(v), top));
      const bool in = v >= low && v > -INFINITY;
      const uint32_t votes = __ballot_sync(0xffffffffu, in);
      if (!votes) continue;
      uint32_t at = 0;
      if (lane == 0) at = atomicAdd(&to->n_list, __popc(votes));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(votes & ((1u << lane) - 1));
      if (in && at < kList) to->list[at] = (unsigned long long)__float_as_uint(v) << 32 | (base + i);
    }
    if (all_mass) {
      mass = warp_sum64(mass);
      __syncthreads();
      if (lane == 0) s->warp_a[warp] = mass;
      __syncthreads();
      mass = 0;
      for (int w = 0; w < kWarps; w++) mass += s->warp_a[w];
    }
    exchange(s, cl, C, rank, set, mass, 0);
    mass = 0;
    for (uint32_t c = 0; c < C; c++) mass += s->xch[set][c][0];
    set ^= 1;
    const uint32_t count = to->n_list;
    bool found = count <= kList;
    if (found && rank == 0) {
      // capped, weighed, sorted by (e, lower index first)
      float xs[4], best = -INFINITY;
      uint32_t id[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t i = threadIdx.x + j * kThreads;
        const unsigned long long it = i < count ? s->list[i] : 0ull;
        xs[j] = i < count ? r.capped(__uint_as_float((uint32_t)(it >> 32))) : -INFINITY;
        id[j] = (uint32_t)it;
        best = fmaxf(best, xs[j]);
      }
      best = warp_max(best);
      if (lane == 0) s->warp_b[warp] = __float_as_uint(best);
      __syncthreads();
      for (int w = 0; w < kWarps; w++) best = fmaxf(best, __uint_as_float(s->warp_b[w]));
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t i = threadIdx.x + j * kThreads;
        if (i >= count) continue;
        const float w = r.weigh(xs[j], best);
        s->list[i] = w > 0.f ? (unsigned long long)__float_as_uint(w) << 32 | (uint32_t)~id[j] : 0ull;
      }
      __syncthreads();
      sort_down(s->list, count);
      auto w_of = [&](uint32_t i) { return weight_of(__uint_as_float((uint32_t)(s->list[i] >> 32))); };
      // (for top-p alone only the first `nucleus` are sure to come before every other token)
      const uint32_t limit = min(count, r.top_k > 0 ? (uint32_t)r.top_k : all_mass ? nucleus : count);
      unsigned long long v[4], inc[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t i = 4 * threadIdx.x + j;
        v[j] = i < limit ? w_of(i) : 0ull;
      }
      scan4(s, v, inc);
      if (threadIdx.x == kThreads - 1) s->found[0] = inc[3];
      if (threadIdx.x == 0) s->pick = 0;
      __syncthreads();
      const unsigned long long here = s->found[0];
      const unsigned long long whole = all_mass ? mass : here;
      unsigned long long need = ~0ull;  // weight that the kept tokens reach
      if (r.top_p < 1.0f) {
        need = (unsigned long long)ceil((double)r.top_p * (double)whole);
        need = need < 1 ? 1 : need;
      }
      found = !all_mass || need <= here;
      uint32_t kept = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) kept += v[j] > 0 && inc[j] - v[j] < need;
      kept = __reduce_add_sync(0xffffffffu, kept);
      if (lane == 0) atomicAdd(&s->pick, kept);
      __syncthreads();
      kept = s->pick;
      if (found) {
        // the same tokens by index, lowest first: key (index complement, weight's place)
        unsigned long long total = 0, it[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t i = 4 * threadIdx.x + j;
          it[j] = i < kept ? s->list[i] << 32 | s->list[i] >> 32 : 0ull;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++) s->list[4 * threadIdx.x + j] = it[j];
        sort_down(s->list, kept);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t i = 4 * threadIdx.x + j;
          v[j] = i < kept ? weight_of(__uint_as_float((uint32_t)s->list[i])) : 0ull;
        }
        scan4(s, v, inc);
        if (threadIdx.x == kThreads - 1) s->found[0] = inc[3];
        __syncthreads();
        total = s->found[0];
        unsigned long long goal = r.u > 0.f ? (unsigned long long)((double)r.u * (double)total) : 0ull;
        goal = min(goal, total - 1);
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (inc[j] - v[j] <= goal && goal < inc[j]) {
            a.tokens[row] = (int32_t)~(uint32_t)(s->list[4 * threadIdx.x + j] >> 32);
            if (a.logprobs) a.logprobs[row] = (float)log((double)v[j] / (double)total);
            if (a.kept) a.kept[row] = (int32_t)kept;
          }
      }
    }
    if (!all_mass) {
      if (found) {  // the first CTA stays until every other one has read its count
        if (rank == 0) cl.sync();
        return;
      }
    } else {  // the first CTA says whether the cut lay among its candidates
      if (rank == 0 && threadIdx.x < C) *cl.map_shared_rank(&s->again, threadIdx.x) = found ? 0u : 1u;
      cl.sync();
      if (!s->again) return;
    }
    cl.sync();
  }

  // ---- many candidates: weights of all tokens; what min-p drops, and what rounds to weight
  // 0, becomes 0 ----
  float top = m;
  if (r.cap > 0.f) {
    top = -INFINITY;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const float v = r.capped(e[i]);
      e[i] = v;
      top = fmaxf(top, v);
    }
    top = warp_max(top);
    __syncthreads();
    if (lane == 0) s->warp_b[warp] = __float_as_uint(top);
    __syncthreads();
    for (int w = 0; w < kWarps; w++) top = fmaxf(top, __uint_as_float(s->warp_b[w]));
    exchange(s, cl, C, rank, set, __float_as_uint(top), 0);
    for (uint32_t c = 0; c < C; c++) top = fmaxf(top, __uint_as_float((uint32_t)s->xch[set][c][0]));
    set ^= 1;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) e[i] = r.weigh(e[i], top);
  __syncthreads();

  Cut cut{kKeyLow, 0xFFFFFFFFu};
  if (r.top_k > 0) cut = select<true>(s, cl, C, rank, e, n, base, cut, (unsigned long long)r.top_k, 0.0, set);
  if (r.top_p < 1.0f) cut = select<false>(s, cl, C, rank, e, n, base, cut, 0, (double)r.top_p, set);

  // ---- the draw, in index order: warp w owns the part [w * seg, (w + 1) * seg) ----
  const uint32_t seg = ((n + kThreads - 1) / kThreads) * 32, w0 = min(n, warp * seg), w1 = min(n, w0 + seg);
  unsigned long long mass = 0;
  uint32_t cnt = 0;
  for (uint32_t i = w0 + lane; i < w1; i += 32) {
    const uint32_t key = __float_as_uint(e[i]);
    if (key != 0 && cut.keeps(key, base + i)) {
      mass += weight_of(e[i]);
      cnt++;
    }
  }
  mass = warp_sum64(mass);
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  __syncthreads();
  if (lane == 0) s->warp_a[warp] = mass, s->warp_b[warp] = cnt;
  __syncthreads();
  unsigned long long mine = 0, before = 0;
  uint32_t kept = 0;
  for (int w = 0; w < kWarps; w++) {
    if (w < warp) before += s->warp_a[w];
    mine += s->warp_a[w];
    kept += s->warp_b[w];
  }
  exchange(s, cl, C, rank, set, mine, kept);
  unsigned long long total = 0;
  kept = 0;
  for (uint32_t c = 0; c < C; c++) {
    if (c < rank) before += s->xch[set][c][0];
    total += s->xch[set][c][0];
    kept += (uint32_t)s->xch[set][c][1];
  }
  unsigned long long goal = r.u > 0.f ? (unsigned long long)((double)r.u * (double)total) : 0ull;
  goal = min(goal, total - 1);
  if (before <= goal && goal < before + mass) {  // this warp's part holds the token
    unsigned long long run = before;
    for (uint32_t i0 = w0; i0 < w1; i0 += 32) {
      const uint32_t i = i0 + lane, key = i < w1 ? __float_as_uint(e[i]) : 0u;
      const unsigned long long w = key != 0 && cut.keeps(key, base + i) ? weight_of(e[i]) : 0ull;
      unsigned long long inc = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, run + inc > goal);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          a.tokens[row] = (int32_t)(base + i);
          if (a.logprobs) a.logprobs[row] = (float)log((double)w / (double)total);
          if (a.kept) a.kept[row] = (int32_t)kept;
        }
        break;
      }
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
}

template <typename T>
cudaError_t launch_rows(const RowsArgs &a, uint32_t rows, uint32_t C, cudaStream_t stream) {
  const size_t smem = sizeof(Shared);
  cudaError_t e = ensure_smem_attr((const void *)sample_rows_kernel<T>, smem);
  if (e != cudaSuccess) return e;
  if (C > 8) {
    e = cudaFuncSetAttribute(sample_rows_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * C);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_rows_kernel<T>, a);
}

int sample_rows(const ch_sample_rows_args *p, void *stream) {
  if (!p) return set_last_error(CH_EINVAL, "sample_rows: args is NULL");
  if (p->n_rows == 0) return CH_OK;
  if (!p->logits || !p->uniform || !p->tokens) return set_last_error(CH_EINVAL, "sample_rows: NULL argument");
  if (p->vocab == 0 || p->vocab > kMaxVocab)
    return set_last_error(CH_EINVAL, "sample_rows: vocab must be 1.." + std::to_string(kMaxVocab));
  if (p->n_rows > 1u << 20) return set_last_error(CH_EINVAL, "sample_rows: at most 2^20 rows");
  if (p->row_stride < (int64_t)p->vocab && p->n_rows > 1)
    return set_last_error(CH_EINVAL, "sample_rows: row_stride is below vocab");
  if (!(p->softcap >= 0.f) || p->softcap > 3e38f)
    return set_last_error(CH_EINVAL, "sample_rows: softcap must be 0 (none) or positive and finite");
  const size_t es = p->dtype == CH_F32 ? 4 : p->dtype == CH_F16 || p->dtype == CH_BF16 ? 2 : 0;
  if (!es) return set_last_error(CH_EINVAL, "sample_rows: dtype must be CH_F32, CH_F16 or CH_BF16");
  if ((uintptr_t)p->logits % es) return set_last_error(CH_EINVAL, "sample_rows: logits are not aligned to their type");
  RowsArgs a{};
  a.logits = p->logits;
  a.row_stride = p->row_stride;
  a.temperature = p->temperature;
  a.top_p = p->top_p;
  a.min_p = p->min_p;
  a.uniform = p->uniform;
  a.top_k = p->top_k;
  a.tokens = p->tokens;
  a.kept = p->kept;
  a.logprobs = p->logprobs;
  a.vocab = p->vocab;
  a.softcap = p->softcap;
  uint32_t C = 1;
  while (C * kSlice < p->vocab) C *= 2;
  a.per = (p->vocab + C - 1) / C;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = p->dtype == CH_F32   ? launch_rows<float>(a, p->n_rows, C, s)
                        : p->dtype == CH_F16 ? launch_rows<__half>(a, p->n_rows, C, s)
                                             : launch_rows<__nv_bfloat16>(a, p->n_rows, C, s);
  if (e != cudaSuccess) return set_last_error(CH_ECUDA, std::string("sample_rows: ") + cudaGetErrorString(e));
  return CH_OK;
}
}  // namespace
}  // namespace ch

extern "C" int ch_sample_rows(const ch_sample_rows_args *args, void *stream) {
  try {
    return ch::sample_rows(args, stream);
  } catch (...) {
    return CH_ENOMEM;
  }
}
