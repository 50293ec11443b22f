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
// order, so together they keep
//   { i : e_i > e_cut  or  (e_i = e_cut and i <= i_cut) },
// and the draw takes the first kept token, in index order, at which the running sum of
// kept weights exceeds floor(u sum).  No sort is needed: e_cut comes from a radix
// selection over the bits of e (non-negative floats order like their bits; 2^-44 <= e <= 1
// spans 1409 bins of 2^18 ulps, then 2048 of 2^7, then 128), by counts for top-k and by
// sums of w for top-p.
//
// Split.  A cluster of C CTAs takes one row, each CTA a contiguous part of at most 16,384
// tokens that it reads once from global memory and keeps in shared memory as e; the
// passes after that touch shared memory only.  The histograms of a round are added over
// distributed shared memory (CTA r adds every CTA's bins of part r and gives the sums to
// all), two cluster barriers per round.
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

struct Shared {
  unsigned long long hist[kBins], tot[kBins];
  unsigned long long xch[2][kMaxCluster][2];  // what every CTA gives to all, two sets in turn
  unsigned long long warp_a[kWarps];
  uint32_t warp_b[kWarps];
  unsigned long long found[3];  // bin, sum above it, its sum
  uint32_t cut_idx;
  alignas(16) float e[kSlice + 8];
};

CH_DEV float load1(const float *p) { return *p; }
CH_DEV float load1(const __half *p) { return __half2float(*p); }
CH_DEV float load1(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
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
    const uint32_t part = (nb + C - 1) / C, b0 = rank * part, b1 = min(nb, b0 + part);
    for (uint32_t b = b0 + threadIdx.x; b < b1; b += kThreads) {
      unsigned long long sum = 0;
      for (uint32_t c = 0; c < C; c++) sum += *cl.map_shared_rank(&s->hist[b], c);
      for (uint32_t c = 0; c < C; c++) *cl.map_shared_rank(&s->tot[b], c) = sum;
    }
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

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const RowsArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared *s = reinterpret_cast<Shared *>(smem_raw);
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t C = cl.num_blocks(), rank = cl.block_rank(), row = blockIdx.x / C;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t base = min(a.vocab, rank * a.per), n = min(a.vocab - base, a.per);
  const T *x = static_cast<const T *>(a.logits) + (long long)row * a.row_stride + base;
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  int set = 0;

  // ---- the logits, once from global memory; 16-byte loads between a ragged head and tail.
  // Element i lies at e[i], with e shifted so that 16-byte loads meet 16-byte stores. ----
  constexpr uint32_t E = 16 / sizeof(T);
  const uint32_t off = (uint32_t)(((uintptr_t)x / sizeof(T)) % E);
  const uint32_t head = min(n, (E - off) % E), vecs = (n - head) / E;
  float *e = s->e + (off & 3u ? off & 3u : 0u);
  float m = -INFINITY;
  auto put = [&](float v) {
    v = v == v ? v : -INFINITY;  // NaN counts as masked
    if (a.softcap > 0.f) v = tanhf(__fdiv_rn(v, a.softcap)) * a.softcap;
    m = fmaxf(m, v);
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
  m = warp_max(m);
  if (lane == 0) s->warp_b[warp] = __float_as_uint(m);
  __syncthreads();
  for (int w = 0; w < kWarps; w++) m = fmaxf(m, __uint_as_float(s->warp_b[w]));
  exchange(s, cl, C, rank, set, __float_as_uint(m), 0);
  for (uint32_t c = 0; c < C; c++) m = fmaxf(m, __uint_as_float((uint32_t)s->xch[set][c][0]));
  set ^= 1;

  if (m == -INFINITY) {  // nothing to choose from
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
      if (a.kept) a.kept[row] = 0;
    }
    return;
  }

  if (!(temp > 0.f)) {  // greedy: the lowest index of the largest logit
    uint32_t best = 0xFFFFFFFFu;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads)
      if (e[i] == m) best = min(best, base + i);
    best = __reduce_min_sync(0xffffffffu, best);
    __syncthreads();
    if (lane == 0) s->warp_b[warp] = best;
    __syncthreads();
    for (int w = 0; w < kWarps; w++) best = min(best, s->warp_b[w]);
    exchange(s, cl, C, rank, set, best, 0);
    for (uint32_t c = 0; c < C; c++) best = min(best, (uint32_t)s->xch[set][c][0]);
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = (int32_t)best;
      if (a.logprobs) a.logprobs[row] = 0.f;
      if (a.kept) a.kept[row] = 1;
    }
    return;
  }

  // ---- weights; what min-p drops, and what rounds to weight 0, becomes 0 ----
  const float min_p = a.min_p ? a.min_p[row] : 0.f;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const float v = e[i];
    float w = v == m ? 1.0f : expf(__fdiv_rn(v - m, temp));
    if (!(w >= __uint_as_float(kKeyLow)) || (min_p > 0.f && w < min_p && w != 1.0f)) w = 0.f;
    e[i] = w;
  }
  __syncthreads();

  Cut cut{kKeyLow, 0xFFFFFFFFu};
  const int32_t top_k = a.top_k ? a.top_k[row] : 0;
  if (top_k > 0 && (uint32_t)top_k < a.vocab)
    cut = select<true>(s, cl, C, rank, e, n, base, cut, (unsigned long long)top_k, 0.0, set);
  const float top_p = a.top_p ? a.top_p[row] : 1.0f;
  if (top_p < 1.0f) cut = select<false>(s, cl, C, rank, e, n, base, cut, 0, (double)top_p, set);

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
  const float u = a.uniform[row];
  unsigned long long goal = u > 0.f ? (unsigned long long)((double)u * (double)total) : 0ull;
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
