// score_rows.cu -- log-probability, entropy, rank and top alternatives of given tokens, from whole
// rows of logits (ch_score_rows).
//
// With x the (capped) logits of a row, m their maximum, S = sum e^(x - m), T = sum (x - m) e^(x - m):
//   log p_t = x_t - m - log S,   entropy = -sum p log p = log S - T / S.
// One pass over the row: a thread keeps its own running m, S and T (rescaled when its m grows) and
// the count of logits in front of the given one.  The alternatives need no second pass: a warp
// keeps the largest logit of each block of 256, and the k largest logits of the row (equal ones by
// index) lie in the k blocks with the largest maxima (equal ones by index): if a block is not
// among them, k blocks each hold a logit that comes before all of its own.  Those blocks are read
// again and taken apart the same way, first into a lane's 8 logits, then one by one.
#include <cuda_bf16.h>

#include <algorithm>
#include <string>

#include "../../include/channel_cuda.h"
#include "common.cuh"
#include "kernels.cuh"

namespace ch {
int set_last_error(int code, const std::string &msg);

namespace {
constexpr uint32_t kMaxVocab = 262144, kMaxTop = 64;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr uint32_t kBlock = 256, kLane = 8;  // logits of a block, and of a lane in it
constexpr uint32_t kMaxBlocks = kMaxVocab / kBlock;

struct ScoreArgs {
  const void *logits;
  const int32_t *targets;
  float *logprobs, *entropy, *top_logprobs;
  int32_t *ranks, *top_ids;
  long long stride;
  uint32_t n, vocab, top;
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
CH_DEV void load8(const T *row, uint32_t i, uint32_t vocab, bool vec, float lowest, float (&x)[kLane]) {
  if (vec && i + kLane <= vocab) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < (int)kLane / kPer; c++) {
      const uint4 u = *reinterpret_cast<const uint4 *>(row + i + c * kPer);
      const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
      for (int e = 0; e < kPer; e++) x[c * kPer + e] = clean(value(t[e]), lowest);
    }
  } else {
#pragma unroll
    for (int e = 0; e < (int)kLane; e++) x[e] = i + e < vocab ? clean(value(row[i + e]), lowest) : -INFINITY;
  }
}

// running maximum, sum of e^(x - m) and of (x - m) e^(x - m).  In the sums +inf stands for f32's
// largest value: tokens of +inf then share the weight, and m tells that there are some.
constexpr float kMax = 3.402823466e38f;
struct Sums {
  float m;
  double s, t;
};
CH_DEV Sums join(const Sums &a, const Sums &b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return Sums{m, 0., 0.};
  Sums r{m, 0., 0.};
  for (const Sums *x : {&a, &b}) {
    if (x->m == -INFINITY) continue;
    const double d = (double)fminf(x->m, kMax) - fminf(m, kMax), f = exp(d);
    if (f == 0.) continue;
    r.s += x->s * f;
    r.t += (x->t + d * x->s) * f;
  }
  return r;
}
CH_DEV double shfl_xor(double v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }

// the want-th largest of the CTA's keys, PER a thread (0: none), want of them at least
template <int PER>
CH_DEV uint32_t kth_largest(const uint32_t (&key)[PER], uint32_t want) {
  uint32_t k = 0;
  for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
    uint32_t mine = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) mine += key[e] >= (k | bit);
    uint32_t all = 0;
    if constexpr (PER == 1) {
      all = __syncthreads_count(mine);
    } else {
#pragma unroll
      for (int e = 0; e < PER; e++) all += __syncthreads_count(key[e] >= (k | bit));
    }
    if (all >= want) k |= bit;
  }
  return k;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) score_rows_kernel(const ScoreArgs a) {
  __shared__ uint32_t best[kMaxBlocks];  // a block's largest logit, ordered
  __shared__ uint32_t list[kMaxTop], keys[kMaxTop * 32], n_list, n_at;
  __shared__ uint32_t last_key[kMaxTop * kLane], last_id[kMaxTop * kLane];
  __shared__ Sums parts[kWarps];
  __shared__ uint32_t counts[kWarps], warp_at[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T *row = static_cast<const T *>(a.logits) + blockIdx.x * a.stride;
  const bool vec = ((uintptr_t)row & 15) == 0;
  const int32_t target = a.targets[blockIdx.x];
  const bool asked = target >= 0 && (uint32_t)target < a.vocab;
  if (tid == 0 && target >= 0 && !asked && a.status) atomicOr(a.status, DEV_ERR_BAD_SLOT);
  const float given = asked ? clean(value(row[target]), a.lowest) : 0.f;

  const uint32_t blocks = (a.vocab + kBlock - 1) / kBlock;
  float m = -INFINITY, s = 0.f, t = 0.f;
  uint32_t before = 0;
  for (uint32_t b = warp; b < blocks; b += kWarps) {
    const uint32_t i = b * kBlock + lane * kLane;
    float x[kLane];
    load8(row, i, a.vocab, vec, a.lowest, x);
    float top = x[0];
#pragma unroll
    for (int e = 1; e < (int)kLane; e++) top = fmaxf(top, x[e]);
    if (asked) {
#pragma unroll
      for (int e = 0; e < (int)kLane; e++)
        before += (x[e] > given || (x[e] == given && i + e < (uint32_t)target)) && i + e < a.vocab;
    }
    const uint32_t most = __reduce_max_sync(0xffffffffu, ordered(top));
    if (lane == 0) best[b] = most;
    if (top == -INFINITY) continue;
    if (a.cap != 0.f) {
#pragma unroll
      for (int e = 0; e < (int)kLane; e++) x[e] = x[e] == -INFINITY ? x[e] : a.cap * tanhf(x[e] / a.cap);
      top = x[0];
#pragma unroll
      for (int e = 1; e < (int)kLane; e++) top = fmaxf(top, x[e]);
    } else {
#pragma unroll
      for (int e = 0; e < (int)kLane; e++) x[e] = fminf(x[e], kMax);
    }
    if (top > m) {
      const float d = m - fminf(top, kMax), f = expf(d);
      t = f == 0.f ? 0.f : (t + d * s) * f;
      s = f == 0.f ? 0.f : s * f;
      m = top;
    }
#pragma unroll
    for (int e = 0; e < (int)kLane; e++) {
      const float d = x[e] - fminf(m, kMax), w = expf(d);
      s += w;
      if (w != 0.f) t = fmaf(d, w, t);
    }
  }
  Sums all{m, s, t};
#pragma unroll
  for (int o = 16; o; o >>= 1) all = join(all, Sums{__shfl_xor_sync(0xffffffffu, all.m, o), shfl_xor(all.s, o), shfl_xor(all.t, o)});
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) parts[warp] = all, counts[warp] = before;
  __syncthreads();
  all = parts[0], before = counts[0];
  for (int w = 1; w < kWarps; w++) all = join(all, parts[w]), before += counts[w];
  const bool any = all.m > -INFINITY;
  const double log_s = any ? log(all.s) : 0.;
  auto logprob = [&](float x) {
    if (x == -INFINITY || (x < INFINITY && all.m == INFINITY)) return -INFINITY;
    x = a.cap != 0.f ? a.cap * tanhf(x / a.cap) : fminf(x, kMax);
    return (float)((double)x - fminf(all.m, kMax) - log_s);
  };
  if (tid == 0) {
    a.logprobs[blockIdx.x] = asked ? logprob(given) : 0.f;
    a.entropy[blockIdx.x] = any ? (float)(log_s - all.t / all.s) : 0.f;
    a.ranks[blockIdx.x] = asked ? (int32_t)before + 1 : 0;
  }
  if (!a.top) return;

  // want keys of the CTA's (PER a thread, in index order by thread), the largest and of equal ones
  // the first: calls take(e) for each
  auto choose = [&](auto &key, uint32_t want, auto take) {
    constexpr int kPer = sizeof(key) / sizeof(uint32_t);
    const uint32_t edge = kth_largest(key, want);
    uint32_t over = 0, same = 0;
#pragma unroll
    for (int e = 0; e < kPer; e++) over += key[e] > edge, same += key[e] == edge;
    if (tid == 0) n_at = 0;
    uint32_t inc = same;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) warp_at[warp] = inc;
    __syncthreads();
    over = __reduce_add_sync(0xffffffffu, over);
    if (lane == 0) atomicAdd(&n_at, over);
    uint32_t rank = inc - same;
    for (int w = 0; w < warp; w++) rank += warp_at[w];
    __syncthreads();
    const uint32_t room = want - n_at;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
      if (key[e] > edge) take(e);
      if (key[e] == edge && rank++ < room) take(e);
    }
  };
  // ---- blocks ----
  uint32_t key[kMaxBlocks / kThreads];
#pragma unroll
  for (int e = 0; e < (int)(kMaxBlocks / kThreads); e++) {
    const uint32_t b = tid * (kMaxBlocks / kThreads) + e;
    key[e] = b < blocks ? best[b] : 0u;
  }
  if (tid == 0) n_list = 0;
  const uint32_t n_blocks = min(a.top, blocks);
  choose(key, n_blocks, [&](int e) { list[atomicAdd(&n_list, 1u)] = tid * (kMaxBlocks / kThreads) + e; });
  __syncthreads();
  // in index order: equal keys go by it
  uint32_t mine = 0, place = 0;
  if (tid < n_blocks) {
    mine = list[tid];
    for (uint32_t j = 0; j < n_blocks; j++) place += list[j] < mine;
  }
  __syncthreads();
  if (tid < n_blocks) list[place] = mine;
  __syncthreads();
  // ---- lanes of those blocks: 8 logits each ----
  for (uint32_t c = warp; c < kMaxTop; c += kWarps) {
    uint32_t k = 0;
    if (c < n_blocks) {
      const uint32_t i = list[c] * kBlock + lane * kLane;
      float x[kLane];
      load8(row, i, a.vocab, vec, a.lowest, x);
#pragma unroll
      for (int e = 1; e < (int)kLane; e++) x[0] = fmaxf(x[0], x[e]);
      if (i < a.vocab) k = ordered(x[0]);
    }
    keys[c * 32 + lane] = k;
  }
  __syncthreads();
  uint32_t lanes[kMaxTop * 32 / kThreads];
#pragma unroll
  for (int e = 0; e < (int)(kMaxTop * 32 / kThreads); e++) lanes[e] = keys[tid * (kMaxTop * 32 / kThreads) + e];
  const uint32_t n_lanes = min(a.top, (a.vocab + kLane - 1) / kLane);
  if (tid == 0) n_list = 0;
  __syncthreads();
  choose(lanes, n_lanes, [&](int e) { keys[atomicAdd(&n_list, 1u)] = tid * (kMaxTop * 32 / kThreads) + e; });
  __syncthreads();
  mine = place = 0;
  if (tid < n_lanes) {
    mine = keys[tid];
    for (uint32_t j = 0; j < n_lanes; j++) place += keys[j] < mine;
  }
  __syncthreads();
  if (tid < n_lanes) keys[place] = mine;
  __syncthreads();
  // ---- logits of those lanes ----
  uint32_t one[1] = {0u}, id = 0;
  if (tid < n_lanes * kLane) {
    const uint32_t l = keys[tid / kLane];
    id = list[l / 32] * kBlock + (l % 32) * kLane + tid % kLane;
    if (id < a.vocab) one[0] = ordered(clean(value(row[id]), a.lowest));
  }
  if (tid == 0) n_list = 0;
  __syncthreads();
  choose(one, a.top, [&](int) {
    const uint32_t at = atomicAdd(&n_list, 1u);
    last_key[at] = one[0];
    last_id[at] = id;
  });
  __syncthreads();
  if (tid < a.top) {
    const uint32_t k = last_key[tid], i = last_id[tid];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < a.top; j++) rank += last_key[j] > k || (last_key[j] == k && last_id[j] < i);
    const size_t at = (size_t)blockIdx.x * a.top + rank;
    a.top_ids[at] = (int32_t)i;
    a.top_logprobs[at] = logprob(from_ordered(k));
  }
}

template <typename T>
cudaError_t launch(const ScoreArgs &a, cudaStream_t s) {
  score_rows_kernel<T><<<a.n, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

int score_rows(const ch_score_args *p, void *stream) {
  if (!p) return set_last_error(CH_EINVAL, "score_rows: args is NULL");
  if (p->n_rows == 0) return CH_OK;
  if (p->vocab == 0 || p->vocab > kMaxVocab)
    return set_last_error(CH_EINVAL, "score_rows: vocab must be 1.." + std::to_string(kMaxVocab));
  if (p->top > kMaxTop || p->top > p->vocab)
    return set_last_error(CH_EINVAL, "score_rows: top must be at most " + std::to_string(kMaxTop) + " and vocab");
  if (p->n_rows > 0x7FFFFFFFu) return set_last_error(CH_EINVAL, "score_rows: a size is 2^31 or more");
  if (!p->logits || !p->targets || !p->logprobs || !p->entropy || !p->ranks || (p->top && (!p->top_ids || !p->top_logprobs)))
    return set_last_error(CH_EINVAL, "score_rows: NULL argument");
  if (!(p->softcap >= 0.f) || p->softcap > 3.402823466e38f)
    return set_last_error(CH_EINVAL, "score_rows: softcap must be a number that is not negative");
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
