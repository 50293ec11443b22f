// prefix_attn.cu -- attention of one query token per stream over a prompt that all streams
// share and each stream's own tokens, both in pages (ch_prefix_attention).
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - m),
// over the visible positions j; m is the running maximum, and sums are f32.
#include <cuda_bf16.h>

#include <string>

#include "../../include/channel_cuda.h"
#include "common.cuh"
#include "kernels.cuh"

namespace ch {
int set_last_error(int code, const std::string &msg);

namespace {
constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32;

struct PrefixArgs {
  const void *q, *k, *v;
  void *out;
  const int32_t *prefix_table, *table, *lens;
  long long qs, qh, os, oh;
  long long page, token, head, ts;
  uint32_t n, nq, nkv, group, shift, n_pages, cols, prefix, window;
  float scale;
  uint32_t *status;
};

CH_DEV float to_f32(__half v) { return __half2float(v); }
CH_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
CH_DEV T from_f32(float v);
template <>
CH_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
CH_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// own tokens of stream b, limited to what its table can hold
CH_DEV uint32_t own_len(const PrefixArgs &a, uint32_t b) {
  const int32_t len = a.lens[b];
  if (len <= 0) return 0;
  return (uint32_t)min((unsigned long long)len, (unsigned long long)a.cols << a.shift);
}

// One (stream, q head) per CTA, a warp per key in turn: the plain form, no sharing.
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) attend_row_kernel(const PrefixArgs a) {
  constexpr int EPL = D / 32;
  __shared__ float s_o[kRowWarps][D], s_m[kRowWarps], s_l[kRowWarps];
  const uint32_t b = blockIdx.y, h = blockIdx.x, kvh = h / a.group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T *q = static_cast<const T *>(a.q) + b * a.qs + h * a.qh;
  const T *kp = static_cast<const T *>(a.k) + kvh * a.head, *vp = static_cast<const T *>(a.v) + kvh * a.head;
  float qr[EPL], o[EPL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < EPL; e++) qr[e] = to_f32(q[lane * EPL + e]) * a.scale, o[e] = 0.f;
  const unsigned long long end = (unsigned long long)a.prefix + own_len(a, b);
  const unsigned long long begin = a.window && end > a.window ? end - a.window : 0;
  for (unsigned long long j = begin + warp; j < end; j += kRowWarps) {
    const bool shared = j < a.prefix;
    const uint32_t i = (uint32_t)(shared ? j : j - a.prefix);
    const int32_t page = shared ? a.prefix_table[i >> a.shift] : a.table[b * a.ts + (i >> a.shift)];
    if (page < 0 || (uint32_t)page >= a.n_pages) {
      if (lane == 0 && a.status) atomicOr(a.status, DEV_ERR_BAD_LIST);
      continue;
    }
    const long long at = page * a.page + (long long)(i & ((1u << a.shift) - 1)) * a.token + lane * EPL;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; e++) s = fmaf(qr[e], to_f32(kp[at + e]), s);
    s = warp_sum(s);
    if (s == -INFINITY) continue;
    const float m1 = fmaxf(m, s), c = expf(m - m1), p = expf(s - m1);
    l = l * c + p;
#pragma unroll
    for (int e = 0; e < EPL; e++) o[e] = fmaf(p, to_f32(vp[at + e]), o[e] * c);
    m = m1;
  }
#pragma unroll
  for (int e = 0; e < EPL; e++) s_o[warp][lane * EPL + e] = o[e];
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < kRowWarps; w++) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < kRowWarps; w++)
    if (s_m[w] != -INFINITY) sum += s_l[w] * expf(s_m[w] - top);
  T *out = static_cast<T *>(a.out) + b * a.os + h * a.oh;
  for (int d = threadIdx.x; d < D; d += kRowThreads) {
    float v = 0.f;
    for (int w = 0; w < kRowWarps; w++)
      if (s_m[w] != -INFINITY) v += s_o[w][d] * expf(s_m[w] - top);
    out[d] = from_f32<T>(sum == 0.f ? 0.f : v / sum);
  }
}

template <typename T, int D>
cudaError_t launch_t(const PrefixArgs &a, cudaStream_t s) {
  attend_row_kernel<T, D><<<dim3(a.nq, a.n), kRowThreads, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch(const PrefixArgs &a, uint32_t D, cudaStream_t s) {
  return D == 64 ? launch_t<T, 64>(a, s) : D == 128 ? launch_t<T, 128>(a, s) : launch_t<T, 256>(a, s);
}

const char *check(const ch_prefix_attn_args *p) {
  if (!p) return "args is NULL";
  if (p->n_streams > 65535) return "at most 65535 streams";
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return "head_dim must be 64, 128 or 256";
  if (p->n_kv == 0 || p->n_q == 0 || p->n_q % p->n_kv || p->n_q / p->n_kv > 16)
    return "n_q must be n_kv times 1..16";
  if (p->n_q > 65535) return "at most 65535 q heads";
  if (p->page_size < 8 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
    return "page_size must be a power of two from 8 to 256";
  if (p->n_pages > 0x7FFFFFFFu || p->table_cols > 0x7FFFFFFFu || p->prefix_len > 0x7FFFFFFFu)
    return "a size is 2^31 or more";
  if (p->dtype != CH_F16 && p->dtype != CH_BF16) return "dtype must be CH_F16 or CH_BF16";
  return nullptr;
}

int prefix_attention(const ch_prefix_attn_args *p, void *workspace, size_t bytes, void *stream) {
  if (const char *why = check(p)) return set_last_error(CH_EINVAL, std::string("prefix_attention: ") + why);
  if (p->n_streams == 0) return CH_OK;
  if (!p->q || !p->out || !p->k_pool || !p->v_pool || !p->lens || (p->prefix_len && !p->prefix_table) ||
      (p->table_cols && !p->table))
    return set_last_error(CH_EINVAL, "prefix_attention: NULL argument");
  if ((p->q_stream_stride | p->q_head_stride | p->out_stream_stride | p->out_head_stride | p->page_stride |
       p->token_stride | p->head_stride) & 7)
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      p->dtype == CH_F16 ? launch<__half>(a, p->head_dim, s) : launch<__nv_bfloat16>(a, p->head_dim, s);
  if (e != cudaSuccess) return set_last_error(CH_ECUDA, std::string("prefix_attention: ") + cudaGetErrorString(e));
  return CH_OK;
}
}  // namespace
}  // namespace ch

extern "C" size_t ch_prefix_attention_workspace(const ch_prefix_attn_args *args) {
  if (ch::check(args)) return 0;
  return 0;
}
extern "C" int ch_prefix_attention(const ch_prefix_attn_args *args, void *workspace, size_t workspace_bytes,
                                   void *stream) {
  try {
    return ch::prefix_attention(args, workspace, workspace_bytes, stream);
  } catch (...) {
    return CH_ENOMEM;
  }
}
