// chunk_attn.cu -- attention of several new tokens per stream over a shared prefix, the stream's
// cached tokens (both in pages) and the new tokens themselves (ch_chunk_attention): packed causal
// prompts and prompt chunks, and trees of drafted tokens.
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - m),
// over the visible positions j; m is the running maximum, and sums are f32.
#include <string>

#include "../../include/channel_cuda.h"
#include "chunk_attn.cuh"

namespace ch {
int set_last_error(int code, const std::string &msg);

namespace {
constexpr uint32_t kMaxStreams = 4096;

// ---------------------------------------------------------------------------
// A warp per (new token, q head).
constexpr int kRowWarps = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32) chunk_rows_kernel(const ChunkArgs a) {
  const unsigned long long rows = (unsigned long long)a.n_tokens * a.nq;
  const uint32_t step = gridDim.x * kRowWarps;
  if (blockIdx.x == 0) chunk_report(a);
  for (unsigned long long r = blockIdx.x * kRowWarps + (threadIdx.x >> 5); r < rows; r += step) {
    const uint32_t t = (uint32_t)(r / a.nq), hq = (uint32_t)(r % a.nq);
    uint32_t lo = 0, hi = a.n;  // the last stream that starts at or before t
    while (lo + 1 < hi) {
      const uint32_t mid = (lo + hi) >> 1;
      if (a.starts[mid] <= (int32_t)t) lo = mid; else hi = mid;
    }
    const ChunkStream s = chunk_stream(a, lo);
    if (t < s.first || t >= s.first + s.count) continue;  // behind the last stream
    chunk_row<T, D>(a, s, lo, t - s.first, hq);
  }
}

template <typename T, int D>
cudaError_t launch_t(const ChunkArgs &a, cudaStream_t s) {
  const unsigned long long rows = (unsigned long long)a.n_tokens * a.nq;
  const unsigned long long grid = (rows + kRowWarps - 1) / kRowWarps, most = 16ull * num_sms();
  chunk_rows_kernel<T, D><<<(uint32_t)(grid < most ? grid : most), kRowWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch(const ChunkArgs &a, uint32_t D, cudaStream_t s) {
  return D == 64 ? launch_t<T, 64>(a, s) : D == 128 ? launch_t<T, 128>(a, s) : launch_t<T, 256>(a, s);
}

const char *check(const ch_chunk_attn_args *p) {
  if (!p) return "args is NULL";
  if (p->n_streams > kMaxStreams) return "at most 4096 streams";
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return "head_dim must be 64, 128 or 256";
  if (p->n_kv == 0 || p->n_q == 0 || p->n_q % p->n_kv || p->n_q / p->n_kv > 16)
    return "n_q must be n_kv times 1..16";
  if (p->n_q > 1024) return "at most 1024 q heads";
  if (p->n_tokens > 0x7FFFFFFFu || p->n_pages > 0x7FFFFFFFu || p->table_cols > 0x7FFFFFFFu || p->prefix_len > 0x7FFFFFFFu ||
      p->window > 0x7FFFFFFFu)
    return "a size is 2^31 or more";
  if (p->prefix_len || p->table_cols) {
    if (p->page_size < 8 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
      return "page_size must be a power of two from 8 to 256";
    if ((unsigned long long)p->table_cols * p->page_size > 0x7FFFFFFFull) return "the table's columns hold 2^31 tokens or more";
  }
  if (p->dtype != CH_F16 && p->dtype != CH_BF16) return "dtype must be CH_F16 or CH_BF16";
  return nullptr;
}

int chunk_attention(const ch_chunk_attn_args *p, void *workspace, size_t bytes, void *stream) {
  if (const char *why = check(p)) return set_last_error(CH_EINVAL, std::string("chunk_attention: ") + why);
  if (p->n_streams == 0 || p->n_tokens == 0) return CH_OK;
  const bool paged = p->prefix_len || p->table_cols;
  if (!p->q || !p->k || !p->v || !p->out || !p->starts || (paged && (!p->k_pool || !p->v_pool)) ||
      (p->prefix_len && !p->prefix_table) || (p->table_cols && (!p->table || !p->lens)))
    return set_last_error(CH_EINVAL, "chunk_attention: NULL argument");
  // (the stride of a dimension of one element is never used, and may be any number)
  int64_t strides = 0;
  if (p->n_tokens > 1) strides |= p->q_token_stride | p->k_token_stride | p->v_token_stride | p->out_token_stride;
  if (p->n_q > 1) strides |= p->q_head_stride | p->out_head_stride;
  if (p->n_kv > 1) strides |= p->k_head_stride | p->v_head_stride | (paged ? p->head_stride : 0);
  if (paged) strides |= p->token_stride | (p->n_pages > 1 ? p->page_stride : 0);
  if (strides & 7) return set_last_error(CH_EINVAL, "chunk_attention: strides must be multiples of 8 elements");
  uintptr_t at = (uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->out;
  if (paged) at |= (uintptr_t)p->k_pool | (uintptr_t)p->v_pool;
  if (at & 15) return set_last_error(CH_EINVAL, "chunk_attention: q, k, v, out and the pools must be 16-byte aligned");
  const size_t need = ch_chunk_attention_workspace(p);
  if (bytes < need || (need && (!workspace || ((uintptr_t)workspace & 15))))
    return set_last_error(CH_EINVAL, "chunk_attention: workspace must be 16-byte aligned, of " + std::to_string(need) + " bytes");
  ChunkArgs a{};
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.k_pool = p->k_pool;
  a.v_pool = p->v_pool;
  a.out = p->out;
  a.starts = p->starts;
  a.parents = p->parents;
  a.prefix_table = p->prefix_table;
  a.table = p->table;
  a.lens = p->table_cols ? p->lens : nullptr;
  a.qs = p->q_token_stride;
  a.qh = p->q_head_stride;
  a.ks = p->k_token_stride;
  a.kh = p->k_head_stride;
  a.vs = p->v_token_stride;
  a.vh = p->v_head_stride;
  a.os = p->out_token_stride;
  a.oh = p->out_head_stride;
  a.page = p->page_stride;
  a.token = p->token_stride;
  a.head = p->head_stride;
  a.ts = p->table_stride;
  a.n_tokens = p->n_tokens;
  a.n = p->n_streams;
  a.nq = p->n_q;
  a.nkv = p->n_kv;
  a.group = p->n_q / p->n_kv;
  while (paged && (1u << a.shift) < p->page_size) a.shift++;
  a.n_pages = p->n_pages;
  a.cols = p->table_cols;
  a.prefix = p->prefix_len;
  a.window = p->window;
  a.scale = p->scale;
  a.status = p->status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = p->dtype == CH_F16 ? launch<__half>(a, p->head_dim, s) : launch<__nv_bfloat16>(a, p->head_dim, s);
  if (e != cudaSuccess) return set_last_error(CH_ECUDA, std::string("chunk_attention: ") + cudaGetErrorString(e));
  return CH_OK;
}
}  // namespace
}  // namespace ch

extern "C" size_t ch_chunk_attention_workspace(const ch_chunk_attn_args *args) {
  return 0;
}
extern "C" int ch_chunk_attention(const ch_chunk_attn_args *args, void *workspace, size_t workspace_bytes, void *stream) {
  try {
    return ch::chunk_attention(args, workspace, workspace_bytes, stream);
  } catch (...) {
    return CH_ENOMEM;
  }
}
