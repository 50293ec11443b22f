// chunk_attn.cu -- attention of several new tokens per stream over a shared prefix, the stream's
// cached tokens (both in pages) and the new tokens themselves (ch_chunk_attention): packed causal
// prompts and prompt chunks, and trees of drafted tokens.
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - m),
// over the visible positions j; m is the running maximum, and sums are f32.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstring>
#include <string>

#include "../../include/channel_cuda.h"
#include "chunk_tc.cuh"

namespace ch {
int set_last_error(int code, const std::string &msg);

namespace {
constexpr uint32_t kMaxStreams = 4096;
std::atomic<uint64_t> wait_ns{kWaitNs};

// ---------------------------------------------------------------------------
// A warp per (new token, q head): for tensors that no tensor map can describe, and scales that are not
// positive (the maximum of scale s is not that of s) or whose product with log2(e) is not finite.
constexpr int kRowWarps = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32) chunk_rows_kernel(const __grid_constant__ ChunkArgs a) {
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
    if (a.parents) chunk_report_parent(a, s.first, t - s.first);
    chunk_row<T, D>(a, s, lo, t - s.first, hq);
  }
}

template <int D>
constexpr size_t tc_smem() {
  return Tc<D>::kMisc + sizeof(TcShared<D>);
}
static_assert(tc_smem<64>() <= 232448 && tc_smem<128>() <= 232448 && tc_smem<256>() <= 232448, "shared memory per CTA");

// pairs of CTAs that run at once on the current device; 0: the device does not say
uint32_t tc_pairs() {
  constexpr int kMaxDev = 64;
  static std::atomic<int> cache[kMaxDev];  // 0: not asked yet, -1: unavailable
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return 0;
  int c = cache[dev].load(std::memory_order_relaxed);
  if (c == 0) {
    c = -1;
    const void *kernel = (const void *)chunk_tc_kernel<__half, 256>;
    if (ensure_smem_attr(kernel, tc_smem<256>()) == cudaSuccess) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2 * (unsigned)(num_sms() / 2));
      cfg.blockDim = dim3(kTcThreads);
      cfg.dynamicSmemBytes = tc_smem<256>();
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0)
        c = std::min(n, num_sms() / 2);
      else
        (void)cudaGetLastError();
    }
    cache[dev].store(c, std::memory_order_relaxed);
  }
  return c > 0 ? (uint32_t)c : 0u;
}

// workspace: w.cut | w.bad | w.ml | w.o, each on 256 bytes (parts of O are stored 32 bytes at a time); the
// caller's base is on 16 only, so there is room to align it
size_t aligned(size_t bytes) { return (bytes + 255) & ~(size_t)255; }
size_t carve(const ch_chunk_attn_args *p, uint8_t *base, ChunkWork *w) {
  base = reinterpret_cast<uint8_t *>(aligned(reinterpret_cast<uintptr_t>(base)));
  w->pairs = tc_pairs();
  const size_t rows = (size_t)w->pairs * 2 * 2 * kRows;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t *r = base + at;
    at += aligned(bytes);
    return r;
  };
  w->cut = reinterpret_cast<Cut *>(take(w->pairs * sizeof(Cut)));
  w->bad = reinterpret_cast<uint2 *>(take(w->pairs * 2 * sizeof(uint2)));
  w->ml = reinterpret_cast<float2 *>(take(rows * sizeof(float2)));
  w->o = reinterpret_cast<float *>(take(rows * p->head_dim * sizeof(float)));
  return at + 256 - 16;
}

// kernel<<<grid, block, smem, s>>>(args...), which may start before the kernel in front of it
// ends: both kernels wait for that one before they read or write anything
template <typename K, typename... A>
cudaError_t start_kernel(K kernel, dim3 grid, uint32_t block, size_t smem, cudaStream_t s, const A &...args) {
  cudaError_t e = ensure_smem_attr((const void *)kernel, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// the tensors as the copies see them; false where a tensor map cannot describe one
template <int D>
bool encode_maps(const ChunkArgs &a, CUtensorMap (&maps)[5]) {
  using C = Tc<D>;
  std::memset(maps, 0, sizeof(maps));
  const uint32_t tpt = kRows / a.group, ps = 1u << a.shift;
  {  // Q: dim, q head, token; boxes of 64 dims of a kv head's q heads and a CTA's tokens
    const cuuint64_t head = stride_or(a.nq, a.qh, 2 * D);
    const MapDims d{3, {D, a.nq, a.n_tokens}, {head, stride_or(a.n_tokens, a.qs, head)}, {64, a.group, tpt}};
    if (encode_map(&maps[0], a.q, d) != cudaSuccess) return false;
  }
  for (int v = 0; v < 2; v++) {  // new K and V: 64 dims, token, group of dims, head
    const cuuint64_t token = stride_or(a.n_tokens, v ? a.vs : a.ks, 2 * D), head = stride_or(a.nkv, v ? a.vh : a.kh, 2 * D);
    const MapDims d{4, {64, a.n_tokens, D / 64, a.nkv}, {token, 128, head},
                    {64, v ? kKeys : kKeys / 2, (cuuint32_t)(v ? C::kVGroups : C::kGroups), 1}};
    if (encode_map(&maps[1 + v], v ? a.v : a.k, d) != cudaSuccess) return false;
  }
  for (int v = 0; v < 2 && (a.prefix || a.cols); v++) {  // pools: 64 dims, token in the page, group of dims, head, page
    const cuuint64_t token = (cuuint64_t)a.token * 2, head = stride_or(a.nkv, a.head, token), page = stride_or(a.n_pages, a.page, token);
    const cuuint32_t rows = std::min(ps, v ? kKeys : kKeys / 2);
    const cuuint32_t groups = v ? C::kVGroups : rows == kKeys / 2 ? C::kGroups : 1;
    const MapDims d{5, {64, ps, D / 64, a.nkv, a.n_pages}, {token, 128, head, page}, {64, rows, groups, 1, 1}};
    if (a.n_pages == 0 || encode_map(&maps[3 + v], v ? a.v_pool : a.k_pool, d) != cudaSuccess) return false;
  }
  return true;
}

template <typename T, int D>
cudaError_t launch_t(const ChunkArgs &a, const ChunkWork &w, cudaStream_t s) {
  alignas(64) CUtensorMap maps[5];
  if (w.pairs && a.scale > 0.f && a.scale < FLT_MAX / kLog2e && encode_maps<D>(a, maps)) {
    const cudaError_t e = start_kernel(chunk_tc_kernel<T, D>, dim3(2 * w.pairs), kTcThreads, tc_smem<D>(), s, a, w, maps[0], maps[1],
                                       maps[2], maps[3], maps[4]);
    if (e != cudaSuccess) return e;
    return start_kernel(chunk_join_kernel<T, D>, dim3(2 * kRows / kJoinRows, w.pairs), kJoinThreads<D>, 0, s, a, w);
  }
  const unsigned long long rows = (unsigned long long)a.n_tokens * a.nq;
  const unsigned long long grid = (rows + kRowWarps - 1) / kRowWarps, most = 16ull * num_sms();
  chunk_rows_kernel<T, D><<<(uint32_t)(grid < most ? grid : most), kRowWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch(const ChunkArgs &a, const ChunkWork &w, uint32_t D, cudaStream_t s) {
  return D == 64 ? launch_t<T, 64>(a, w, s) : D == 128 ? launch_t<T, 128>(a, w, s) : launch_t<T, 256>(a, w, s);
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
  a.lens = paged ? p->lens : nullptr;  // (positions count without columns too)
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
  a.most = p->parents ? kMaxNodes : ~0u;
  a.scale = p->scale;
  a.status = p->status;
  a.wait_ns = wait_ns.load(std::memory_order_relaxed);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ChunkWork w;
  carve(p, static_cast<uint8_t *>(workspace), &w);
  const cudaError_t e =
      p->dtype == CH_F16 ? launch<__half>(a, w, p->head_dim, s) : launch<__nv_bfloat16>(a, w, p->head_dim, s);
  if (e != cudaSuccess) return set_last_error(CH_ECUDA, std::string("chunk_attention: ") + cudaGetErrorString(e));
  return CH_OK;
}
}  // namespace
}  // namespace ch

extern "C" size_t ch_chunk_attention_workspace(const ch_chunk_attn_args *args) {
  if (ch::check(args) || args->n_tokens == 0 || args->n_streams == 0) return 0;
  ch::ChunkWork w;
  return ch::carve(args, nullptr, &w);
}
extern "C" int ch_chunk_attention(const ch_chunk_attn_args *args, void *workspace, size_t workspace_bytes, void *stream) {
  try {
    return ch::chunk_attention(args, workspace, workspace_bytes, stream);
  } catch (...) {
    return CH_ENOMEM;
  }
}
// For tests: sets after how many nanoseconds the kernel's waits give up, and returns what was set.
extern "C" uint64_t ch_test_chunk_wait_ns(uint64_t ns) { return ch::wait_ns.exchange(ns); }
