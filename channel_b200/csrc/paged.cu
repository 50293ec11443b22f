// paged.cu -- bookkeeping of K/V caches in pages: a step's block tables, slot map,
// positions and row map from the streams' lengths (ch_page_plan), and the step's K/V rows
// into the pages by that slot map (ch_paged_kv_write).
//
// A pool of pages [n_pages][page_size][n_kv][head_dim] holds the K rows of one layer, a
// second one its V rows; a stream owns the pages its block table names, in order, and its
// token i lies in slot table[i / page_size] * page_size + i % page_size.
#include <cuda_bf16.h>

#include <algorithm>
#include <numeric>
#include <string>

#include "../../include/channel_cuda.h"
#include "common.cuh"
#include "kernels.cuh"

namespace ch {
int set_last_error(int code, const std::string &msg);

namespace {
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kMaxStreams = 8192;

// ---------------------------------------------------------------------------
// ch_page_plan.  With h_b = ceil(len_b / page) pages held and a_b = min(ceil((len_b +
// new_b) / page), columns) pages needed, stream b takes the free pages of rank
// F_b .. F_b + a_b - h_b - 1, F the exclusive prefix sum of a - h over the streams; packed
// token t of stream b (S_b <= t < S_{b+1}, S the prefix sum of new) is the stream's token
// i = len_b + t - S_b.
//
// Bound: at one token per stream the launch itself; for packed prompts the 12 bytes written
// per token.  So one launch without any exchange between CTAs: each CTA repeats both
// prefix sums over the (at most 8,192) streams in shared memory and then looks its own
// tokens up by bisection.  Measured on the device: 64 streams of one token 6.2 us, 64 prompts
// of 16 to 16,384 tokens (525,000 tokens, 6.3 MB written) 8.2 us, of which the launch and the
// prefix sums are some 6.
struct PlanArgs {
  const int32_t *lens, *fresh, *free_pages;
  int32_t *table, *lens_out, *starts, *slots, *positions, *rows, *counts;
  uint32_t n, cols, n_free, shift, max_tokens, prefix_len;
  long long stride;
  bool vec;  // the token arrays are 16-byte aligned
  uint32_t *status;
};

CH_DEV int32_t to_i32(long long v) { return (int32_t)min(v, 0x7FFFFFFFll); }
CH_DEV uint32_t pages_for(long long tokens, uint32_t shift) {
  return (uint32_t)((tokens + (1ll << shift) - 1) >> shift);
}

__global__ void __launch_bounds__(kThreads) page_plan_kernel(const PlanArgs a) {
  extern __shared__ uint32_t sm[];
  uint32_t *start = sm;               // [n + 1] first packed token of a stream
  uint32_t *first = sm + a.n + 1;     // [n + 1] first free-page rank of a stream
  __shared__ unsigned long long carry[kWarps];
  __shared__ uint32_t bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t per = (a.n + kThreads - 1) / kThreads;
  const uint32_t b0 = min(a.n, tid * per), b1 = min(a.n, b0 + per);
  if (tid == 0) bad = 0;
  // tokens in the low half, pages in the high half of one sum; both are limited to 2^31 - 1
  // (a stream's share by its 32-bit length, the sums by the clamp below)
  auto of = [&](uint32_t b, long long &len, long long &add, uint32_t &take) {
    len = a.lens[b], add = a.fresh[b];
    const bool neg = len < 0 || add < 0;
    len = max(len, 0ll), add = max(add, 0ll);
    const uint32_t have = pages_for(len, a.shift), after = min(pages_for(len + add, a.shift), a.cols);
    take = after > have ? after - have : 0u;
    // (the new length, and the last position one below prefix + length, have to fit 31 bits)
    return neg || pages_for(len + add, a.shift) > a.cols || len + add + max(a.prefix_len, 1u) > 1ll << 31;
  };
  unsigned long long tok = 0, pg = 0;
  bool odd = false;
  for (uint32_t b = b0; b < b1; b++) {
    long long len, add;
    uint32_t take;
    odd |= of(b, len, add, take);
    tok += (unsigned long long)add;
    pg += take;
  }
  auto scan = [&](unsigned long long v, unsigned long long &all) {  // exclusive over the CTA
    unsigned long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) carry[warp] = inc;
    __syncthreads();
    unsigned long long before = inc - v;
    all = 0;
    for (int w = 0; w < kWarps; w++) {
      if (w < warp) before += carry[w];
      all += carry[w];
    }
    return before;
  };
  unsigned long long tokens, pages;
  tok = scan(tok, tokens);
  pg = scan(pg, pages);
  if (odd) bad = 1;
  constexpr unsigned long long kTop = 0x7FFFFFFFull;
  for (uint32_t b = b0; b < b1; b++) {
    long long len, add;
    uint32_t take;
    of(b, len, add, take);
    start[b] = (uint32_t)min(tok, kTop);
    first[b] = (uint32_t)min(pg, kTop);
    tok += (unsigned long long)add;
    pg += take;
    if (blockIdx.x == 0) {
      a.starts[b] = (int32_t)start[b];
      a.lens_out[b] = to_i32(len + add);
    }
  }
  if (tid == 0) {
    start[a.n] = (uint32_t)min(tokens, kTop);
    first[a.n] = (uint32_t)min(pages, kTop);
    if (blockIdx.x == 0) {
      a.starts[a.n] = (int32_t)start[a.n];
      a.counts[0] = (int32_t)start[a.n];
      a.counts[1] = (int32_t)first[a.n];
    }
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0 && a.status && (bad || pages > a.n_free || tokens > a.max_tokens))
    atomicOr(a.status, DEV_ERR_NO_PAGES);

  // stream b with at[b] <= t < at[b + 1]
  auto find = [&](const uint32_t *at, uint32_t t) {
    uint32_t lo = 0, hi = a.n;
    while (lo + 1 < hi) {
      const uint32_t mid = (lo + hi) >> 1;
      if (at[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
  };
  const uint32_t step = gridDim.x * kThreads, me = blockIdx.x * kThreads + tid;
  // table entries of the pages taken; no token reads these entries (see below), so the
  // table may be read and written in one launch
  const uint32_t taken = first[a.n];
  for (uint32_t r = me; r < taken; r += step) {
    const uint32_t b = find(first, r);
    const uint32_t col = pages_for(max(a.lens[b], 0), a.shift) + (r - first[b]);
    a.table[(long long)b * a.stride + col] = r < a.n_free ? a.free_pages[r] : -1;
  }
  // packed tokens, four per thread
  const uint32_t total = min(start[a.n], a.max_tokens), mask = (1u << a.shift) - 1;
  for (uint32_t g = me; g < (a.max_tokens + 3) / 4; g += step) {
    int32_t slot[4], pos[4], row[4];
    uint32_t b = 4 * g < total ? find(start, 4 * g) : 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t t = 4 * g + j;
      slot[j] = pos[j] = row[j] = -1;
      if (t >= total) continue;
      while (start[b + 1] <= t) b++;
      const long long len = max(a.lens[b], 0), i = len + (t - start[b]);
      const uint32_t have = pages_for(len, a.shift), block = (uint32_t)(i >> a.shift);
      int32_t page = -1;
      if (block < a.cols) {
        if (block < have) {
          page = a.table[(long long)b * a.stride + block];
        } else {
          const uint32_t r = first[b] + (block - have);
          page = r < a.n_free ? a.free_pages[r] : -1;
        }
      }
      if (page >= 0) {
        const long long at = ((long long)page << a.shift) + (i & mask);
        if (at <= 0x7FFFFFFFll)
          slot[j] = (int32_t)at;
        else if (a.status)  // no slot number for it
          atomicOr(a.status, DEV_ERR_NO_PAGES);
      }
      pos[j] = to_i32(i + a.prefix_len);
      row[j] = (int32_t)b;
    }
    if (a.vec && 4 * g + 4 <= a.max_tokens) {
      reinterpret_cast<int4 *>(a.slots)[g] = make_int4(slot[0], slot[1], slot[2], slot[3]);
      reinterpret_cast<int4 *>(a.positions)[g] = make_int4(pos[0], pos[1], pos[2], pos[3]);
      reinterpret_cast<int4 *>(a.rows)[g] = make_int4(row[0], row[1], row[2], row[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (4 * g + j < a.max_tokens) {
          a.slots[4 * g + j] = slot[j];
          a.positions[4 * g + j] = pos[j];
          a.rows[4 * g + j] = row[j];
        }
    }
  }
}

int page_plan(const ch_page_plan_args *p, void *stream) {
  if (!p) return set_last_error(CH_EINVAL, "page_plan: args is NULL");
  if (p->n_streams > kMaxStreams)
    return set_last_error(CH_EINVAL, "page_plan: at most " + std::to_string(kMaxStreams) + " streams");
  if (p->page_size == 0 || (p->page_size & (p->page_size - 1)) || p->page_size > 65536)
    return set_last_error(CH_EINVAL, "page_plan: page_size must be a power of two up to 65536");
  if (!p->starts || !p->counts || (p->n_streams && (!p->lens || !p->new_tokens || !p->lens_out)))
    return set_last_error(CH_EINVAL, "page_plan: NULL argument");
  if (p->n_streams && p->lens_out == p->lens)
    return set_last_error(CH_EINVAL, "page_plan: lens_out must not be lens");
  if (p->n_streams && p->table_cols && !p->table) return set_last_error(CH_EINVAL, "page_plan: table is NULL");
  if (p->n_streams > 1 && p->table_stride < (int64_t)p->table_cols)
    return set_last_error(CH_EINVAL, "page_plan: table_stride is below table_cols");
  if (p->n_free && !p->free_pages) return set_last_error(CH_EINVAL, "page_plan: free_pages is NULL");
  if (p->n_free > 0x7FFFFFFFu || p->max_tokens > 0x7FFFFF00u || p->table_cols > 0x7FFFFFFFu ||
      p->prefix_len > 0x7FFFFFFFu)
    return set_last_error(CH_EINVAL, "page_plan: a size is 2^31 or more");
  if (p->max_tokens && (!p->slots || !p->positions || !p->rows))
    return set_last_error(CH_EINVAL, "page_plan: NULL token array");
  PlanArgs a{};
  a.lens = p->lens;
  a.fresh = p->new_tokens;
  a.free_pages = p->free_pages;
  a.table = p->table;
  a.lens_out = p->lens_out;
  a.starts = p->starts;
  a.slots = p->slots;
  a.positions = p->positions;
  a.rows = p->rows;
  a.counts = p->counts;
  a.n = p->n_streams;
  a.cols = p->table_cols;
  a.n_free = p->n_free;
  a.max_tokens = p->max_tokens;
  a.prefix_len = p->prefix_len;
  a.stride = p->table_stride;
  while ((1u << a.shift) < p->page_size) a.shift++;
  a.vec = (((uintptr_t)p->slots | (uintptr_t)p->positions | (uintptr_t)p->rows) & 15) == 0;
  a.status = p->status;
  // 2,048 tokens per CTA, up to two CTAs per SM: below that a CTA's prefix sums cost more
  // than the tokens it takes
  const uint32_t grid = std::max(1u, std::min((uint32_t)num_sms() * 2, (p->max_tokens + 2047) / 2048));
  const size_t smem = 2 * ((size_t)p->n_streams + 1) * sizeof(uint32_t);
  cudaError_t e = ensure_smem_attr((const void *)page_plan_kernel, smem);
  if (e == cudaSuccess) {
    page_plan_kernel<<<grid, kThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return set_last_error(CH_ECUDA, std::string("page_plan: ") + cudaGetErrorString(e));
  return CH_OK;
}

// ---------------------------------------------------------------------------
// ch_paged_kv_write: pool[slot_t] = (pool type) x_t for K and V rows, rounded to nearest
// when the types differ.  Bound by HBM: each value is read and written once.  A thread
// moves 8 values (16 or 32 bytes in, 16 out) at a time and has four such rows in flight.
// 8,191 tokens of 8 x 256 bf16 (134 MB) take 25 us, 5.4 TB/s, where one row in flight took 28.6;
// a step of 64 tokens 4.1 us, the launch.
struct WriteArgs {
  const void *k, *v;
  long long ks, kh, vs, vh;  // token and head strides of k and v
  const int32_t *slots;
  void *k_pool, *v_pool;
  long long page, token, head;  // pool strides
  uint32_t n_tokens, n_kv, d8, shift;
  long long n_slots;
  uint32_t *status;
};

CH_DEV uint4 to_pool(const float *src, const __half *) {
  const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
  return make_uint4(pack_half2(__float2half_rn(a.x), __float2half_rn(a.y)),
                    pack_half2(__float2half_rn(a.z), __float2half_rn(a.w)),
                    pack_half2(__float2half_rn(b.x), __float2half_rn(b.y)),
                    pack_half2(__float2half_rn(b.z), __float2half_rn(b.w)));
}
CH_DEV uint32_t pack_bf16(float lo, float hi) {
  return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(lo)) |
         ((uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(hi)) << 16);
}
CH_DEV uint4 to_pool(const float *src, const __nv_bfloat16 *) {
  const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
  return make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
}
template <typename T>
CH_DEV uint4 to_pool(const T *src, const T *) {
  return *reinterpret_cast<const uint4 *>(src);
}

template <typename S, typename T>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const WriteArgs a) {
  const uint32_t row = a.n_kv * a.d8;  // 8-value pieces of a token's K (or V) rows
  const S *x = static_cast<const S *>(blockIdx.y ? a.v : a.k);
  T *pool = static_cast<T *>(blockIdx.y ? a.v_pool : a.k_pool);
  const long long ts = blockIdx.y ? a.vs : a.ks, hs = blockIdx.y ? a.vh : a.kh;
  // the grid is a whole number of rows wide, so a thread keeps its place in the row
  const uint32_t me = blockIdx.x * kThreads + threadIdx.x, dt = gridDim.x * kThreads / row;
  const uint32_t r = me % row, h = r / a.d8, c = r % a.d8;
  x += h * hs + c * 8;
  pool += h * a.head + c * 8;
  constexpr uint32_t kU = 4;  // rows whose loads are in flight together
  for (unsigned long long t0 = me / row; t0 < a.n_tokens; t0 += kU * dt) {
    int32_t slot[kU];
    uint4 val[kU];
#pragma unroll
    for (uint32_t u = 0; u < kU; u++) {
      const unsigned long long t = t0 + u * dt;
      slot[u] = -1;
      if (t >= a.n_tokens) continue;
      slot[u] = a.slots[t];
      val[u] = to_pool(x + (long long)t * ts, static_cast<const T *>(nullptr));
    }
#pragma unroll
    for (uint32_t u = 0; u < kU; u++) {
      if (slot[u] < 0) continue;  // padding
      if (slot[u] >= a.n_slots) {
        if (a.status) atomicOr(a.status, DEV_ERR_BAD_SLOT);
        continue;
      }
      const long long page = slot[u] >> a.shift, at = slot[u] & ((1 << a.shift) - 1);
      *reinterpret_cast<uint4 *>(pool + page * a.page + at * a.token) = val[u];
    }
  }
}

template <typename S, typename T>
cudaError_t launch_write(const WriteArgs &a, cudaStream_t s) {
  const uint32_t row = a.n_kv * a.d8;
  const unsigned long long pieces = (unsigned long long)a.n_tokens * row;
  // whole rows: a multiple of row / gcd(row, threads) CTAs; eight CTAs per SM at most for K and
  // for V, or what the rows need
  const uint32_t unit = row / std::gcd(row, (uint32_t)kThreads);
  const unsigned long long want = std::min<unsigned long long>((pieces + kThreads - 1) / kThreads, num_sms() * 8ull);
  const uint32_t grid = (uint32_t)((want + unit - 1) / unit) * unit;
  kv_write_kernel<S, T><<<dim3(grid, 2), kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

int kv_write(const ch_kv_write_args *p, void *stream) {
  if (!p) return set_last_error(CH_EINVAL, "paged_kv_write: args is NULL");
  if (p->n_tokens == 0) return CH_OK;
  if (!p->k || !p->v || !p->slots || !p->k_pool || !p->v_pool)
    return set_last_error(CH_EINVAL, "paged_kv_write: NULL argument");
  if (p->n_kv == 0 || p->head_dim == 0 || p->head_dim % 8 || p->head_dim > 1024 || p->n_kv > 1024)
    return set_last_error(CH_EINVAL, "paged_kv_write: head_dim must be a multiple of 8 up to 1024, n_kv at most 1024");
  if (p->page_size == 0 || (p->page_size & (p->page_size - 1)) || p->page_size > 65536)
    return set_last_error(CH_EINVAL, "paged_kv_write: page_size must be a power of two up to 65536");
  // (the stride of a dimension of one element is never used, and may be any number)
  const int64_t tokens = p->n_tokens > 1 ? p->k_token_stride | p->v_token_stride : 0;
  const int64_t heads = p->n_kv > 1 ? p->k_head_stride | p->v_head_stride | p->head_stride : 0;
  if ((tokens | heads | (p->n_pages > 1 ? p->page_stride : 0) | (p->page_size > 1 ? p->token_stride : 0)) & 7)
    return set_last_error(CH_EINVAL, "paged_kv_write: strides must be multiples of 8 elements");
  if (((uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->k_pool | (uintptr_t)p->v_pool) & 15)
    return set_last_error(CH_EINVAL, "paged_kv_write: k, v and the pools must be 16-byte aligned");
  if (p->n_tokens > 0x7FFFFFFFu || p->n_pages > 0x7FFFFFFFu)
    return set_last_error(CH_EINVAL, "paged_kv_write: a size is 2^31 or more");
  WriteArgs a{};
  a.k = p->k;
  a.v = p->v;
  a.ks = p->k_token_stride;
  a.kh = p->k_head_stride;
  a.vs = p->v_token_stride;
  a.vh = p->v_head_stride;
  a.slots = p->slots;
  a.k_pool = p->k_pool;
  a.v_pool = p->v_pool;
  a.page = p->page_stride;
  a.token = p->token_stride;
  a.head = p->head_stride;
  a.n_tokens = p->n_tokens;
  a.n_kv = p->n_kv;
  a.d8 = p->head_dim / 8;
  while ((1u << a.shift) < p->page_size) a.shift++;
  a.n_slots = (long long)p->n_pages * p->page_size;
  a.status = p->status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  const int from = p->src_dtype, to = p->dst_dtype;
  if (from == CH_F32 && to == CH_F16)
    e = launch_write<float, __half>(a, s);
  else if (from == CH_F32 && to == CH_BF16)
    e = launch_write<float, __nv_bfloat16>(a, s);
  else if (from == to && (to == CH_F16 || to == CH_BF16))
    e = launch_write<uint16_t, uint16_t>(a, s);
  else
    return set_last_error(CH_EINVAL, "paged_kv_write: from CH_F32 to CH_F16 or CH_BF16, or 16-bit rows of one type");
  if (e != cudaSuccess) return set_last_error(CH_ECUDA, std::string("paged_kv_write: ") + cudaGetErrorString(e));
  return CH_OK;
}
}  // namespace
}  // namespace ch

extern "C" int ch_page_plan(const ch_page_plan_args *args, void *stream) {
  try {
    return ch::page_plan(args, stream);
  } catch (...) {
    return CH_ENOMEM;
  }
}
extern "C" int ch_paged_kv_write(const ch_kv_write_args *args, void *stream) {
  try {
    return ch::kv_write(args, stream);
  } catch (...) {
    return CH_ENOMEM;
  }
}
