// prefix_attn.cuh -- what the two kernels of ch_prefix_attention share: prefix_tc.cu (the
// shared prefix, tcgen05) and prefix_attn.cu (positions read stream by stream, the join).
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "kernels.cuh"

namespace ch {

struct PrefixArgs {
  const void *q, *k, *v;
  void *out;
  const int32_t *prefix_table, *table, *lens;
  long long qs, qh, os, oh;
  long long page, token, head, ts;
  uint32_t n, nq, nkv, group, shift, n_pages, cols, prefix, window;
  uint32_t from;  // first position read stream by stream
  float scale;
  uint32_t *status;
};

CH_DEV float to_f32(__half v) { return __half2float(v); }
CH_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// own tokens of stream b, limited to what its table can hold
CH_DEV uint32_t own_len(const PrefixArgs &a, uint32_t b) {
  const long long len = a.lens[b];
  return (uint32_t)min(max(len, 0ll), (long long)a.cols << a.shift);
}

CH_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
CH_DEV uint32_t pack2(float lo, float hi, const __half *) { return pack_half2(__float2half_rn(lo), __float2half_rn(hi)); }
CH_DEV uint32_t pack2(float lo, float hi, const __nv_bfloat16 *) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// positions stream b attends to: [lo, hi)
CH_DEV void visible(const PrefixArgs &a, uint32_t b, uint32_t &lo, uint32_t &hi) {
  hi = a.prefix + own_len(a, b);  // both below 2^31
  lo = a.window && hi > a.window ? hi - a.window : 0u;
}
// page and row inside it of position j of stream b; -1 when the page is not in the pool
CH_DEV int32_t page_of(const PrefixArgs &a, uint32_t b, uint32_t j, uint32_t &row) {
  const bool shared = j < a.prefix;
  const uint32_t i = shared ? j : j - a.prefix;
  row = i & ((1u << a.shift) - 1);
  const int32_t page = shared ? a.prefix_table[i >> a.shift] : a.table[b * a.ts + (i >> a.shift)];
  if (page < 0 || (uint32_t)page >= a.n_pages) {
    if (a.status) atomicOr(a.status, DEV_ERR_BAD_LIST);
    return -1;
  }
  return page;
}

// The shared prefix's parts in the caller's workspace: per split and kv head the n * group
// query rows (row b * group + g), unnormalised O, and the maximum (units of log2) and sum.
struct PrefixParts {
  float *o;         // [splits][n_kv][n * group][D]
  float2 *ml;       // [splits][n_kv][n * group]
  uint32_t splits;  // 0: the prefix is read stream by stream
};
// splits of the prefix's keys for this shape
uint32_t prefix_tc_splits(uint32_t prefix, uint32_t n, uint32_t group, uint32_t nkv);
// bf16: the type of q and the pools.  cudaErrorNotSupported when a tensor map cannot describe the pools.
cudaError_t launch_prefix_tc(const PrefixArgs &a, const PrefixParts &w, uint32_t D, bool bf16, cudaStream_t s);

}  // namespace ch
