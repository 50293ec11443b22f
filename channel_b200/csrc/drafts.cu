// drafts.cu -- which drafted tokens of each stream's tree the sampled ones confirm
// (ch_accept_drafts).
//
// A stream's walk starts at its node 0 and goes from a node to its first child whose token is
// the one sampled at the node; the nodes on the way are accepted, in packed order over all
// streams.  Bound: latency (the nodes are a few KB): a warp walks a stream, its lanes look at 32
// nodes each step, and since a child lies behind its parent, one pass over the nodes is the whole
// walk.  Then the accepted nodes of the streams in front are added to each rank: in the same launch,
// by a cluster of up to 8 CTAs, for up to 1,024 streams; for more of them by a second launch, with a warp to
// every stream again.  A call, which is the host's time, takes 10.4 us in one launch and 13.2 in two
// (up to 1,024 streams of 16 nodes); on the device 64 streams take 4.1 and 4.1 us, 1,024 8.2 and 5.1, 4,096
// 23.2 and 5.9.
#include <algorithm>
#include <string>

#include "../../include/channel_cuda.h"
#include "common.cuh"
#include "kernels.cuh"

namespace ch {
int set_last_error(int code, const std::string &msg);

namespace {
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kOneThreads = 1024, kOneWarps = kOneThreads / 32, kMaxCtas = 8;  // of the one launch
constexpr uint32_t kOneMost = 1024;  // streams
constexpr uint32_t kMaxStreams = 8192;

struct AcceptArgs {
  const int32_t *drafted, *parents, *starts, *sampled;
  int32_t *counts, *next, *kept;
  uint32_t n, n_tokens;
  uint32_t *status;
};

// packed rows [first, end) of stream b, inside the arrays whatever starts holds
CH_DEV void rows_of(const AcceptArgs &a, uint32_t b, uint32_t &first, uint32_t &end) {
  const long long lo = a.starts[b], hi = a.starts[b + 1], top = a.n_tokens;
  first = (uint32_t)min(max(lo, 0ll), top);
  end = max((uint32_t)min(max(hi, 0ll), top), first);
}

// the walk of stream b, by a warp: its accepted nodes, each node's rank among them (or -1) in kept
CH_DEV uint32_t walk(const AcceptArgs &a, uint32_t b) {
  const int lane = threadIdx.x & 31;
  uint32_t first, end;
  rows_of(a, b, first, end);
  if (lane == 0 && a.status && (a.starts[b] < 0 || a.starts[b + 1] < a.starts[b] || a.starts[b + 1] > (long long)a.n_tokens))
    atomicOr(a.status, DEV_ERR_BAD_LIST);
  const uint32_t n = end - first;
  uint32_t at = 0, count = n ? 1u : 0u;  // the node reached, and nodes accepted
  int32_t want = n ? a.sampled[first] : -1;
  for (uint32_t j0 = 0; j0 < n; j0 += 32) {
    const uint32_t j = j0 + lane;
    const bool in = j < n;
    const int32_t parent = in ? a.parents[first + j] : -1, token = in ? a.drafted[first + j] : -1, then = in ? a.sampled[first + j] : -1;
    int32_t rank = j == 0 ? 0 : -1;
    for (;;) {
      const bool match = want >= 0 && in && j > at && parent == (int32_t)at && token == want;
      const uint32_t who = __ballot_sync(0xffffffffu, match);
      if (!who) break;
      const int l = __ffs(who) - 1;
      if (lane == l) rank = (int32_t)count;
      at = j0 + l;
      want = __shfl_sync(0xffffffffu, then, l);
      count++;
    }
    if (in) a.kept[first + j] = rank;
  }
  if (lane == 0) a.counts[b] = (int32_t)count, a.next[b] = want;
  return count;
}
// rank in stream b -> place among all accepted nodes, `before` of them in the streams in front, by a
// warp (each lane its own nodes of the walk); rows of no stream -> -1
CH_DEV void place(const AcceptArgs &a, uint32_t b, uint32_t before) {
  const int lane = threadIdx.x & 31;
  uint32_t first, end;
  rows_of(a, b, first, end);
  for (uint32_t t = first + lane; t < end; t += 32)
    if (a.kept[t] >= 0) a.kept[t] += (int32_t)before;
  if (b + 1 == a.n)
    for (uint32_t t = end + lane; t < a.n_tokens; t += 32) a.kept[t] = -1;
  if (b == 0)
    for (uint32_t t = lane; t < first; t += 32) a.kept[t] = -1;
}

// all of it by one cluster: a warp takes `per` streams, one after the other
__global__ void __launch_bounds__(kOneThreads) accept_kernel(const AcceptArgs a, uint32_t per) {
  __shared__ uint32_t warps[kOneWarps], ctas[kMaxCtas];  // accepted nodes
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // waited for ahead of stores to other CTAs
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = blockIdx.x, b0 = min(a.n, (rank * kOneWarps + warp) * per), b1 = min(a.n, b0 + per);
  uint32_t mine = 0;
  for (uint32_t b = b0; b < b1; b++) mine += walk(a, b);
  if (lane == 0) warps[warp] = mine;
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  __syncthreads();
  if (warp == 0) {
    const uint32_t sum = __reduce_add_sync(0xffffffffu, warps[lane]);
    if (lane < (int)gridDim.x) {
      uint32_t at;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&ctas[rank])), "r"(lane));
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(sum) : "memory");
    }
    __syncwarp();
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  uint32_t before = 0;
  for (uint32_t r = 0; r < rank; r++) before += ctas[r];
  for (int w = 0; w < warp; w++) before += warps[w];
  for (uint32_t b = b0; b < b1; b++) {
    place(a, b, before);
    before += __shfl_sync(0xffffffffu, lane == 0 ? (uint32_t)a.counts[b] : 0u, 0);
  }
}

__global__ void __launch_bounds__(kThreads) accept_walk_kernel(const AcceptArgs a) {
  const uint32_t b = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (b < a.n) walk(a, b);
}
__global__ void __launch_bounds__(kThreads) accept_place_kernel(const AcceptArgs a) {
  __shared__ uint32_t sums[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t b0 = blockIdx.x * kWarps;
  uint32_t before = 0;  // accepted nodes of the streams in front of b0
  for (uint32_t b = threadIdx.x; b < b0; b += kThreads) before += (uint32_t)a.counts[b];
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) sums[warp] = before;
  __syncthreads();
  before = 0;
  for (int w = 0; w < kWarps; w++) before += sums[w];
  const uint32_t b = b0 + warp;
  for (uint32_t c = b0; c < b && c < a.n; c++) before += (uint32_t)a.counts[c];
  if (b < a.n) place(a, b, before);
}

cudaError_t launch(const AcceptArgs &a, cudaStream_t s) {
  if (a.n > kOneMost) {
    const uint32_t grid = (a.n + kWarps - 1) / kWarps;
    accept_walk_kernel<<<grid, kThreads, 0, s>>>(a);
    accept_place_kernel<<<grid, kThreads, 0, s>>>(a);
    return cudaGetLastError();
  }
  uint32_t ctas = 1;
  while (ctas < kMaxCtas && ctas * kOneWarps < a.n) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kOneThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, accept_kernel, a, (a.n + ctas * kOneWarps - 1) / (ctas * kOneWarps));
}

int accept_drafts(const ch_accept_args *p, void *stream) {
  if (!p) return set_last_error(CH_EINVAL, "accept_drafts: args is NULL");
  if (p->n_streams > kMaxStreams)
    return set_last_error(CH_EINVAL, "accept_drafts: at most " + std::to_string(kMaxStreams) + " streams");
  if (p->n_tokens > 0x7FFFFFFFu) return set_last_error(CH_EINVAL, "accept_drafts: a size is 2^31 or more");
  if ((p->n_streams && (!p->starts || !p->counts || !p->next)) || (p->n_tokens && (!p->drafted || !p->parents || !p->sampled || !p->kept)))
    return set_last_error(CH_EINVAL, "accept_drafts: NULL argument");
  AcceptArgs a{};
  a.drafted = p->drafted;
  a.parents = p->parents;
  a.starts = p->starts;
  a.sampled = p->sampled;
  a.counts = p->counts;
  a.next = p->next;
  a.kept = p->kept;
  a.n = p->n_streams;
  a.n_tokens = p->n_tokens;
  a.status = p->status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (p->n_streams) {
    e = launch(a, s);
  } else if (p->n_tokens) {  // rows of no stream
    e = cudaMemsetAsync(p->kept, 0xFF, p->n_tokens * sizeof(int32_t), s);
  }
  if (e != cudaSuccess) return set_last_error(CH_ECUDA, std::string("accept_drafts: ") + cudaGetErrorString(e));
  return CH_OK;
}
}  // namespace
}  // namespace ch

extern "C" int ch_accept_drafts(const ch_accept_args *args, void *stream) {
  try {
    return ch::accept_drafts(args, stream);
  } catch (...) {
    return CH_ENOMEM;
  }
}
