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
// top-k the logits: if each of the C CTAs has ceil(k / C) tokens not below b, the k largest
// logits are not below b, and the threads' own maxima (32 tokens each) give each CTA such a
// b.  The tokens above such a bound -- lowered by more than the rounding of the soft cap, the
// division and the exponential can reorder -- are gathered into one CTA in index order, at
// most 2,048 of them, and weighed and cut there.
//
// The cut.  By counts for top-k and by sums of w for top-p, a radix selection over the bits
// of e (non-negative floats order like their bits; 2^-44 <= e <= 1 spans 1409 bins of 2^18
// ulps, then 512 of 2^9, then 512) finds e_cut and i_cut with which
//   { i : e_i > e_cut  or  (e_i = e_cut and i <= i_cut) }
// stays: over the gathered tokens in one CTA (up to 256 are ranked by comparing all with all),
// or else over all CTAs' tokens, whose histograms are added over distributed shared memory
// (CTA r adds every CTA's bins of part r and gives the sums to all, two cluster barriers a
// round).  After the first round only the tokens of one bin matter: each CTA collects their
// keys, and 16-bit logits, whose bins often hold one key, need no further round then.  The
// tokens of a bin share the exponent of e, so a bin's sum of w is exactly a count and a sum of
// low mantissa bits, both in 32 bits: 64-bit shared-memory atomics were several times slower.
//
// Bound.  For one row the chain of passes, scans and cluster barriers, not HBM.  One row of
// 262,144 capped f32 logits takes 12 us with top-k 64 and 31 us by top-p alone (58,000 cycles:
// the cap 7,400, weights and first bins 9,400, a round of the cut 7,000 to 8,000, collecting a
// bin's tokens 5,000, the kept sum 3,300).  64 such rows of mixed settings take 46 to 47 us, where
// reading them takes 10.4; 48 rows of 100,003 bf16 logits by top-p and min-p 35 to 37 us.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <type_traits>

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
constexpr uint32_t kBins = 1409, kSub = 512;  // of the first round, of the others
constexpr uint32_t kFew = 256;     // candidates that are ranked by comparing all with all
constexpr int32_t kLeft = -2;      // the token of a row that the second kernel takes

// Which rows a launch takes: all; those whose settings leave many candidates; those of the rest
// whose token is kLeft
enum class Rows { kAll, kMany, kLeftOver };
struct RowsArgs {
  const void *logits;
  long long row_stride;
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t *top_k;
  int32_t *tokens, *kept;
  float *logprobs;
  uint32_t rows, vocab, per;  // per: tokens per CTA
  float softcap;
  Rows which;
};

constexpr uint32_t kList = 2048;    // candidates one CTA takes
constexpr uint32_t kMaxima = 1024;  // bins of a CTA's threads' maxima
constexpr int32_t kMostK = 1024;    // largest top-k that goes by the maxima

struct Shared {
  union {
    unsigned long long tot[kBins];
    uint32_t maxima[kMaxima];
  };
  uint32_t cnt[kBins], low[kBins];  // tokens of a bin, and their sum above the bin's least
  float list[kList];                // candidates: logits, then weights, by index
  uint32_t list_id[kList];
  unsigned long long xch[2][kMaxCluster][2];  // what every CTA gives to all, two sets in turn
  unsigned long long warp_a[kWarps];
  uint32_t warp_b[kWarps];
  unsigned long long found[3];  // bin, sum above it, its sum
  uint32_t cut_at, pick, least, most;
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
CH_DEV void answer(const RowsArgs &a, uint32_t row, int32_t token, float logprob, int32_t kept) {
  a.tokens[row] = token;
  if (a.logprobs) a.logprobs[row] = logprob;
  if (a.kept) a.kept[row] = kept;
}
// A token's place in the order of greedy rows: by its (capped) logit, equal ones by index from the
// lowest on.  + 0.0f: zeros of either sign are equal, and their bits are not.
CH_DEV unsigned long long greedy_key(float x, uint32_t token) {
  const uint32_t bits = __float_as_uint(x + 0.0f), key = bits >> 31 ? ~bits : bits | 0x80000000u;
  return (unsigned long long)key << 32 | (uint32_t)~token;
}
// floor(2^44 e) for 0 <= e <= 1: the mantissa shifted (a conversion to 64 bits is many times slower)
CH_DEV unsigned long long weight_of(float e) {
  const uint32_t bits = __float_as_uint(e), mant = (bits & 0x7FFFFFu) | 0x800000u;
  return (unsigned long long)mant << 21 >> min(127u - (bits >> 23), 63u);
}
CH_DEV unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Cut {  // kept: key > key_, or key == key_ and place <= at_
  uint32_t key, at;
  CH_DEV bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= at); }
};

// The tokens a cut is taken over: those of all CTAs of the cluster, place = base + i, or
// (CLUSTER false) the list of this CTA
template <bool CLUSTER>
struct Tokens {
  Shared *s;
  cg::cluster_group &cl;
  uint32_t C, rank;  // 1, 0 for a list
  const float *e;    // weights
  uint32_t n, base;
  int &set;
  bool coarse;  // logits of 16 bits: a bin often holds one key only

  CH_DEV void sync() const {
    if (CLUSTER) cl.sync(); else __syncthreads();
  }
  // gives (a, b) of this CTA to every CTA; afterwards s->xch[set][c] holds CTA c's pair
  CH_DEV void exchange(unsigned long long a, unsigned long long b) const {
    if (threadIdx.x < C) {
      unsigned long long *to = &s->xch[set][rank][0];
      if (CLUSTER) to = cl.map_shared_rank(to, threadIdx.x);
      to[0] = a;
      to[1] = b;
    }
    sync();
  }
};

// The bins of a round: tokens of one bin differ in the `shift` low bits of their keys only.
// (16,384 tokens of a CTA sum to less than 2^32 of low bits.)
// Below 2^-21 a weight loses mantissa bits: there the sum is of weights above the bin's least.
struct Round {
  uint32_t bins, shift;
  CH_DEV uint32_t low_of(uint32_t key) const {
    const uint32_t lost = 127 - (key >> 23) > 21 ? 106 - (key >> 23) : 0u, mant = (key & 0x7FFFFFu) | 0x800000u;
    return (mant >> lost) - ((mant & ~((1u << shift) - 1)) >> lost);
  }
  CH_DEV unsigned long long sum_of(uint32_t count, uint32_t low, uint32_t key0) const {
    const uint32_t ex = 127 - (key0 >> 23);
    return count * weight_of(__uint_as_float(key0)) + ((unsigned long long)low << (ex > 21 ? 0 : 21 - ex));
  }
};

// bin of s->tot[0, nb) (from the highest) with sum above < target <= sum above + its own;
// s->found = {bin, sum above, its sum}; bin = nb when the bins hold less than target.
// target 0: ceil(p * the sum of all bins), at least 1.  Returns the target.
CH_DEV unsigned long long find_bin(Shared *s, uint32_t nb, unsigned long long target, double p) {
  constexpr int kPer = (kBins + kThreads - 1) / kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t per = (nb + kThreads - 1) / kThreads;
  unsigned long long v[kPer], mine = 0;
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    const uint32_t at = threadIdx.x * per + j;
    v[j] = j < (int)per && at < nb ? s->tot[nb - 1 - at] : 0;
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
  unsigned long long above = inc - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    const unsigned long long x = s->warp_a[w];
    if (w < warp) above += x;
    all += x;
  }
  if (target == 0) {
    const unsigned long long need = (unsigned long long)ceil(p * (double)all);
    target = need < 1 ? 1 : need;
  }
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    if (above < target && target <= above + v[j]) {
      s->found[0] = nb - 1 - (threadIdx.x * per + j);
      s->found[1] = above;
      s->found[2] = v[j];
    }
    above += v[j];
  }
  __syncthreads();
  return target;
}

// The bin of a token in the first round, added to the CTA's bins
template <bool COUNT>
CH_DEV void add_first(Shared *s, uint32_t key) {
  const Round rd = {kBins, 18};
  const uint32_t bin = (key - kKeyLow) >> 18;
  atomicAdd(&s->cnt[bin], 1u);
  if (!COUNT) atomicAdd(&s->low[bin], rd.low_of(key));
}

// Narrows `cut` to the first part of the order that holds `target` tokens (COUNT) or the
// weight ceil(p * sum of all kept so far).  binned: the first round's bins are filled already.
template <bool COUNT, bool CLUSTER>
CH_DEV Cut select(const Tokens<CLUSTER> &t, Cut cut, unsigned long long target, double p, bool binned) {
  Shared *s = t.s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float *e = t.e;
  uint32_t prefix = 0;
  unsigned long long in_bin = 0;
  // one key holds what is left, `in_bin` in all: its first places stay
  auto of_one_key = [&](uint32_t low) {
    const unsigned long long w = COUNT ? 1 : weight_of(__uint_as_float(low));
    const unsigned long long take = (target + w - 1) / w;
    if (take == in_bin / w) {
      if (low > cut.key) cut = Cut{low, 0xFFFFFFFFu};
      return cut;
    }
    // thread t counts those of the places from t * run on (an odd run spreads the lanes over the banks)
    const uint32_t run = ((t.n + kThreads - 1) / kThreads) | 1u, p0 = threadIdx.x * run, p1 = min(t.n, p0 + run);
    auto is = [&](uint32_t i) { return __float_as_uint(e[i]) == low && cut.keeps(low, t.base + i); };
    uint32_t cnt = 0;
#pragma unroll 4
    for (uint32_t i = p0; i < p1; i++) cnt += is(i);
    const uint32_t all = __reduce_add_sync(0xffffffffu, cnt);
    if (lane == 0) s->warp_b[warp] = all;
    __syncthreads();
    uint32_t mine = 0, before = 0;
    for (int k = 0; k < kWarps; k++) {
      if (k < warp) before += s->warp_b[k];
      mine += s->warp_b[k];
    }
    t.exchange(mine, 0);
    for (uint32_t c = 0; c < t.rank; c++) before += (uint32_t)s->xch[t.set][c][0];
    t.set ^= 1;
    if (before < take && take <= before + all) {  // this warp's part holds the last one that stays
      uint32_t inc = cnt;  // the lane that does, then the place in its run
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      const int owner = __ffs(__ballot_sync(0xffffffffu, before + inc >= take)) - 1;
      uint32_t left = (uint32_t)take - before - __shfl_sync(0xffffffffu, inc - cnt, owner);
      const uint32_t q0 = (warp * 32 + owner) * run, q1 = min(t.n, q0 + run);
      for (uint32_t i0 = q0; i0 < q1; i0 += 32) {
        const uint32_t i = i0 + lane;
        const bool hit = i < q1 && is(i);
        const uint32_t hits = __ballot_sync(0xffffffffu, hit), c = __popc(hits);
        if (left <= c) {
          if (hit && __popc(hits & ((1u << lane) - 1)) == (int)left - 1) {
            for (uint32_t c = 0; c < t.C; c++) (CLUSTER ? *t.cl.map_shared_rank(&s->cut_at, c) : s->cut_at) = t.base + i;
          }
          break;
        }
        left -= c;
      }
    }
    t.sync();
    return Cut{low, s->cut_at};
  };
  for (int round = 0; round < 3; round++) {
    const Round rd = {round == 0 ? kBins : kSub, round == 0 ? 18u : round == 1 ? 9u : 0u};
    const uint32_t nb = rd.bins;
    if (round > 0 || !binned) {
      for (uint32_t i = threadIdx.x; i < nb; i += kThreads) s->cnt[i] = s->low[i] = 0;
      __syncthreads();
    }
    if (round == 0) {
      for (uint32_t i = threadIdx.x; i < t.n && !binned; i += kThreads) {
        const uint32_t key = __float_as_uint(e[i]);
        if (key != 0 && cut.keeps(key, t.base + i)) add_first<COUNT>(s, key);
      }
    } else {
      // the tokens of the bin found last, collected in the first of these rounds where they fit
      auto matches = [&](uint32_t key, uint32_t i) { return key >> (rd.shift + 9) == prefix && cut.keeps(key, t.base + i); };
      if (CLUSTER && round == 1) {
        if (threadIdx.x == 0) s->pick = 0, s->least = 0xFFFFFFFFu, s->most = 0;
        __syncthreads();
        uint32_t least = 0xFFFFFFFFu, most = 0;
        // 16-byte groups around the tokens; the places that fill them up have weight 0
        const uint32_t shift = (uint32_t)(e - s->e);
        for (uint32_t g = threadIdx.x; g < (shift + t.n + 3) / 4; g += kThreads) {
          const uint4 four = reinterpret_cast<const uint4 *>(s->e)[g];
          const uint32_t keys[4] = {four.x, four.y, four.z, four.w};
          bool any = false;
#pragma unroll
          for (int j = 0; j < 4; j++) any |= keys[j] >> 18 == prefix;
          if (!any) continue;
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (matches(keys[j], 4 * g + j - shift)) {
              const uint32_t at = atomicAdd(&s->pick, 1u);
              if (at < kList) s->list_id[at] = keys[j];
              least = min(least, keys[j]);
              most = max(most, keys[j]);
            }
        }
        if (t.coarse) {
          least = __reduce_min_sync(0xffffffffu, least);
          most = __reduce_max_sync(0xffffffffu, most);
          if (lane == 0 && most) atomicMin(&s->least, least), atomicMax(&s->most, most);
        }
        __syncthreads();
        if (t.coarse && threadIdx.x < t.C) {  // read after the next barrier of the cluster
          unsigned long long *to = t.cl.map_shared_rank(&s->xch[t.set][t.rank][0], threadIdx.x);
          to[0] = s->least;
          to[1] = s->most;
        }
      }
      const bool listed = CLUSTER && s->pick <= kList;
      const uint32_t many = listed ? s->pick : t.n;
      // few bins hold many tokens here (16-bit logits have few distinct values), and additions
      // to one address go one by one: a warp adds its first bins once each
      for (uint32_t i0 = warp * 32; i0 < many; i0 += kThreads) {
        const uint32_t i = i0 + lane;
        uint32_t key = i < many ? listed ? s->list_id[i] : __float_as_uint(e[i]) : 0u;
        if (listed ? key >> (rd.shift + 9) != prefix : !matches(key, i)) key = 0;
        const uint32_t bin = (key >> rd.shift) & (kSub - 1);
        uint32_t left = __ballot_sync(0xffffffffu, key != 0);
        for (int k = 0; k < 4 && left; k++) {
          const int first = __ffs(left) - 1;
          const uint32_t its = __shfl_sync(0xffffffffu, bin, first);  // by every lane
          const bool mine = key != 0 && bin == its;
          const uint32_t same = __ballot_sync(0xffffffffu, mine);
          if (lane == first) atomicAdd(&s->cnt[bin], __popc(same));
          if (!COUNT && rd.shift > 0) {
            const uint32_t sum = __reduce_add_sync(0xffffffffu, mine ? rd.low_of(key) : 0u);
            if (lane == first) atomicAdd(&s->low[bin], sum);
          }
          left &= ~same;
        }
        if ((left >> lane) & 1u) {
          atomicAdd(&s->cnt[bin], 1u);
          if (!COUNT && rd.shift > 0) atomicAdd(&s->low[bin], rd.low_of(key));
        }
      }
    }
    t.sync();  // every CTA's bins are complete
    if (CLUSTER && t.coarse && round == 1) {  // one key: nothing is left to find
      unsigned long long least = ~0ull, most = 0;
      for (uint32_t c = 0; c < t.C; c++) least = min(least, s->xch[t.set][c][0]), most = max(most, s->xch[t.set][c][1]);
      t.set ^= 1;
      if (least == most) return of_one_key((uint32_t)most);
    }
    const uint32_t key_base = round == 0 ? kKeyLow : prefix << (rd.shift + 9);
    if (CLUSTER) {
      // this CTA's part of the bins: warp w reads CTA w's (neighbouring words), the sums go
      // through the list's memory, and warp w gives them to CTA w
      const uint32_t part = (nb + t.C - 1) / t.C, b0 = min(nb, t.rank * part), mine = min(nb, b0 + part) - b0;
      unsigned long long *sums = reinterpret_cast<unsigned long long *>(s->list);  // [C][part]
      static_assert((kBins + kMaxCluster) * sizeof(unsigned long long) <= sizeof(s->list) + sizeof(s->list_id), "room");
      static_assert((kSub + kMaxCluster) * sizeof(unsigned long long) <= sizeof(s->list), "beside the collected tokens");
      for (uint32_t c = warp; c < t.C; c += kWarps) {
        const uint32_t *cnt = t.cl.map_shared_rank(s->cnt, c) + b0, *lows = t.cl.map_shared_rank(s->low, c) + b0;
#pragma unroll 4
        for (uint32_t b = lane; b < mine; b += 32) {
          const uint32_t n = cnt[b];
          sums[c * part + b] = COUNT ? n : rd.sum_of(n, lows[b], key_base + ((b0 + b) << rd.shift));
        }
      }
      __syncthreads();
      for (uint32_t b = threadIdx.x; b < mine; b += kThreads) {
        unsigned long long sum = 0;
        for (uint32_t c = 0; c < t.C; c++) sum += sums[c * part + b];
        sums[b] = sum;  // read by this thread alone
      }
      __syncthreads();
      for (uint32_t c = warp; c < t.C; c += kWarps) {
        unsigned long long *tot = t.cl.map_shared_rank(s->tot, c) + b0;
        for (uint32_t b = lane; b < mine; b += 32) tot[b] = sums[b];
      }
    } else {
      for (uint32_t b = threadIdx.x; b < nb; b += kThreads)
        s->tot[b] = COUNT ? s->cnt[b] : rd.sum_of(s->cnt[b], s->low[b], key_base + (b << rd.shift));
    }
    t.sync();  // every CTA has every sum, and is done with every CTA's bins
    target = find_bin(s, nb, target, p);
    const uint32_t bin = (uint32_t)s->found[0];
    const unsigned long long above = s->found[1];
    in_bin = s->found[2];
    if (bin >= nb) return cut;  // fewer tokens than asked for: all stay
    const uint32_t low = key_base + (bin << rd.shift);  // the bin's lowest key
    prefix = low >> rd.shift;
    target -= above;
    // the whole bin stays when all its tokens are asked for; by weight, when it holds one token
    const bool whole = COUNT ? target == in_bin : in_bin < 2 * weight_of(__uint_as_float(low));
    if (whole) {
      if (low > cut.key) cut = Cut{low, 0xFFFFFFFFu};
      return cut;
    }
    if (round == 2) return of_one_key(low);
  }
  return cut;
}

// Top-k and top-p among the tokens (what min-p drops has weight 0), then the draw, in the
// order of their places.  id: a place's token,
// or NULL for the place itself.
template <bool CLUSTER>
CH_DEV void cut_and_draw(const RowsArgs &a, uint32_t row, const Tokens<CLUSTER> &t, int32_t top_k, float top_p, float u,
                         const uint32_t *id, bool binned) {
  Shared *s = t.s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float *e = t.e;
  Cut cut{kKeyLow, 0xFFFFFFFFu};
  if (top_k > 0) cut = select<true>(t, cut, (unsigned long long)top_k, 0.0, binned);
  if (top_p < 1.0f) cut = select<false>(t, cut, 0, (double)top_p, binned && top_k <= 0);
  // thread t owns the `run` places from t * run on, an odd number, which spreads the lanes over
  // the banks
  const uint32_t run = ((t.n + kThreads - 1) / kThreads) | 1u, p0 = threadIdx.x * run;
  uint32_t cnt = 0;
  auto kept_weight = [&](uint32_t i) {
    const uint32_t key = i < t.n ? __float_as_uint(e[i]) : 0u;
    return key != 0 && cut.keeps(key, t.base + i) ? weight_of(__uint_as_float(key)) : 0ull;
  };
  // The thread's sum of floor(2^44 e), below 2^52 (run <= 33), as a double from 2^52 on, where one
  // step is 1: an addition that rounds towards zero takes the floor.  2^44 e is e's bits moved.
  double sum = 4503599627370496.0;
  const uint32_t p1 = min(t.n, p0 + run);
#pragma unroll 4
  for (uint32_t i = p0; i < p1; i++) {
    uint32_t key = __float_as_uint(e[i]);
    if (!cut.keeps(key, t.base + i)) key = 0;
    sum = __dadd_rz(sum, __hiloint2double((int)((key >> 3) + ((1023u - 127u + 44u) << 20)), (int)(key << 29)));
    cnt += key != 0;
  }
  const unsigned long long own = (unsigned long long)(sum - 4503599627370496.0);
  unsigned long long mass = own;
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
  unsigned long long total = mine;
  if (CLUSTER) {
    t.exchange(mine, kept);
    total = kept = 0;
    for (uint32_t c = 0; c < t.C; c++) {
      if (c < t.rank) before += s->xch[t.set][c][0];
      total += s->xch[t.set][c][0];
      kept += (uint32_t)s->xch[t.set][c][1];
    }
  }
  unsigned long long goal = u > 0.f ? (unsigned long long)((double)u * (double)total) : 0ull;
  goal = min(goal, total - 1);
  if (before <= goal && goal < before + mass) {  // this warp's part holds the token
    unsigned long long inc = own;  // the lane that does, then the place in its run
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const int owner = __ffs(__ballot_sync(0xffffffffu, before + inc > goal)) - 1;
    unsigned long long sum = before + __shfl_sync(0xffffffffu, inc - own, owner);
    const uint32_t q0 = (warp * 32 + owner) * run;
    for (uint32_t j0 = 0; j0 < run; j0 += 32) {
      const uint32_t i = q0 + j0 + lane;
      const unsigned long long w = j0 + lane < run ? kept_weight(i) : 0ull;
      inc = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, sum + inc > goal);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          answer(a, row, (int32_t)(id ? id[i] : t.base + i), (float)log((double)w / (double)total), (int32_t)kept);
        }
        break;
      }
      sum += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
}

// What one row asks for
struct Row {
  float temp, inv, top_p, min_p, least, cap, cap_inv, lowest, u;  // least: e that stays at least
  int32_t top_k;
  bool quick, cap_quick;  // divisions by temp, by cap may go by multiplication

  // whether the settings leave few tokens: the largest one, up to kFew, or those min-p keeps
  CH_DEV bool few() const { return !(temp > 0.f) || (top_k > 0 && top_k <= (int32_t)kFew) || min_p > 0.f; }
  // x / y correctly rounded, from r = 1 / y correctly rounded: with q = x r the quotient is
  // q + (x - q y) r, each step one FMA (P. Markstein, IBM J. Res. Dev. 34, 1990), for y far from
  // the ends of the range and with a mantissa that is not all ones
  static CH_DEV bool divides(float y) {
    return y > 1e-15f && y < 1e15f && (__float_as_uint(y) & 0x7FFFFFu) != 0x7FFFFFu;
  }
  static CH_DEV float divide(float x, float y, float r) {
    const float q = x * r;
    return __fmaf_rn(__fmaf_rn(-y, q, x), r, q);
  }

  // (a logit of -inf or the type's lowest value masks its token and stays as it is)
  CH_DEV float capped(float v) const {
    if (!(cap > 0.f && v > lowest)) return v;
    return tanhf(__fdiv_rn(v, cap)) * cap;
  }
  // the same for a cap that divides(); past 1e30 the quotient's rounding is lost in tanh = 1
  CH_DEV float capped_quick(float v) const {
    const float c = tanhf(divide(fminf(fmaxf(v, -1e30f), 1e30f), cap, cap_inv)) * cap;
    return v > lowest ? c : v;
  }
  // e, or 0 where the weight is 0 or min-p drops the token, for the quotient (x - m) / T,
  // correctly rounded (where it is below -64 only the sign matters).  No branches in the common
  // form (QUICK: quick is true): x = m gives exp(0), and what over- or underflows on the way (x
  // far below m, or masked) gives 0 or NaN, which the comparison drops.
  template <bool QUICK>
  CH_DEV float weigh_as(float x, float m) const {
    const float d = x - m, q = QUICK ? divide(d, temp, inv) : __fdiv_rn(d, temp);
    const float w = x == m ? 1.0f : expf(q);
    return w >= least ? w : 0.f;
  }
  CH_DEV float weigh(float x, float m) const { return quick ? weigh_as<true>(x, m) : weigh_as<false>(x, m); }
  // A logit below which no capped one exceeds c: the cap's inverse, lowered until the cap
  // itself says so
  CH_DEV float below(float c) const {
    if (!(cap > 0.f)) return c;
    const float y = __fdiv_rn(c, cap);
    if (!(y > -0.9999f)) return -INFINITY;
    float v = cap * atanhf(fminf(y, 0.9999998f)), step = (fabsf(v) + cap) * 1e-6f;
    v -= 3.f * step;
    for (int i = 0; i < 40; i++) {
      if (capped(v) <= c - cap * 5e-7f) return v;
      v -= step;
      step *= 2.f;
    }
    return -INFINITY;
  }
  // A bound on the logits that can stay, from the largest capped logit and a logit that top_k
  // tokens are not below (or -inf)
  CH_DEV float least_logit(float mc, float bound) const {
    float c = -INFINITY;
    if (min_p > 0.f) c = mc + temp * (logf(fminf(min_p, 1.f)) - 1e-5f) - slack(mc);
    if (bound > -INFINITY) c = fmaxf(c, capped(bound) - slack(mc));
    return c > -INFINITY ? below(c) : c;
  }
  // by how much a capped logit has to be lower for its e to be lower too, whatever the
  // roundings of the cap (3 ulp), the difference, the division (31 2^-23) and exp (2 ulp)
  CH_DEV float slack(float m) const { return temp * 1.6e-5f + (cap > 0.f ? cap : fabsf(m)) * 1e-6f; }
};

// The CTA's largest logit m from its threads' (own) and, for want > 0, a bound that `want` of
// them are not below (or -inf), by a histogram over the range of the threads' maxima.
// maxima[kMaxima] is 0 and *pick kMaxima before.
CH_DEV void cta_bound(float own, uint32_t want, uint32_t *maxima, unsigned long long *warp_a, uint32_t *warp_b,
                      uint32_t *pick, float &m, float &bound) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float least = own > -INFINITY ? own : INFINITY;
  m = warp_max(own);
  bound = -INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  if (lane == 0) warp_a[warp] = (unsigned long long)__float_as_uint(m) << 32 | __float_as_uint(least);
  __syncthreads();
  for (int w = 0; w < kWarps; w++) {
    m = fmaxf(m, __uint_as_float((uint32_t)(warp_a[w] >> 32)));
    least = fminf(least, __uint_as_float((uint32_t)warp_a[w]));
  }
  if (want == 0) return;
  const float per_bin = least < m && m < INFINITY ? (kMaxima - 1) / (m - least) : 0.f;
  if (own > -INFINITY) atomicAdd(&maxima[min(kMaxima - 1, (uint32_t)((m - own) * per_bin))], 1u);
  __syncthreads();
  const uint32_t v0 = maxima[2 * threadIdx.x], v1 = maxima[2 * threadIdx.x + 1];
  static_assert(kMaxima == 2 * kThreads, "two bins per thread");
  uint32_t run = v0 + v1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += u;
  }
  if (lane == 31) warp_b[warp] = run;
  __syncthreads();
  uint32_t before = run - v0 - v1;
  for (int w = 0; w < warp; w++) before += warp_b[w];
  if (before < want && want <= before + v0) *pick = 2 * threadIdx.x;
  if (before + v0 < want && want <= before + v0 + v1) *pick = 2 * threadIdx.x + 1;
  __syncthreads();
  if (*pick < kMaxima - 1 && per_bin > 0.f) {
    const float end = m - (*pick + 1) / per_bin;  // the bin's lower end, lowered by its rounding
    bound = end - (fabsf(end) + fabsf(m)) * 1e-6f;
  }
}

CH_DEV Row row_of(const RowsArgs &a, uint32_t row, float lowest) {
  Row r;
  r.temp = a.temperature ? a.temperature[row] : 1.0f;
  r.top_p = a.top_p ? a.top_p[row] : 1.0f;
  r.min_p = a.min_p ? a.min_p[row] : 0.f;
  r.top_k = a.top_k ? a.top_k[row] : 0;
  r.u = a.uniform[row];
  r.least = fmaxf(__uint_as_float(kKeyLow), r.min_p > 0.f ? fminf(r.min_p, 1.f) : 0.f);  // e = 1 always stays
  r.cap = a.softcap;
  r.lowest = lowest;
  r.inv = __frcp_rn(r.temp);
  r.quick = Row::divides(r.temp);
  r.cap_inv = __frcp_rn(r.cap);
  r.cap_quick = Row::divides(r.cap);
  if (r.top_k <= 0 || (uint32_t)r.top_k >= a.vocab) r.top_k = 0;
  return r;
}

struct Few {
  unsigned long long key[kFew], w[kFew], warp_a[kWarps];
};
// cut_and_draw for n <= kFew tokens with weights e and indices id, in any order: two threads
// compare one with all others.
CH_DEV void rank_and_draw(const RowsArgs &a, uint32_t row, Few *s, const float *e, const uint32_t *id, uint32_t n,
                          int32_t top_k, float top_p, float u) {
  static_assert(kFew * 2 == kThreads, "threads");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t i = threadIdx.x >> 1, part = threadIdx.x & 1;
  __syncthreads();
  if (threadIdx.x < n) {
    s->key[threadIdx.x] = (unsigned long long)__float_as_uint(e[threadIdx.x]) << 32 | (uint32_t)~id[threadIdx.x];
    s->w[threadIdx.x] = weight_of(e[threadIdx.x]);
  }
  __syncthreads();
  const unsigned long long k = i < n ? s->key[i] : ~0ull, wi = i < n ? s->w[i] : 0ull;
  uint32_t rank = 0;
  unsigned long long above = 0;
  if (warp * 16u < n) {
#pragma unroll 4
    for (uint32_t j = part; j < n; j += 2)
      if (s->key[j] > k) rank++, above += s->w[j];
  }
  rank += __shfl_xor_sync(0xffffffffu, rank, 1);
  above += __shfl_xor_sync(0xffffffffu, above, 1);
  bool keep = wi > 0 && (top_k <= 0 || rank < (uint32_t)top_k);
  auto sum_of = [&](unsigned long long v) {
    v = warp_sum64(v);
    __syncthreads();
    if (lane == 0) s->warp_a[warp] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int x = 0; x < kWarps; x++) v += s->warp_a[x];
    return v;
  };
  if (top_p < 1.0f) {
    const unsigned long long need = (unsigned long long)ceil((double)top_p * (double)sum_of(keep && part == 0 ? wi : 0ull));
    keep = keep && above < (need < 1 ? 1 : need);
  }
  __syncthreads();  // every thread has compared
  if (part == 0 && i < n) s->w[i] = keep ? wi : 0ull;  // read after the barriers of the sum
  const unsigned long long total = sum_of(keep && part == 0 ? wi : 0ull);
  const int kept = __syncthreads_count(keep && part == 0);
  unsigned long long goal = u > 0.f ? (unsigned long long)((double)u * (double)total) : 0ull, before = 0;
  goal = min(goal, total - 1);
  const uint32_t mine = ~(uint32_t)k;
  if (warp * 16u < n) {
#pragma unroll 4
    for (uint32_t j = part; j < n; j += 2)
      if (~(uint32_t)s->key[j] < mine) before += s->w[j];
  }
  before += __shfl_xor_sync(0xffffffffu, before, 1);
  if (keep && part == 0 && before <= goal && goal < before + wi) {
    answer(a, row, (int32_t)mine, (float)log((double)wi / (double)total), kept);
  }
}

// One row by a cluster that keeps it in shared memory.  first: the cluster's first row, before
// which every CTA has arrived at the cluster's barrier; it is waited for ahead of the first store
// to another CTA, which must have started by then (the barrier costs nothing behind the row's read).
template <typename T>
CH_DEV void keep_row(const RowsArgs &a, uint32_t row, const Row &r, Shared *s, cg::cluster_group &cl, bool first) {
  const uint32_t C = cl.num_blocks(), rank = cl.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t base = min(a.vocab, rank * a.per), n = min(a.vocab - base, a.per);
  const T *x = static_cast<const T *>(a.logits) + (long long)row * a.row_stride + base;
  int set = 0;
  for (uint32_t i = threadIdx.x; i < kMaxima; i += kThreads) s->maxima[i] = 0;
  if (threadIdx.x == 0) s->pick = kMaxima;

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
#pragma unroll 8
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
  // as 16-byte groups, filled up with masked places
  const uint32_t shift = off & 3u, groups = (shift + n + 3) / 4;
  float4 *e4 = reinterpret_cast<float4 *>(s->e);
  if (threadIdx.x < shift) s->e[threadIdx.x] = -INFINITY;
  if (threadIdx.x < 4 * groups - shift - n) e[n + threadIdx.x] = -INFINITY;
  const Tokens<true> all{s, cl, C, rank, e, n, base, set, sizeof(T) == 2};
  // the CTA's maximum of v
  auto cta_max = [&](float v) {
    v = warp_max(v);
    __syncthreads();
    if (lane == 0) s->warp_b[warp] = __float_as_uint(v);
    __syncthreads();
    for (int w = 0; w < kWarps; w++) v = fmaxf(v, __uint_as_float(s->warp_b[w]));
    return v;
  };

  // ---- the largest logit m; beside it, for top-k, a bound that at least top_k tokens of the
  // row are not below: what every CTA's share of them is not below, the least of these ----
  const bool by_k = r.top_k > 0 && r.top_k <= kMostK, bounded = a.vocab > kList && by_k && r.temp > 0.f;
  float m, bound;
  cta_bound(own, bounded ? ((uint32_t)r.top_k + C - 1) / C : 0u, s->maxima, s->warp_a, s->warp_b, &s->pick, m, bound);
  if (first) cl.barrier_wait();
  all.exchange(__float_as_uint(m), __float_as_uint(bound));
  for (uint32_t c = 0; c < C; c++) {
    m = fmaxf(m, __uint_as_float((uint32_t)s->xch[set][c][0]));
    bound = fminf(bound, __uint_as_float((uint32_t)s->xch[set][c][1]));
  }
  set ^= 1;

  if (m == -INFINITY) {  // nothing to choose from
    if (rank == 0 && threadIdx.x == 0) answer(a, row, -1, -INFINITY, 0);
    return;
  }
  const float mc = r.capped(m);  // the largest capped logit, up to the cap's rounding

  if (!(r.temp > 0.f)) {  // greedy: the lowest index of the largest capped logit
    const float low = r.cap > 0.f ? r.below(mc - r.cap * 1e-6f) : m;
    unsigned long long best = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      if (!(e[i] >= low)) continue;
      best = max(best, greedy_key(r.capped(e[i]), base + i));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) s->warp_a[warp] = best;
    __syncthreads();
    for (int w = 0; w < kWarps; w++) best = max(best, s->warp_a[w]);
    all.exchange(best, 0);
    for (uint32_t c = 0; c < C; c++) best = max(best, s->xch[set][c][0]);
    if (rank == 0 && threadIdx.x == 0) answer(a, row, (int32_t)~(uint32_t)best, 0.f, 1);
    return;
  }

  // ---- few candidates: a bound `low` on the logits that can stay ----
  if (m < INFINITY && (a.vocab <= kList || by_k || r.min_p > 0.f)) {
    const float low = r.least_logit(mc, bound);
    // which of its tokens each lane gives: four neighbouring ones per 128 of the warp's part
    constexpr uint32_t kPart = kSlice / kWarps, kSteps = kPart / 128 + 1;  // one more for the shift
    static_assert(kSteps * 4 <= 64, "bits");
    const uint32_t skip = off & 3u, ends = skip + n;  // token i lies at place skip + i of 16-byte groups
    const uint32_t g0 = warp * kPart + (warp ? 8u : 0u), g1 = min(ends, (warp + 1) * kPart + 8u);
    unsigned long long in = 0;
    uint32_t cnt = 0;
#pragma unroll
    for (uint32_t t = 0; t < kSteps; t++) {
      const uint32_t g = g0 + t * 128 + lane * 4;
      if (g0 + t * 128 >= g1) break;
      uint32_t four = 0;
      if (g < g1) {
        const float4 q = *reinterpret_cast<const float4 *>(s->e + g);
        const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; j++)
          four |= (v[j] >= low && v[j] > -INFINITY && g + j >= skip && g + j < g1 ? 1u : 0u) << j;
      }
      in |= (unsigned long long)four << (4 * t);
      cnt += __popc(four);
    }
    const uint32_t warp_cnt = __reduce_add_sync(0xffffffffu, cnt);
    __syncthreads();
    if (lane == 0) s->warp_b[warp] = warp_cnt;
    __syncthreads();
    uint32_t at = 0, count = 0, mine = 0;
    for (int w = 0; w < kWarps; w++) {
      if (w < warp) at += s->warp_b[w];
      mine += s->warp_b[w];
    }
    all.exchange(mine, 0);
    for (uint32_t c = 0; c < C; c++) {
      if (c < rank) at += (uint32_t)s->xch[set][c][0];
      count += (uint32_t)s->xch[set][c][0];
    }
    set ^= 1;
    if (count <= kList) {
      if (warp_cnt) {  // into the first CTA's list, by index
        float *list = cl.map_shared_rank(s->list, 0);
        uint32_t *list_id = cl.map_shared_rank(s->list_id, 0);
        for (uint32_t t = 0; t < kSteps; t++) {
          const uint32_t four = (uint32_t)(in >> (4 * t)) & 15u;
          if (!__any_sync(0xffffffffu, four)) continue;
          uint32_t sum = __popc(four);
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
          }
          uint32_t to = at + sum - __popc(four);
          const uint32_t g = g0 + t * 128 + lane * 4;
#pragma unroll
          for (int j = 0; j < 4; j++)
            if ((four >> j) & 1) {
              list[to] = s->e[g + j];
              list_id[to++] = base + g + j - skip;
            }
          at += __shfl_sync(0xffffffffu, sum, 31);
        }
      }
      cl.sync();
      if (rank != 0) return;
      float x4[kList / kThreads], top = -INFINITY;
#pragma unroll
      for (uint32_t j = 0; j < kList / kThreads; j++) {
        const uint32_t i = threadIdx.x + j * kThreads;
        x4[j] = i < count ? r.capped(s->list[i]) : -INFINITY;
        top = fmaxf(top, x4[j]);
      }
      top = cta_max(top);
#pragma unroll
      for (uint32_t j = 0; j < kList / kThreads; j++) {
        const uint32_t i = threadIdx.x + j * kThreads;
        if (i < count) s->list[i] = r.weigh(x4[j], top);
      }
      if (count <= kFew) {
        rank_and_draw(a, row, reinterpret_cast<Few *>(s->tot), s->list, s->list_id, count, r.top_k, r.top_p, r.u);
        return;
      }
      __syncthreads();
      cut_and_draw(a, row, Tokens<false>{s, cl, 1, 0, s->list, count, 0, set, false}, r.top_k, r.top_p, r.u, s->list_id,
                   false);
      return;
    }
  }

  // ---- many candidates: weights of all tokens; what min-p drops, and what rounds to weight
  // 0, becomes 0 ----
  float top = m;
  if (r.cap > 0.f) {  // in a pass of its own, which finds the largest capped logit
    auto cap_all = [&](auto quick) {
      top = -INFINITY;
      for (uint32_t g = threadIdx.x; g < groups; g += kThreads) {
        const float4 x4 = e4[g];
        float v[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
          v[j] = decltype(quick)::value ? r.capped_quick(v[j]) : r.capped(v[j]);
          top = fmaxf(top, v[j]);
        }
        e4[g] = make_float4(v[0], v[1], v[2], v[3]);
      }
    };
    if (r.cap_quick) cap_all(std::true_type()); else cap_all(std::false_type());
    top = cta_max(top);
    all.exchange(__float_as_uint(top), 0);
    for (uint32_t c = 0; c < C; c++) top = fmaxf(top, __uint_as_float((uint32_t)s->xch[set][c][0]));
    set ^= 1;
  }
  // (the first round's bins are filled on the way)
  for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) s->cnt[i] = s->low[i] = 0;
  __syncthreads();
  // four tokens at a time; the kind of row is decided outside the loop, whose body then has no
  // calls and no branches (with them inside it the loop took twice as long)
  auto weigh_all = [&](auto quick, auto bin) {
    for (uint32_t g = threadIdx.x; g < groups; g += kThreads) {
      const float4 x4 = e4[g];
      float v[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = r.template weigh_as<decltype(quick)::value>(v[j], top);
      e4[g] = make_float4(v[0], v[1], v[2], v[3]);
      if constexpr (decltype(bin)::value > 0) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (v[j] > 0.f) add_first<decltype(bin)::value == 1>(s, __float_as_uint(v[j]));
      }
    }
  };
  using std::integral_constant;
  auto weigh_binned = [&](auto quick) {
    if (r.top_k > 0)
      weigh_all(quick, integral_constant<int, 1>());
    else if (r.top_p < 1.0f)
      weigh_all(quick, integral_constant<int, 2>());
    else
      weigh_all(quick, integral_constant<int, 0>());
  };
  if (r.quick) weigh_binned(std::true_type()); else weigh_binned(std::false_type());
  __syncthreads();
  cut_and_draw(a, row, all, r.top_k, r.top_p, r.u, nullptr, true);
}

// Number `want`, from 0, of the rows from, from + step, ... below `rows` that `takes`; `rows`
// when there are fewer.  The same for every thread of the cluster.
template <typename F>
CH_DEV uint32_t nth_row(Shared *s, uint32_t rows, uint32_t from, uint32_t step, uint32_t want, F takes) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (; from < rows; from += step * kThreads) {
    const uint32_t row = from + step * threadIdx.x;
    const bool it = row < rows && takes(row);
    const uint32_t its = __ballot_sync(0xffffffffu, it);
    __syncthreads();
    if (lane == 0) s->warp_b[warp] = __popc(its);
    __syncthreads();
    uint32_t before = __popc(its & ((1u << lane) - 1)), total = 0;
    for (int w = 0; w < kWarps; w++) {
      if (w < warp) before += s->warp_b[w];
      total += s->warp_b[w];
    }
    if (want < total) {
      if (it && before == want) s->cut_at = row;
      __syncthreads();
      return s->cut_at;
    }
    want -= total;
  }
  return rows;
}

// Counts the CTAs of launches of kMany that have seen the end of the work in front of them (it wraps,
// and is shared by all streams: only the order of its additions matters, never its value)
__device__ uint32_t seen_before;

// As many clusters as rows (kAll), or as run at once.  The rows with many candidates are dealt
// to them in turn, each cluster counting them for itself.  Of the rows left over a cluster takes
// those whose number is its own modulo the number of clusters, so that nobody else changes the
// tokens it looks at.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const RowsArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared *s = reinterpret_cast<Shared *>(smem_raw);
  cg::cluster_group cl = cg::this_cluster();
  cl.barrier_arrive();
  const uint32_t N = gridDim.x / cl.num_blocks(), number = blockIdx.x / cl.num_blocks();
  const float lowest = lowest_of(static_cast<const T *>(a.logits));
  grid_dep_wait();
  if (a.which == Rows::kMany && threadIdx.x == 0)
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(&seen_before) : "memory");
  grid_dep_launch();
  auto many = [&](uint32_t row) { return !row_of(a, row, lowest).few(); };
  auto left = [&](uint32_t row) { return a.tokens[row] == kLeft; };
  uint32_t row = number;
  if (a.which == Rows::kMany) row = nth_row(s, a.rows, 0, 1, number, many);
  if (a.which == Rows::kLeftOver) row = nth_row(s, a.rows, number, N, 0, left);
  if (row >= a.rows) cl.barrier_wait();  // no row; an arrival is not left without its wait
  for (bool first = true; row < a.rows; first = false) {
    keep_row<T>(a, row, row_of(a, row, lowest), s, cl, first);
    if (a.which == Rows::kAll) return;
    cl.sync();  // every CTA is done with the row
    row = a.which == Rows::kMany ? nth_row(s, a.rows, row + 1, 1, N - 1, many) : nth_row(s, a.rows, row + N, N, 0, left);
  }
}

// Many rows: those with few candidates by a kernel that keeps no logits in shared memory, so
// that all rows are on the SMs at once (the kernel above holds 14 rows of 262,144
// logits).  A cluster reads its row once for the threads' maxima; only the threads whose maximum
// is not below the bound read theirs again, from L2.  Rows with more than 256 candidates are
// left for the other kernel.
struct FewMem {
  uint32_t maxima[kMaxima];
  float list[kFew];
  uint32_t list_id[kFew];
  Few few;
  unsigned long long xch[2][kMaxCluster], warp_a[kWarps];
  uint32_t warp_b[kWarps], pick, n_list;
};
template <typename T>
CH_DEV void few_row(const RowsArgs &a, FewMem &mem) {
  cg::cluster_group cl = cg::this_cluster();
  cl.barrier_arrive();  // waited for ahead of the first store to another CTA
  const uint32_t C = cl.num_blocks(), rank = cl.block_rank(), row = blockIdx.x / C;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t base = min(a.vocab, rank * a.per), n = min(a.vocab - base, a.per);
  const T *x = static_cast<const T *>(a.logits) + (long long)row * a.row_stride + base;
  const Row r = row_of(a, row, lowest_of(x));
  if (!r.few()) return cl.barrier_wait();
  const bool greedy = !(r.temp > 0.f), by_k = r.top_k > 0 && r.top_k <= (int32_t)kFew;
  for (uint32_t i = threadIdx.x; i < kMaxima; i += kThreads) mem.maxima[i] = 0;
  if (threadIdx.x == 0) mem.pick = kMaxima, mem.n_list = 0;

  // f(place, logit) for this thread's tokens: 16-byte pieces, and single ones at the ragged ends
  constexpr uint32_t E = 16 / sizeof(T);
  const uint32_t head = min(n, (E - (uint32_t)(((uintptr_t)x / sizeof(T)) % E)) % E), vecs = (n - head) / E;
  const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
  auto each = [&](auto f) {
#pragma unroll 8
    for (uint32_t j = threadIdx.x; j < vecs; j += kThreads) {
      float v[E];
      unpack16(xv[j], v, x);
#pragma unroll
      for (uint32_t k = 0; k < E; k++) f(head + j * E + k, v[k]);
    }
    if (threadIdx.x < head) f(threadIdx.x, load1(x + threadIdx.x));
    const uint32_t tail = head + vecs * E + threadIdx.x;
    if (tail < n) f(tail, load1(x + tail));
  };
  float own = -INFINITY;  // NaN counts as masked: fmaxf drops it
  each([&](uint32_t, float v) { own = fmaxf(own, v); });
  // The same for the tokens of the warp's threads in `owners`, by the whole warp: one thread alone
  // would wait for its pieces several times (10 us for 128 tokens), the warp waits once per two
  // threads.
  auto each_of = [&](uint32_t owners, auto f) {
    constexpr uint32_t kNone = 1u << 30;
    while (owners) {
      const uint32_t t0 = warp * 32 + __ffs(owners) - 1;
      owners &= owners - 1;
      const uint32_t t1 = owners ? warp * 32 + __ffs(owners) - 1 : kNone;
      owners &= owners - 1;
      for (uint32_t j = lane * kThreads; j < vecs; j += 32 * kThreads) {
        uint4 r0, r1;
        float v[E];
        if (j + t0 < vecs) r0 = xv[j + t0];
        if (j + t1 < vecs && t1 != kNone) r1 = xv[j + t1];
        if (j + t0 < vecs) {
          unpack16(r0, v, x);
#pragma unroll
          for (uint32_t k = 0; k < E; k++) f(head + (j + t0) * E + k, v[k]);
        }
        if (j + t1 < vecs && t1 != kNone) {
          unpack16(r1, v, x);
#pragma unroll
          for (uint32_t k = 0; k < E; k++) f(head + (j + t1) * E + k, v[k]);
        }
      }
      if (lane < 2 && (lane ? t1 : t0) != kNone) {
        const uint32_t t = lane ? t1 : t0, tail = head + vecs * E + t;
        if (t < head) f(t, load1(x + t));
        if (tail < n) f(tail, load1(x + tail));
      }
    }
  };
  float m, bound;
  cta_bound(own, by_k && !greedy ? ((uint32_t)r.top_k + C - 1) / C : 0u, mem.maxima, mem.warp_a, mem.warp_b, &mem.pick, m,
            bound);
  cl.barrier_wait();
  if (threadIdx.x < C)
    cl.map_shared_rank(&mem, threadIdx.x)->xch[0][rank] = (unsigned long long)__float_as_uint(m) << 32 | __float_as_uint(bound);
  cl.sync();
  for (uint32_t c = 0; c < C; c++) {
    m = fmaxf(m, __uint_as_float((uint32_t)(mem.xch[0][c] >> 32)));
    bound = fminf(bound, __uint_as_float((uint32_t)mem.xch[0][c]));
  }
  if (m == -INFINITY || m == INFINITY) {  // nothing to choose from; infinite ones go the other way
    if (rank == 0 && threadIdx.x == 0) answer(a, row, m > 0.f ? kLeft : -1, -INFINITY, 0);
    return;
  }
  const float mc = r.capped(m);
  if (greedy) {  // the lowest index of the largest capped logit
    const float low = r.cap > 0.f ? r.below(mc - r.cap * 1e-6f) : m;
    unsigned long long best = 0;
    each_of(__ballot_sync(0xffffffffu, own >= low), [&](uint32_t i, float v) {
      if (!(v >= low)) return;
      best = max(best, greedy_key(r.capped(v), base + i));
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) mem.warp_a[warp] = best;
    __syncthreads();
    for (int w = 0; w < kWarps; w++) best = max(best, mem.warp_a[w]);
    if (threadIdx.x == 0) cl.map_shared_rank(&mem, 0)->xch[1][rank] = best;
    cl.sync();
    if (rank == 0 && threadIdx.x == 0) {
      for (uint32_t c = 0; c < C; c++) best = max(best, mem.xch[1][c]);
      answer(a, row, (int32_t)~(uint32_t)best, 0.f, 1);
    }
    return;
  }
  const float low = r.least_logit(mc, bound);
  FewMem *to = cl.map_shared_rank(&mem, 0);
  each_of(__ballot_sync(0xffffffffu, own >= low && own > -INFINITY), [&](uint32_t i, float v) {
    if (!(v >= low) || v == -INFINITY) return;
    const uint32_t at = atomicAdd(&to->n_list, 1u);
    if (at < kFew) to->list[at] = v, to->list_id[at] = base + i;
  });
  cl.sync();
  if (rank != 0) return;
  const uint32_t count = mem.n_list;
  if (count > kFew) {
    if (threadIdx.x == 0) a.tokens[row] = kLeft;
    return;
  }
  float v = threadIdx.x < count ? r.capped(mem.list[threadIdx.x]) : -INFINITY, top = warp_max(v);
  if (lane == 0) mem.warp_b[warp] = __float_as_uint(top);
  __syncthreads();
  for (int w = 0; w < kWarps; w++) top = fmaxf(top, __uint_as_float(mem.warp_b[w]));
  if (threadIdx.x < count) mem.list[threadIdx.x] = r.weigh(v, top);
  rank_and_draw(a, row, &mem.few, mem.list, mem.list_id, count, r.top_k, r.top_p, r.u);
}
// Runs beside the launch in front of it, which takes the rows with many candidates, and ends
// after it.  Its own griddepcontrol.wait comes last, so what orders its reads after the work before
// both is this: it starts when every CTA of that launch has waited for that work, added to
// seen_before with release and only then let dependents start; its load of seen_before with
// acquire therefore takes one of those additions or a later one (additions carry a release on).
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) sample_few_kernel(const RowsArgs a) {
  __shared__ FewMem mem;
  uint32_t seen;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(&seen_before) : "memory");
  grid_dep_launch();
  few_row<T>(a, mem);
  grid_dep_wait();
}

// The kernel's attributes, once per device and cluster size: its shared memory, clusters of 16, and
// the same split of L1 for both kernels (an SM changes it only when it is empty).  running (if
// not NULL): how many clusters of C CTAs run at once
cudaError_t allow(const void *kernel, size_t smem, uint32_t C, uint32_t *running) {
  static std::mutex mu;
  static std::map<std::tuple<int, const void *, uint32_t>, int> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_tuple(dev, kernel, C);
  auto at = done.find(key);
  if (at == done.end()) {
    e = ensure_smem_attr(kernel, smem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(C);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
    if (e != cudaSuccess) return e;
    at = done.emplace(key, std::max(n, 1)).first;
  }
  if (running) *running = (uint32_t)at->second;
  return cudaSuccess;
}

template <typename K>
cudaError_t start_clusters(K kernel, const RowsArgs &a, uint32_t clusters, uint32_t C, size_t smem, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * C);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T>
cudaError_t launch_rows(RowsArgs a, uint32_t rows, cudaStream_t stream) {
  uint32_t C = 1;
  while (C * kSlice < a.vocab) C *= 2;
  a.rows = rows;
  uint32_t running = 0, few = std::min(C, 8u), few_running = 0;
  cudaError_t e = allow((const void *)sample_rows_kernel<T>, sizeof(Shared), C, &running);
  if (e != cudaSuccess) return e;
  auto launch = [&](Rows which) {
    a.which = which;
    a.per = (a.vocab + C - 1) / C;
    return start_clusters(sample_rows_kernel<T>, a, std::min(rows, running), C, sizeof(Shared), stream);
  };
  // Rows that run at once in the kernel that keeps them (14 of 262,144 logits) all go there: one
  // launch (8 rows of mixed settings 18 us, 2 less than by the other way).  More rows: first those with
  // many candidates, dealt to the clusters that run at once, beside them those with few, then
  // what those left (64 rows: all of them through the first kernel 70 us, so 46).
  if (rows <= running) return launch(Rows::kAll);
  // Rows with few candidates in clusters of 8, which read faster (48 such rows 28 to 29 us, in clusters
  // of 4 37), or of 4 where 8 leave less than a quarter of the SMs for the rows with many: 64
  // rows, 7 of them with many, take 47 us in clusters of 4, 54 in clusters of 8.
  e = allow((const void *)sample_few_kernel<T>, 0, few, &few_running);
  if (e == cudaSuccess && few == 8 && rows > few_running * 3 / 4) {
    few = 4;
    e = allow((const void *)sample_few_kernel<T>, 0, few, nullptr);
  }
  if (e == cudaSuccess) e = launch(Rows::kMany);
  if (e != cudaSuccess) return e;
  a.per = (a.vocab + few - 1) / few;
  e = start_clusters(sample_few_kernel<T>, a, rows, few, 0, stream);
  if (e != cudaSuccess) return e;
  return launch(Rows::kLeftOver);
}

int sample_rows(const ch_sample_rows_args *p, void *stream) {
  if (!p) return set_last_error(CH_EINVAL, "sample_rows: args is NULL");
  if (p->n_rows == 0) return CH_OK;
  if (!p->logits || !p->uniform || !p->tokens) return set_last_error(CH_EINVAL, "sample_rows: NULL argument");
  if (p->vocab == 0 || p->vocab > kMaxVocab)
    return set_last_error(CH_EINVAL, "sample_rows: vocab must be 1.." + std::to_string(kMaxVocab));
  if (p->n_rows > 1u << 20) return set_last_error(CH_EINVAL, "sample_rows: at most 2^20 rows");
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = p->dtype == CH_F32   ? launch_rows<float>(a, p->n_rows, s)
                        : p->dtype == CH_F16 ? launch_rows<__half>(a, p->n_rows, s)
                                             : launch_rows<__nv_bfloat16>(a, p->n_rows, s);
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
