// Sampling the next token of each row of logits, with temperature, top-k, top-p
// and min-p, from given random numbers.
//
// Each row's tokens are ordered by logit (larger first, ties by lower index).
// With M the row's maximum and p_i = exp((l_i - M) / T), a token is kept iff
//   its place in that order is below top_k,
//   the mass before it is below top_p * (mass of the top_k tokens)  (the first
//     token is always kept), and
//   p_i >= min_p;
// the kept tokens are a prefix of the order. The answer is the kept token with the
// largest p_i / e_i, e_i the row's exponential random numbers: of independent
// Exp(1) variables divided by rates p_i the smallest belongs to i with
// probability p_i / sum p, so this is a draw from the kept tokens' softmax.
//
// What bounds it: the row's logits and random numbers are read once, and everything
// after that is latency -- a row is a chain of reductions. So a row is a cluster of
// CTAs that keep their slices of the logits in shared memory and exchange sums and
// maxima through distributed shared memory, and no step sorts the vocabulary:
//   1. the row's maximum M;
//   2. sum of exp(l - M), for the log-probability, and either
//      a. top_k up to kList: a count of the tokens by floor((M - l) * 16); the bins that
//         hold the first top_k tokens (found by finer counts where these are not
//         enough) are gathered and sorted by one CTA, which
//         applies every filter and runs the race among the few kept (the random
//         numbers of all other tokens are not read); or
//      b. the race among all tokens. Its winner is the answer if it is kept. If it
//         is not, nothing after it in the order is kept either, so the race is run
//         again among the tokens before it: gathered and sorted as in a. once they
//         are few, otherwise another round. A round throws away a random share of
//         what is left, so rounds are few; after kRounds of them (random numbers
//         made to defeat this) the cut is found by halving instead.
//
// The race compares log2(p_i) - log2(e_i), one multiply-add and one approximate
// logarithm per token, and evaluates p_i / e_i in full only for the tokens within
// kNear of the largest: the answer is that of the full evaluation.
#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>
#include <vector>

#include "wbk_common.cuh"
#include "wbk_kv8.cuh"

namespace cg = cooperative_groups;

namespace wbk {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kSliceElems = 8192;       // per CTA, if a cluster of kMaxCluster allows
constexpr int kSliceBytes = 100 * 1024; // most that is kept in shared memory (two CTAs per SM)
constexpr int kList = 2048;             // most tokens that one CTA sorts
constexpr int kBins = kThreads;
constexpr float kBinsPerUnit = 16.0f;
constexpr int kRounds = 6;
// Error of the approximate race in log2 units: two roundings of a product up to 150 (tokens below 2^-149 have
// p = 0), 1.8e-5, and of a logarithm up to 126, 0.8e-5, plus the approximate logarithm's 2^-22.
constexpr float kNear = 1e-4f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMinNoise = 1.17549435e-38f;

struct SampleParams {
  const void* logits;
  int64_t logits_stride;
  const float* noise;
  int64_t noise_stride;
  const float *temperature, *top_p, *min_p;  // per row, or NULL: the numbers below
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int vocab, slice;  // slice: tokens per CTA, a multiple of 8
  int64_t* tokens;
  float* logprobs;
};

// Logit as an ordered fp32: NaN is never drawn (-inf), +inf is the largest finite
// number, -0 is +0.
template <int kDtype>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  float x;
  if constexpr (kDtype == WBK_DT_F32) x = static_cast<const float*>(p)[i];
  else if constexpr (kDtype == WBK_DT_F16) x = __half2float(static_cast<const __half*>(p)[i]);
  else x = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return isnan(x) ? -INFINITY : fminf(x, 3.402823466e38f) + 0.0f;
}

// Order-preserving key of an fp32 and back, and the place of token i in its row's
// order: larger is earlier. No place is 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}
__device__ __forceinline__ uint64_t place_of(float x, int i) {
  return (static_cast<uint64_t>(order_key(x)) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int place_index(uint64_t place) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(place)); }
__device__ __forceinline__ float place_logit(uint64_t place) { return key_value(static_cast<uint32_t>(place >> 32)); }

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint64_t warp_max_u64(uint64_t v) {
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

// What a CTA tells its cluster in one exchange, and what it keeps for itself. All
// sums run in a fixed order (thread, warp, rank), so equal inputs give equal bits.
struct Message {
  uint64_t u;
  float f, g;
  int c;
};
struct SampleSmem {
  Message warp[kWarps];
  Message said[2];          // exchanges alternate between the two
  int bins[kBins];          // this CTA's counts
  int all[kBins];           // the row's
  int count;
  float scan[kWarps];
  uint64_t list[kList];     // of rank 0: places
  float mass[kList];
};

// Joins every thread's (max u, sum f, sum g, sum c) over the CTA and the cluster.
__device__ __forceinline__ Message exchange(Message m, SampleSmem& s, cg::cluster_group& cluster, int& turn) {
  m.u = warp_max_u64(m.u);
  m.f = warp_sum(m.f);
  m.g = warp_sum(m.g);
  m.c = __reduce_add_sync(~0u, m.c);
  if ((threadIdx.x & 31) == 0) s.warp[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x < 32) {
    m = threadIdx.x < kWarps ? s.warp[threadIdx.x] : Message{0, 0.0f, 0.0f, 0};
    m.u = warp_max_u64(m.u);
    m.f = warp_sum(m.f);
    m.g = warp_sum(m.g);
    m.c = __reduce_add_sync(~0u, m.c);
    if (threadIdx.x == 0) s.said[turn] = m;
  }
  cluster.sync();
  Message r{0, 0.0f, 0.0f, 0};
  for (unsigned i = 0; i < cluster.num_blocks(); ++i) {
    const Message& o = *cluster.map_shared_rank(&s.said[turn], i);
    r.u = max(r.u, o.u);
    r.f += o.f;
    r.g += o.g;
    r.c += o.c;
  }
  turn ^= 1;
  return r;
}

// The key of a non-negative score above the index that breaks ties.
__device__ __forceinline__ uint64_t score_place(float score, int i) {
  return (static_cast<uint64_t>(__float_as_uint(score)) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

// A row as its cluster sees it.
template <int kDtype, bool kResident>
struct Row {
  const void* x;       // the CTA's slice: of shared memory, or of the row itself
  const float* noise;  // the whole row's
  int begin, end;      // the CTA's tokens
  float top, temperature, scale;  // scale = log2(e) / temperature

  __device__ __forceinline__ float logit(int i) const { return load_logit<kDtype>(x, i - begin); }
  __device__ __forceinline__ float weight(float l) const { return expf((l - top) / temperature); }
  __device__ __forceinline__ float score(float l, int i) const { return weight(l) / fmaxf(noise[i], kMinNoise); }
};

// The race among the tokens placed before (above) `limit`: score_place of the CTA's
// winner in full evaluation, 0 if it has no token there; and per thread, where
// asked, the sum of exp(l - top) and of exp((l - top) / temperature).
template <int kDtype, bool kResident, bool kSums>
__device__ __forceinline__ uint64_t race(const Row<kDtype, kResident>& r, uint64_t limit, float least, SampleSmem& s,
                                         float& raw, float& all) {
  float best = -INFINITY, second = -INFINITY;
  int best_i = -1;
  // groups of four that are 16-byte aligned in the random numbers
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(r.noise + r.begin) >> 2) & 3);
  for (int i0 = r.begin - shift + 4 * static_cast<int>(threadIdx.x); i0 < r.end; i0 += 4 * kThreads) {
    float e[4];
    if (i0 >= r.begin && i0 + 4 <= r.end) {
      const float4 v = *reinterpret_cast<const float4*>(r.noise + i0);
      e[0] = v.x, e[1] = v.y, e[2] = v.z, e[3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = i0 + j >= r.begin && i0 + j < r.end ? r.noise[i0 + j] : 1.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j;
      if (i < r.begin || i >= r.end) continue;
      const float l = r.logit(i), gap = l - r.top, power = gap * r.scale;
      if (kSums) {
        raw += ex2(gap * kLog2e);
        all += ex2(power);
      }
      const float t = power - lg2(fmaxf(e[j], kMinNoise));
      if (t > second && power >= least && (limit == 0 || place_of(l, i) > limit)) {
        if (t > best) second = best, best = t, best_i = i;
        else second = t;
      }
    }
  }
  // the CTA's largest, then full evaluation of all that come near it
  float top = best;
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  if ((threadIdx.x & 31) == 0) s.scan[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) top = fmaxf(top, s.scan[i]);
  __syncthreads();
  uint64_t won = 0;
  if (best_i >= 0 && best >= top - kNear) {
    won = score_place(r.score(r.logit(best_i), best_i), best_i);
    if (second >= top - kNear) {  // two of this thread's tokens are near: look at all of them again
      for (int i0 = r.begin - shift + 4 * static_cast<int>(threadIdx.x); i0 < r.end; i0 += 4 * kThreads)
        for (int i = max(i0, r.begin); i < min(i0 + 4, r.end); ++i) {
          const float l = r.logit(i), power = (l - r.top) * r.scale;
          if (l > -INFINITY && power >= least && (limit == 0 || place_of(l, i) > limit))
            won = max(won, score_place(r.score(l, i), i));
        }
    }
  }
  return won;
}

// The CTAs' counts in s.bins, added over the cluster: the first bin up to which they reach `least` (kBins where
// none does), the sum up to there and the sum before it. Ends with the cluster in step.
struct Cut {
  int bin, upto, before;
};
__device__ __forceinline__ Cut cut_bins(int least, SampleSmem& s, cg::cluster_group& cluster) {
  cluster.sync();
  int c = 0;
  for (unsigned i = 0; i < cluster.num_blocks(); ++i) c += *cluster.map_shared_rank(&s.bins[threadIdx.x], i);
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, c, o);
    if ((threadIdx.x & 31) >= o) c += y;
  }
  s.all[threadIdx.x] = c;  // up to this bin, within its 32
  cluster.sync();
  Cut r{kBins, 0, 0};
  for (int b0 = 0; b0 < kBins && r.bin == kBins; b0 += 32) {
    const int upto = r.upto + s.all[b0 + (threadIdx.x & 31)];
    const uint32_t enough = __ballot_sync(~0u, upto >= least);
    const int at = enough != 0 ? __ffs(enough) - 1 : 31;
    r.before = enough != 0 && at > 0 ? __shfl_sync(~0u, upto, max(at - 1, 0)) : enough != 0 ? r.upto : 0;
    r.upto = __shfl_sync(~0u, upto, at);
    if (enough != 0) r.bin = b0 + at;
  }
  return r;
}

// A place that the first top_k tokens lie before (above), and the number of tokens before it: top_k, or for
// small top_k at most kList. By counts of the range that the last of them lies in, kBins-fold smaller each time.
template <int kDtype, bool kResident>
__device__ __forceinline__ uint64_t kth_limit(const Row<kDtype, kResident>& r, int top_k, uint64_t first, SampleSmem& s,
                                              cg::cluster_group& cluster, int& left) {
  uint64_t lo = 0, hi = first;  // the last of the first top_k lies in (lo, hi]
  int above = 0;                // tokens above hi
  for (;;) {
    int shift = 0;
    while (((hi - lo - 1) >> shift) >= kBins) ++shift;
    s.bins[threadIdx.x] = 0;
    __syncthreads();
    for (int i = r.begin + threadIdx.x; i < r.end; i += kThreads) {
      const uint64_t place = place_of(r.logit(i), i);
      if (place > lo && place <= hi) atomicAdd(&s.bins[(hi - place) >> shift], 1);
    }
    const Cut cut = cut_bins(top_k - above, s, cluster);
    const uint64_t to = hi - (static_cast<uint64_t>(cut.bin) << shift);
    const uint64_t step = 1ull << shift;
    lo = to - lo > step ? to - step : lo;
    hi = to;
    left = above + cut.upto;
    above += cut.before;
    if (shift == 0 || left <= kList) return lo;
  }
}

// Number and mass of the tokens placed before `limit`.
template <int kDtype, bool kResident>
__device__ __forceinline__ Message before(const Row<kDtype, kResident>& r, uint64_t limit, SampleSmem& s,
                                          cg::cluster_group& cluster, int& turn) {
  Message m{0, 0.0f, 0.0f, 0};
  for (int i = r.begin + threadIdx.x; i < r.end; i += kThreads) {
    const float l = r.logit(i);
    if (place_of(l, i) > limit) ++m.c, m.f += r.weight(l);
  }
  return exchange(m, s, cluster, turn);
}

// Rank 0's list of n places, sorted, then every filter and the race among the kept:
// the winner's place. `whole` is the mass that top_p refers to, or < 0: that of
// the first top_k in the list.
template <int kDtype, bool kResident>
__device__ __forceinline__ uint64_t finish(const Row<kDtype, kResident>& r, int n, int top_k, float top_p, float min_p,
                                           float whole, SampleSmem& s) {
  int size = 32;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kThreads) s.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int t = threadIdx.x; t < size / 2; t += kThreads) {
        const int a = 2 * t - (t & (j - 1)), b = a + j;
        const uint64_t x = s.list[a], y = s.list[b];
        if ((x < y) == ((a & k) == 0)) s.list[a] = y, s.list[b] = x;  // larger (earlier) first
      }
      __syncthreads();
    }
  const int kept = min(n, top_k);
  // running masses: each thread a run of the list, then over the threads
  const int run = (kept + kThreads - 1) / kThreads, i0 = threadIdx.x * run, i1 = min(i0 + run, kept);
  float own = 0.0f;
  for (int i = i0; i < i1; ++i) {
    s.mass[i] = r.weight(place_logit(s.list[i]));
    own += s.mass[i];
  }
  float upto = own;
  for (int o = 1; o < 32; o <<= 1) {
    const float y = __shfl_up_sync(~0u, upto, o);
    if ((threadIdx.x & 31) >= o) upto += y;
  }
  if ((threadIdx.x & 31) == 31) s.scan[threadIdx.x >> 5] = upto;
  __syncthreads();
  float total = 0.0f, mass = upto - own;
  for (int i = 0; i < kWarps; ++i) {
    if (i == static_cast<int>(threadIdx.x >> 5)) mass += total;
    total += s.scan[i];
  }
  const double cut = static_cast<double>(top_p) * (whole >= 0.0f ? whole : total);
  uint64_t won = 0;
  for (int i = i0; i < i1; ++i) {
    const float w = s.mass[i];
    if (i == 0 || ((top_p >= 1.0f || static_cast<double>(mass) < cut) && w >= min_p && place_logit(s.list[i]) > -INFINITY)) {
      const int token = place_index(s.list[i]);
      won = max(won, score_place(w / fmaxf(r.noise[token], kMinNoise), token));
    }
    mass += w;
  }
  won = warp_max_u64(won);
  if ((threadIdx.x & 31) == 0) s.warp[threadIdx.x >> 5].u = won;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) won = max(won, s.warp[i].u);
  const int token = place_index(won);
  // back to the place, for its logit
  uint64_t place = 0;
  for (int i = i0; i < i1; ++i)
    if (place_index(s.list[i]) == token) place = s.list[i];
  place = warp_max_u64(place);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.warp[threadIdx.x >> 5].u = place;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) place = max(place, s.warp[i].u);
  return place;
}

// One cluster per row.
template <int kDtype, bool kResident>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleSmem& s = *reinterpret_cast<SampleSmem*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t row = blockIdx.x / cluster.num_blocks();
  constexpr int kItem = kDtype == WBK_DT_F32 ? 4 : 2, kVec = 16 / kItem;
  int turn = 0;
  const uint8_t* logits = static_cast<const uint8_t*>(p.logits) + row * p.logits_stride * kItem;
  Row<kDtype, kResident> r;
  r.noise = p.noise + row * p.noise_stride;
  r.begin = min(rank * p.slice, p.vocab);
  r.end = min(r.begin + p.slice, p.vocab);
  const float temperature = p.temperature != nullptr ? p.temperature[row] : p.temperature_all;
  const float top_p = p.top_p != nullptr ? p.top_p[row] : p.top_p_all;
  const float min_p = p.min_p != nullptr ? p.min_p[row] : p.min_p_all;
  const int k_given = p.top_k != nullptr ? p.top_k[row] : p.top_k_all;
  const int top_k = k_given > 0 && k_given < p.vocab ? k_given : p.vocab;

  // ---- 1. the first token of the order; the slice goes to shared memory
  const uint8_t* slice = logits + static_cast<int64_t>(r.begin) * kItem;
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(slice) & 15) / kItem);  // slice begins so far into a vector
  uint8_t* held = smem_raw + (sizeof(SampleSmem) + 15) / 16 * 16;
  r.x = kResident ? static_cast<const void*>(held + shift * kItem) : slice;
  Message m{0, 0.0f, 0.0f, 0};
  for (int i0 = r.begin - shift + kVec * static_cast<int>(threadIdx.x); i0 < r.end; i0 += kVec * kThreads) {
    if (i0 >= r.begin && i0 + kVec <= r.end) {
      const uint4 v = *reinterpret_cast<const uint4*>(logits + static_cast<int64_t>(i0) * kItem);
      if (kResident) *reinterpret_cast<uint4*>(held + (i0 - r.begin + shift) * kItem) = v;
#pragma unroll
      for (int j = 0; j < kVec; ++j) m.u = max(m.u, place_of(load_logit<kDtype>(&v, j), i0 + j));
    } else {
      for (int i = max(i0, r.begin); i < min(i0 + kVec, r.end); ++i) {
        if (kResident) {
          if constexpr (kItem == 4) reinterpret_cast<float*>(held)[i - r.begin + shift] = reinterpret_cast<const float*>(logits)[i];
          else reinterpret_cast<uint16_t*>(held)[i - r.begin + shift] = reinterpret_cast<const uint16_t*>(logits)[i];
        }
        m.u = max(m.u, place_of(load_logit<kDtype>(logits, i), i));
      }
    }
  }
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.bins[i] = 0;
  if (threadIdx.x == 0) s.count = 0;
  m = exchange(m, s, cluster, turn);
  const uint64_t first = m.u;
  r.top = place_logit(first);
  r.temperature = temperature;
  r.scale = fminf(kLog2e / temperature, 3e38f);

  uint64_t winner = first;  // a place
  float raw = 0.0f;
  const bool empty = r.top == -INFINITY;
  if (!empty && !(temperature > 0.0f)) {
    for (int i = r.begin + threadIdx.x; i < r.end; i += kThreads) raw += ex2((r.logit(i) - r.top) * kLog2e);
    raw = exchange(Message{0, raw, 0.0f, 0}, s, cluster, turn).f;
  } else if (!empty) {
    const bool few = top_k <= kList && top_k < p.vocab;
    const float least = min_p > 0.0f ? lg2(min_p) - kNear : -INFINITY;  // of log2 p, for the race
    uint64_t limit = 0;       // every token at or after this place is out
    int left = p.vocab;       // tokens before it
    float whole = -1.0f;      // the mass top_p refers to
    int cut_bin = -1;         // or: what is left are the tokens of the bins up to this
    bool gather = false;      // what is left fits one CTA's list
    if (few) {
      // ---- 2a. count by distance from the maximum
      for (int i = r.begin + threadIdx.x; i < r.end; i += kThreads) {
        const float gap = r.top - r.logit(i);
        raw += ex2(-gap * kLog2e);
        const float bin = gap * kBinsPerUnit;
        if (bin < kBins) atomicAdd(&s.bins[static_cast<int>(bin)], 1);
      }
      raw = exchange(Message{0, raw, 0.0f, 0}, s, cluster, turn).f;
      const Cut cut = cut_bins(top_k, s, cluster);
      gather = true;
      if (cut.bin < kBins && cut.upto <= kList) cut_bin = cut.bin, left = cut.upto;
      else limit = kth_limit(r, top_k, first, s, cluster, left);  // far from the maximum, or many ties
    }
    if (!gather) {
      if (top_k < p.vocab) {
        limit = kth_limit(r, top_k, first, s, cluster, left);
        whole = before(r, limit, s, cluster, turn).f;
      }
      // ---- 2b. rounds
      uint64_t lo = 0, hi = first;  // the cut lies between these places, once halving has begun
      for (int round = 0;; ++round) {
        float all = 0.0f, dummy = 0.0f;
        Message w{0, 0.0f, 0.0f, 0};
        if (round == 0) {
          raw = 0.0f;
          w.u = race<kDtype, kResident, true>(r, limit, least, s, raw, all);
          w.f = raw;
          w.g = all;
          w = exchange(w, s, cluster, turn);
          raw = w.f;
          if (whole < 0.0f) whole = w.g;
        } else {
          w.u = race<kDtype, kResident, false>(r, limit, least, s, dummy, dummy);
          w = exchange(w, s, cluster, turn);
        }
        // the winner's place: its logit is with the CTA that has it
        const int token = place_index(w.u);
        Message mine{0, 0.0f, 0.0f, 0};
        if (threadIdx.x == 0 && token >= r.begin && token < r.end) mine.u = place_of(r.logit(token), token);
        winner = exchange(mine, s, cluster, turn).u;
        if (winner == first) break;
        const bool likely = r.weight(place_logit(winner)) >= min_p;
        if (top_p >= 1.0f && likely) break;
        const Message b = before(r, winner, s, cluster, turn);
        if (likely && static_cast<double>(b.f) < static_cast<double>(top_p) * whole) break;
        limit = winner;
        left = b.c;
        gather = left <= kList;
        if (gather) break;
        if (round >= kRounds) {
          lo = limit;
          while (hi - lo > 1 && left > kList) {
            const uint64_t mid = lo + (hi - lo) / 2;
            const Message c = before(r, mid, s, cluster, turn);
            if ((top_p >= 1.0f || static_cast<double>(c.f) < static_cast<double>(top_p) * whole) &&
                r.weight(place_logit(mid)) >= min_p)
              hi = mid;
            else
              lo = mid, left = c.c;
          }
          limit = lo;
          gather = left <= kList;
          if (gather) break;
          // every token before `limit` is kept: one more race decides
          w = Message{0, 0.0f, 0.0f, 0};
          w.u = race<kDtype, kResident, false>(r, limit, -INFINITY, s, dummy, dummy);
          w = exchange(w, s, cluster, turn);
          const int last = place_index(w.u);
          mine = Message{0, 0.0f, 0.0f, 0};
          if (threadIdx.x == 0 && last >= r.begin && last < r.end) mine.u = place_of(r.logit(last), last);
          winner = exchange(mine, s, cluster, turn).u;
          break;
        }
      }
    }
    if (gather) {
      // ---- gather what is left at rank 0: a run of its list for each CTA
      Message mine{0, 0.0f, 0.0f, 0};
      for (int i = r.begin + threadIdx.x; i < r.end; i += kThreads) {
        const float l = r.logit(i);
        if (cut_bin >= 0 ? (r.top - l) * kBinsPerUnit < cut_bin + 1 : place_of(l, i) > limit) ++mine.c;
      }
      exchange(mine, s, cluster, turn);  // said[turn ^ 1].c of each rank
      int base = 0;
      for (int i = 0; i < rank; ++i) base += cluster.map_shared_rank(&s.said[turn ^ 1], i)->c;
      uint64_t* list = cluster.map_shared_rank(&s.list[0], 0);
      for (int i = r.begin + threadIdx.x; i < r.end; i += kThreads) {
        const float l = r.logit(i);
        if (cut_bin >= 0 ? (r.top - l) * kBinsPerUnit < cut_bin + 1 : place_of(l, i) > limit) {
          const int at = base + atomicAdd(&s.count, 1);
          if (at < kList) list[at] = place_of(l, i);
        }
      }
      cluster.sync();
      if (rank == 0) winner = finish(r, min(left, kList), top_k, top_p, min_p, whole, s);
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    p.tokens[row] = empty ? -1 : place_index(winner);
    p.logprobs[row] = empty ? -INFINITY : (place_logit(winner) - r.top) - logf(raw);
  }
  cluster.sync();  // no CTA ends while another may read its shared memory
}

template <int kDtype, bool kResident>
int launch_sample(const SampleParams& p, int64_t rows, int ctas, cudaStream_t stream) {
  constexpr int kItem = kDtype == WBK_DT_F32 ? 4 : 2;
  constexpr int kFixed = (sizeof(SampleSmem) + 15) / 16 * 16;
  static std::mutex mu;
  static std::vector<char> configured;
  const int dev = current_device();
  if (dev < 0) return fail(WBK_ERR_CUDA, "no current CUDA device");
  {
    std::lock_guard<std::mutex> lock(mu);
    if (static_cast<int>(configured.size()) <= dev) configured.resize(dev + 1, 0);
    if (!configured[dev]) {
      if (int e = cuda_check(cudaFuncSetAttribute(sample_kernel<kDtype, kResident>,
                                                  cudaFuncAttributeMaxDynamicSharedMemorySize, kFixed + kSliceBytes + 32),
                             "sample smem attribute"))
        return e;
      configured[dev] = 1;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = kFixed + (kResident ? p.slice * kItem + 32 : 0);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_check(cudaLaunchKernelEx(&cfg, sample_kernel<kDtype, kResident>, p), "sample launch");
}

template <int kDtype>
int dispatch_sample(SampleParams p, int64_t rows, cudaStream_t stream) {
  constexpr int kItem = kDtype == WBK_DT_F32 ? 4 : 2;
  int ctas = 1;
  while (ctas < kMaxCluster && (p.vocab + ctas - 1) / ctas > kSliceElems) ctas *= 2;
  p.slice = ((p.vocab + ctas - 1) / ctas + 7) / 8 * 8;
  if (rows * ctas > (int64_t(1) << 31) - 1) return fail(WBK_ERR_UNSUPPORTED, "wbk_sample: too many rows");
  return static_cast<int64_t>(p.slice) * kItem <= kSliceBytes ? launch_sample<kDtype, true>(p, rows, ctas, stream)
                                                              : launch_sample<kDtype, false>(p, rows, ctas, stream);
}

}  // namespace
}  // namespace wbk

using namespace wbk;

extern "C" {

int wbk_sample(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t logits_stride, const float* noise,
               int64_t noise_stride, const float* temperature, const int32_t* top_k, const float* top_p,
               const float* min_p, float temperature_all, int top_k_all, float top_p_all, float min_p_all,
               int64_t* tokens_out, float* logprobs_out, wbk_stream_t stream) {
  if (rows < 0 || vocab < 0) return fail(WBK_ERR_INVALID_ARG, "wbk_sample: negative size");
  if (dtype != WBK_DT_F16 && dtype != WBK_DT_BF16 && dtype != WBK_DT_F32)
    return fail(WBK_ERR_INVALID_ARG, "wbk_sample: unknown dtype %d", dtype);
  if (rows == 0) return WBK_OK;
  if (vocab == 0) return fail(WBK_ERR_INVALID_ARG, "wbk_sample: vocab = 0 with rows present");
  if (logits == nullptr || noise == nullptr || tokens_out == nullptr || logprobs_out == nullptr)
    return fail(WBK_ERR_INVALID_ARG, "wbk_sample: null pointer");
  if (rows > (int64_t(1) << 31) - 1 || vocab > (1 << 30))
    return fail(WBK_ERR_UNSUPPORTED, "wbk_sample: more than 2^31 - 1 rows or 2^30 logits per row");
  if (logits_stride < vocab || noise_stride < vocab)
    return fail(WBK_ERR_INVALID_ARG, "wbk_sample: a row stride is smaller than the vocabulary");
  if (!aligned(logits, dtype == WBK_DT_F32 ? 4 : 2) || !aligned(noise, 4) || !aligned(tokens_out, 8) ||
      !aligned(logprobs_out, 4) || (temperature != nullptr && !aligned(temperature, 4)) ||
      (top_k != nullptr && !aligned(top_k, 4)) || (top_p != nullptr && !aligned(top_p, 4)) ||
      (min_p != nullptr && !aligned(min_p, 4)))
    return fail(WBK_ERR_INVALID_ARG, "wbk_sample: misaligned pointer");
  SampleParams p{};
  p.logits = logits;
  p.logits_stride = logits_stride;
  p.noise = noise;
  p.noise_stride = noise_stride;
  p.temperature = temperature, p.top_k = top_k, p.top_p = top_p, p.min_p = min_p;
  p.temperature_all = temperature_all, p.top_k_all = top_k_all, p.top_p_all = top_p_all, p.min_p_all = min_p_all;
  p.vocab = static_cast<int>(vocab);
  p.tokens = tokens_out;
  p.logprobs = logprobs_out;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == WBK_DT_F16) return dispatch_sample<WBK_DT_F16>(p, rows, st);
  if (dtype == WBK_DT_BF16) return dispatch_sample<WBK_DT_BF16>(p, rows, st);
  return dispatch_sample<WBK_DT_F32>(p, rows, st);
}

}  // extern "C"
