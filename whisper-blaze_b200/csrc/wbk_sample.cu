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
// maxima through distributed shared memory (each CTA writes to all others before
// their one barrier), and no step sorts the vocabulary:
//   1. the row's maximum M;
//   2. sum of exp(l - M), for the log-probability, and either
//      a. top_k up to kList: where as many threads' maxima lie as top_k asks for, there
//         are as many tokens, and few more as a rule; these (or where that rule does
//         not apply those of the first bins of a count by floor((M - l) * 16), or of
//         finer counts) are gathered by one CTA, which applies every filter and runs
//         the race among the few kept (the random numbers of all other tokens are
//         not read); or
//      b. the race among all tokens. Its winner is the answer if it is kept. If it
//         is not, nothing after it in the order is kept either, so the race is run
//         again among the tokens before it: gathered by one CTA as in a. once they
//         are few, otherwise another round. A round throws away a random share of
//         what is left, so rounds are few; after kRounds of them (random numbers
//         made to defeat this) the cut is found by halving instead.
//
// The race compares log2(p_i) - log2(e_i) with a log2 that is linear between powers
// of two (no special-function instruction: the exponentials of step 2 keep that unit
// busy), takes the largest of kAhead tokens at a time, and evaluates p_i / e_i in
// full only for the tokens within kNear of the largest: the answer is that of the
// full evaluation.
//
// Measured (logits in fp16, everything in L2): one row of 51866 4.2 us greedy, 6.2 us
// without filters, 8.5 us with top_k 40, 8.4 us with top_p 0.9; 64 such rows 7.4, 10.9,
// 13.6 and 21.6 us (20 MB are 3.0 us of HBM's time; each exchange takes 1.2 us, a pass over
// a slice 1 to 4 us). 256 rows of 131072 in fp32 come in seven waves of clusters: 70,
// 107, 106 and 154 us (268 MB are 41 us of HBM's time).
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
constexpr int kCtasPerSm = 2;
constexpr int kLeastSlice = 2048;       // tokens per CTA, below which a row is not split further
constexpr int kSliceElems = 25600;      // most tokens per CTA kept in shared memory (two CTAs per SM up to 22000)
constexpr int kList = 2048;             // most tokens that one CTA gathers
constexpr int kBins = kThreads;
constexpr float kBinsPerUnit = 16.0f;
constexpr int kFew = 64;                // tokens whose order is found by comparing all pairs
static_assert(kFew * 2 <= kBins, "they lie where the counts were");
constexpr int kRounds = 6;
constexpr int kAhead = 4;               // a thread's tokens of one step of the race, loaded one step ahead
constexpr int kVecs = 4;                // 16-byte loads of logits in flight per thread
// Error of the approximate race in log2 units: log2_below() is at most 0.08608 too small, and two roundings of values
// below 2^10 and its 23 of 31 bits make 2e-4.
constexpr float kNear = 0.0863f;
// Of a log2 p below 150 and of an approximate logarithm.
constexpr float kSlack = 1e-4f;
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

// A logit as it is ordered: NaN is never drawn (-inf, fmaxf returns the operand that
// is not NaN), +inf is the largest finite number, -0 is +0.
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), 3.402823466e38f) + 0.0f; }
template <int kDtype>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  if constexpr (kDtype == WBK_DT_F32) return clean(static_cast<const float*>(p)[i]);
  else if constexpr (kDtype == WBK_DT_F16) return clean(__half2float(static_cast<const __half*>(p)[i]));
  else return clean(__bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]));
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
// log2 of a positive normal number, linear between the powers of two (Mitchell 1962): its exponent and mantissa bits
// read as a fixed-point number, the upper 23 of them as the mantissa of 2^23 + them. + 383.
__device__ __forceinline__ float log2_below_383(float x) {
  return __uint_as_float(__byte_perm(__float_as_uint(x), 0x4B000000u, 0x7321)) * 3.0517578125e-5f;
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

// What a CTA tells its cluster in one exchange. All sums run in a fixed order
// (thread, warp, rank), so equal inputs give equal bits.
struct Message {
  uint64_t u;  // maximum
  float f, g;  // sums
  int c;       // sum
  float l;     // the logit of the token that u names, filled in by the CTA
};
struct SampleSmem {
  Message warp[kWarps];
  Message said[2][kMaxCluster];  // what each CTA said; exchanges alternate between the two
  int bins[kBins];          // this CTA's counts
  int all[kBins];           // the row's, summed up within each 32
  int base;
  float scan[kWarps];
  uint64_t list[kList];     // of rank 0: places
};

// The key of a non-negative score above the index that breaks ties.
__device__ __forceinline__ uint64_t score_place(float score, int i) {
  return (static_cast<uint64_t>(__float_as_uint(score)) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

// A row as one CTA of its cluster sees it: tokens [begin, end). x points at the
// cleaned slice in shared memory, or at the row's own logits.
template <int kDtype, bool kResident>
struct Row {
  const void* x;
  const float* noise;  // the whole row's
  int begin, end;
  float top, temperature, scale;  // scale = log2(e) / temperature

  __device__ __forceinline__ float logit(int i) const {
    if constexpr (kResident) return static_cast<const float*>(x)[i - begin];
    else return load_logit<kDtype>(x, i);
  }
  __device__ __forceinline__ float weight(float l) const { return expf((l - top) / temperature); }
};

__device__ __forceinline__ Message warp_join(Message m) {
  m.u = warp_max_u64(m.u);
  m.f = warp_sum(m.f);
  m.g = warp_sum(m.g);
  m.c = __reduce_add_sync(~0u, m.c);
  return m;
}

// Joins every thread's (max u, sum f, sum g, sum c) over the CTA and tells it to every CTA of the cluster; returns what
// they all said, joined, and in `prior` the sum of c over the CTAs of lower rank. s.warp keeps the warps' parts. A
// message is overwritten two exchanges later, when every CTA has passed the cluster.sync() in between.
template <class R>
__device__ __forceinline__ Message exchange(Message m, const R& r, SampleSmem& s, cg::cluster_group& cluster, int& turn,
                                            int& prior) {
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  m = warp_join(m);
  if ((threadIdx.x & 31) == 0) s.warp[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x < 32) {
    m = warp_join(threadIdx.x < kWarps ? s.warp[threadIdx.x] : Message{0, 0.0f, 0.0f, 0, 0.0f});
    const int token = place_index(m.u);
    m.l = token >= r.begin && token < r.end ? r.logit(token) : 0.0f;
    if (static_cast<int>(threadIdx.x) < ctas) *cluster.map_shared_rank(&s.said[turn][rank], threadIdx.x) = m;
  }
  cluster.sync();
  Message all{0, 0.0f, 0.0f, 0, 0.0f};
  for (int i = 0; i < ctas; ++i) {
    const Message o = s.said[turn][i];
    if (o.u > all.u) all.u = o.u, all.l = o.l;
    all.f += o.f;
    all.g += o.g;
    if (i == rank) prior = all.c;
    all.c += o.c;
  }
  turn ^= 1;
  return all;
}
template <class R>
__device__ __forceinline__ Message exchange(const Message& m, const R& r, SampleSmem& s, cg::cluster_group& cluster,
                                            int& turn) {
  int prior;
  return exchange(m, r, s, cluster, turn, prior);
}

// The random numbers of the thread's kAhead tokens from i0 on.
template <int kDtype, bool kResident>
struct Noise {
  float e[kAhead];
  __device__ __forceinline__ Noise(const Row<kDtype, kResident>& r, int i0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * kThreads;
      e[j] = i < r.end ? r.noise[i] : 1.0f;
    }
  }
};

// The race among the tokens placed before (above) `limit` (0: all): score_place of
// the CTA's winner in full evaluation, 0 if it has no token there. kFirst: also, per
// thread, the sums of exp(l - top) and, if asked, of exp((l - top) / temperature).
template <bool kFirst, int kDtype, bool kResident>
__device__ __forceinline__ uint64_t race(const Row<kDtype, kResident>& r, uint64_t limit, float least, bool mass,
                                         const Noise<kDtype, kResident>& ahead, SampleSmem& s, float& raw, float& all) {
  // kAhead tokens at a time: their largest, and which kAhead the thread's largest came from
  float best = -INFINITY, second = -INFINITY, e[kAhead];
  int best_at = r.end;
  const bool filtered = limit != 0 || least > -INFINITY;
#pragma unroll
  for (int j = 0; j < kAhead; ++j) e[j] = ahead.e[j];
  for (int i0 = r.begin + static_cast<int>(threadIdx.x); i0 < r.end; i0 += kAhead * kThreads) {
    float t[kAhead];
    const Noise<kDtype, kResident> next(r, i0 + kAhead * kThreads);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * kThreads;
      const float l = i < r.end ? r.logit(i) : -INFINITY, gap = l - r.top;
      if constexpr (kFirst) {
        raw += ex2(gap * kLog2e);
        if (mass) all += ex2(gap * r.scale);
      }
      t[j] = fmaf(gap, r.scale, 383.0f) - log2_below_383(fmaxf(e[j], kMinNoise));
      if (filtered && (gap * r.scale < least || (limit != 0 && place_of(l, i) <= limit))) t[j] = -INFINITY;
    }
#pragma unroll
    for (int n = kAhead / 2; n > 0; n /= 2)
#pragma unroll
      for (int j = 0; j < n; ++j) t[j] = fmaxf(t[j], t[j + n]);
    second = fmaxf(second, fminf(t[0], best));
    if (t[0] > best) best = t[0], best_at = i0;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) e[j] = next.e[j];
  }
  // the CTA's largest, then full evaluation of all that come near it
  float top = best;
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  if ((threadIdx.x & 31) == 0) s.scan[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) top = fmaxf(top, s.scan[i]);
  uint64_t won = 0;
  if (best > -INFINITY && best >= top - kNear) {
    // two of this thread's kAhead are near: look at all its tokens again
    const int from = second >= top - kNear ? r.begin + static_cast<int>(threadIdx.x) : best_at;
    const int to = second >= top - kNear ? r.end : min(best_at + kAhead * kThreads, r.end);
#pragma unroll 4
    for (int i = from; i < to; i += kThreads) {
      const float l = r.logit(i), gap = l - r.top, e = fmaxf(r.noise[i], kMinNoise);
      if (fmaf(gap, r.scale, 383.0f) - log2_below_383(e) >= top - kNear && gap * r.scale >= least && (limit == 0 || place_of(l, i) > limit))
        won = max(won, score_place(r.weight(l) / e, i));
    }
  }
  return won;
}

// Of a count per thread (cut_sums), or the CTAs' counts in s.bins added over the
// cluster, completed before a cluster.sync() (cut_bins): the first bin up to which
// they reach `least` (kBins where none does), the sum up to it and the sum before it.
struct Cut {
  int bin, upto, before;
};
__device__ __forceinline__ Cut cut_sums(int c, int least, SampleSmem& s) {
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, c, o);
    if ((threadIdx.x & 31) >= o) c += y;
  }
  s.all[threadIdx.x] = c;
  __syncthreads();
  Cut r{kBins, 0, 0};
  for (int b0 = 0; b0 < kBins && r.bin == kBins; b0 += 32) {
    const int upto = r.upto + s.all[b0 + (threadIdx.x & 31)];
    const uint32_t enough = __ballot_sync(~0u, upto >= least);
    const int at = enough != 0 ? __ffs(enough) - 1 : 31;
    const int prior = __shfl_sync(~0u, upto, max(at - 1, 0));
    r.before = at > 0 ? prior : r.upto;
    r.upto = __shfl_sync(~0u, upto, at);
    if (enough != 0) r.bin = b0 + at;
  }
  return r;
}
__device__ __forceinline__ Cut cut_bins(int least, SampleSmem& s, cg::cluster_group& cluster) {
  int c = 0;
  const int ctas = static_cast<int>(cluster.num_blocks());
#pragma unroll
  for (int i = 0; i < kMaxCluster; ++i)
    if (i < ctas) c += *cluster.map_shared_rank(&s.bins[threadIdx.x], i);
  return cut_sums(c, least, s);
}

// A place that the first top_k tokens lie before (above), and the number of tokens
// before it: top_k, or for small top_k at most kList. By counts of the range that the
// last of them lies in, kBins-fold smaller each time.
template <int kDtype, bool kResident>
__device__ __forceinline__ uint64_t kth_limit(const Row<kDtype, kResident>& r, int top_k, SampleSmem& s,
                                              cg::cluster_group& cluster, int& left) {
  uint64_t lo = 0, hi = place_of(r.top, 0);  // the last of the first top_k lies in (lo, hi]
  int above = 0;                             // tokens above hi
  for (;;) {
    int shift = 0;
    while (((hi - lo - 1) >> shift) >= kBins) ++shift;
    cluster.sync();  // the counts of the step before were read
    s.bins[threadIdx.x] = 0;
    __syncthreads();
    for (int i = r.begin + static_cast<int>(threadIdx.x); i < r.end; i += kThreads) {
      const uint64_t place = place_of(r.logit(i), i);
      if (place > lo && place <= hi) atomicAdd(&s.bins[(hi - place) >> shift], 1);
    }
    cluster.sync();
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
  Message m{0, 0.0f, 0.0f, 0, 0.0f};
  for (int i = r.begin + static_cast<int>(threadIdx.x); i < r.end; i += kThreads) {
    const float l = r.logit(i);
    if (place_of(l, i) > limit) ++m.c, m.f += r.weight(l);
  }
  return exchange(m, r, s, cluster, turn);
}

__device__ __forceinline__ uint64_t block_max(uint64_t v, SampleSmem& s) {
  v = warp_max_u64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.warp[threadIdx.x >> 5].u = v;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) v = max(v, s.warp[i].u);
  return v;
}
__device__ __forceinline__ float block_sum(float v, SampleSmem& s) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.scan[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < kWarps; ++i) v += s.scan[i];
  return v;
}

// Every filter and the race among the n places of rank 0's list: the winner's place.
// The last of the first top_k lies in (lo, hi]. `whole` is the mass that top_p refers to, or < 0: that of the first top_k.
template <int kDtype, bool kResident>
__device__ __forceinline__ uint64_t finish(const Row<kDtype, kResident>& r, int n, int top_k, uint64_t lo, uint64_t hi,
                                           float top_p, float min_p, float whole, SampleSmem& s) {
  constexpr int kPer = kList / kThreads;
  uint64_t v[kPer];  // 0: none, or out
  float e[kPer];
#pragma unroll
  for (int m = 0; m < kPer; ++m) {
    const int i = m * kThreads + static_cast<int>(threadIdx.x);
    v[m] = i < n ? s.list[i] : 0;
    e[m] = i < n ? fmaxf(r.noise[place_index(v[m])], kMinNoise) : 1.0f;
  }
  if (n > top_k && n <= kFew) {  // count for each how many come before it
    int place = 0;
    for (int i = 0; i < n; ++i) place += s.list[i] > v[0];
    if (place >= top_k) v[0] = 0;
  } else if (n > top_k) {
    // the place that top_k tokens lie above, as in kth_limit
    int above = 0;
#pragma unroll
    for (int m = 0; m < kPer; ++m) above += __syncthreads_count(v[m] > hi);
    for (int shift = 64; shift > 0;) {
      for (shift = 0; ((hi - lo - 1) >> shift) >= kBins;) ++shift;
      __syncthreads();
      s.bins[threadIdx.x] = 0;
      __syncthreads();
#pragma unroll
      for (int m = 0; m < kPer; ++m)
        if (v[m] > lo && v[m] <= hi) atomicAdd(&s.bins[(hi - v[m]) >> shift], 1);
      __syncthreads();
      const Cut cut = cut_sums(s.bins[threadIdx.x], top_k - above, s);
      const uint64_t to = hi - (static_cast<uint64_t>(cut.bin) << shift), step = 1ull << shift;
      lo = to - lo > step ? to - step : lo;
      hi = to;
      if (above + cut.upto == top_k) break;
      above += cut.before;
      if (cut.upto - cut.before <= kFew) {  // few in this bin: count for each how many of them come before it
        uint64_t* few = reinterpret_cast<uint64_t*>(s.bins);
        if (threadIdx.x == 0) s.base = 0;
        __syncthreads();  // also: the counts were read
#pragma unroll
        for (int m = 0; m < kPer; ++m)
          if (v[m] > lo && v[m] <= hi) few[atomicAdd(&s.base, 1)] = v[m];
        __syncthreads();
#pragma unroll
        for (int m = 0; m < kPer; ++m)
          if (v[m] > lo && v[m] <= hi) {
            int place = above;
            for (int i = 0; i < cut.upto - cut.before; ++i) place += few[i] > v[m];
            if (place >= top_k) v[m] = 0;
          }
        break;
      }
    }
#pragma unroll
    for (int m = 0; m < kPer; ++m)
      if (v[m] <= lo) v[m] = 0;
  }
  float w[kPer], own = 0.0f;
  uint64_t score[kPer];
#pragma unroll
  for (int m = 0; m < kPer; ++m) {
    w[m] = v[m] != 0 ? r.weight(place_logit(v[m])) : 0.0f;
    own += w[m];
    score[m] = 0;
    if (v[m] != 0 && w[m] >= min_p && place_logit(v[m]) > -INFINITY) {
      score[m] = score_place(w[m] / e[m], place_index(v[m]));
    }
  }
  if (whole < 0.0f && top_p < 1.0f) whole = block_sum(own, s);
  const double cut = static_cast<double>(top_p) * whole;
  for (uint64_t limit = 0;;) {
    uint64_t best = 0;
#pragma unroll
    for (int m = 0; m < kPer; ++m)
      if (v[m] > limit) best = max(best, score[m]);
    best = block_max(best, s);
#pragma unroll
    for (int m = 0; m < kPer; ++m)
      if (score[m] == best && v[m] > limit) s.list[0] = v[m];  // one thread: a token's score_place is its own
    __syncthreads();
    const uint64_t winner = s.list[0];
    if (top_p >= 1.0f) return winner;
    float mass = 0.0f;
#pragma unroll
    for (int m = 0; m < kPer; ++m)
      if (v[m] > winner) mass += w[m];
    if (static_cast<double>(block_sum(mass, s)) < cut) return winner;
    limit = winner;
  }
}

// One cluster per row.
template <int kDtype, bool kResident>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleSmem& s = *reinterpret_cast<SampleSmem*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t row = blockIdx.x / cluster.num_blocks();
  constexpr int kItem = kDtype == WBK_DT_F32 ? 4 : 2, kVec = 16 / kItem;
  int turn = 0;
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  griddep_launch_dependents();
  griddep_wait();
  const uint8_t* logits = static_cast<const uint8_t*>(p.logits) + row * p.logits_stride * kItem;
  Row<kDtype, kResident> r;
  r.noise = p.noise + row * p.noise_stride;
  r.begin = min(rank * p.slice, p.vocab);
  r.end = min(r.begin + p.slice, p.vocab);

  // ---- 1. the row's largest logit; the cleaned slice goes to shared memory
  // whole 16-byte vectors [v0, v1) of the slice, and the few tokens before and after them
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(logits + static_cast<int64_t>(r.begin) * kItem) & 15) / kItem);
  const int head = min((kVec - shift) % kVec, r.end - r.begin);
  const int vecs = (r.end - r.begin - head) / kVec;
  float* held = reinterpret_cast<float*>(smem_raw + (sizeof(SampleSmem) + 15) / 16 * 16) + (kVec - head) % kVec;
  const uint8_t* from = logits + static_cast<int64_t>(r.begin + head) * kItem;
  float top = -INFINITY;
  for (int v0 = threadIdx.x; v0 < vecs; v0 += kVecs * kThreads) {
    uint4 v[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
      if (v0 + j * kThreads < vecs) v[j] = reinterpret_cast<const uint4*>(from)[v0 + j * kThreads];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      if (v0 + j * kThreads >= vecs) break;
      float f[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        f[i] = load_logit<kDtype>(&v[j], i);
        top = fmaxf(top, f[i]);
      }
      if constexpr (kResident) {
        float4* to = reinterpret_cast<float4*>(held + head + (v0 + j * kThreads) * kVec);
        to[0] = make_float4(f[0], f[1], f[2], f[3]);
        if constexpr (kVec == 8) to[1] = make_float4(f[4], f[5], f[6], f[7]);
      }
    }
  }
  const int rest = r.end - r.begin - vecs * kVec;  // fewer than 2 * kVec tokens, the first `head` of them in front
  if (static_cast<int>(threadIdx.x) < rest) {
    const int i = static_cast<int>(threadIdx.x) < head ? threadIdx.x : vecs * kVec + threadIdx.x;
    const float f = load_logit<kDtype>(logits, r.begin + i);
    top = fmaxf(top, f);
    if constexpr (kResident) held[i] = f;
  }
  r.x = kResident ? static_cast<const void*>(held) : logits;
  s.bins[threadIdx.x] = 0;
  const float temperature = p.temperature != nullptr ? p.temperature[row] : p.temperature_all;
  const float top_p = p.top_p != nullptr ? p.top_p[row] : p.top_p_all;
  const float min_p = p.min_p != nullptr ? p.min_p[row] : p.min_p_all;
  const int k_given = p.top_k != nullptr ? p.top_k[row] : p.top_k_all;
  const int top_k = k_given > 0 && k_given < p.vocab ? k_given : p.vocab;
  r.temperature = fminf(temperature, 1e30f);  // an infinite one, too, leaves masked tokens at p = 0
  r.scale = fminf(kLog2e / r.temperature, 3e38f);
  const Message none{0, 0.0f, 0.0f, 0, 0.0f};
  Message m = none;
  m.u = place_of(top, -1);  // no token's place
  const Noise<kDtype, kResident> first(r, r.begin + static_cast<int>(threadIdx.x));  // for the race, on its way meanwhile
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // every CTA of the cluster has started
  r.top = place_logit(exchange(m, r, s, cluster, turn).u);

  uint64_t winner = 0;  // a place
  float raw = 0.0f;     // sum of exp(l - top)
  const bool empty = r.top == -INFINITY;
  const bool first_only = !(temperature > 0.0f) || !(top_p > 0.0f) || !(min_p <= 1.0f);  // nothing else is kept
  if (!empty && first_only) {
    m = none;
    for (int i = r.begin + static_cast<int>(threadIdx.x); i < r.end; i += kThreads) {
      const float gap = r.logit(i) - r.top;
      m.f += ex2(gap * kLog2e);
      if (gap == 0.0f) m.u = max(m.u, place_of(r.top, i));
    }
    m = exchange(m, r, s, cluster, turn);
    winner = m.u;
    raw = m.f;
  } else if (!empty) {
    const float least = min_p > 0.0f ? lg2(min_p) - kSlack : -INFINITY;  // of log2 p, for the race
    uint64_t limit = 0;    // every token at or after this place is out
    int left = p.vocab;    // tokens before it
    float whole = -1.0f;   // the mass top_p refers to
    Cut cut{kBins, 0, 0};  // or: what is left are the tokens of the bins up to this
    bool tight = false;    // .. and the last of the first top_k lies in the last of them
    bool gather = false;   // what is left fits one CTA's list
    int mine = -1, prior;  // this thread's tokens of what is left, where they were counted; those of the CTAs before
    const auto in = [&](int i, float l) {
      return cut.bin < kBins ? (r.top - l) * kBinsPerUnit < cut.bin + 1 : place_of(l, i) > limit;
    };
    if (top_k <= kList && top_k < p.vocab) {
      // ---- 2a. bins by distance from the maximum. Up to where as many threads' maxima lie as top_k there are at least
      // as many tokens, and not many more where these are few.
      if (top_k <= static_cast<int>(cluster.num_blocks()) * kThreads / 2) {
        const float bin = (r.top - top) * kBinsPerUnit;
        if (bin < kBins) atomicAdd(&s.bins[static_cast<int>(bin)], 1);
        cluster.sync();
        cut = cut_bins(top_k, s, cluster);
      }
      m = none;
      for (int i = r.begin + static_cast<int>(threadIdx.x); i < r.end; i += kThreads) {
        const float gap = r.top - r.logit(i);
        m.f += ex2(-gap * kLog2e);
        m.c += gap * kBinsPerUnit < cut.bin + 1;
      }
      mine = m.c;
      m = exchange(m, r, s, cluster, turn, prior);
      raw = m.f;
      left = m.c;
      gather = true;
      if (cut.bin == kBins || left > kList) {  // count the tokens
        mine = -1;
        s.bins[threadIdx.x] = 0;
        __syncthreads();
        for (int i = r.begin + static_cast<int>(threadIdx.x); i < r.end; i += kThreads) {
          const float bin = (r.top - r.logit(i)) * kBinsPerUnit;
          if (bin < kBins) atomicAdd(&s.bins[static_cast<int>(bin)], 1);
        }
        cluster.sync();
        cut = cut_bins(top_k, s, cluster);
        tight = cut.bin < kBins && cut.upto <= kList;
        if (tight) left = cut.upto;
        else cut.bin = kBins, limit = kth_limit(r, top_k, s, cluster, left);  // still further, or many ties
      }
    } else {
      if (top_k < p.vocab) {
        limit = kth_limit(r, top_k, s, cluster, left);
        whole = before(r, limit, s, cluster, turn).f;
      }
      // ---- 2b. rounds
      for (int round = 0;; ++round) {
        float all = 0.0f;
        Message w = none;
        if (round == 0) {
          w.u = race<true>(r, limit, least, top_p < 1.0f && whole < 0.0f, first, s, w.f, w.g);
          w = exchange(w, r, s, cluster, turn);
          raw = w.f;
          if (whole < 0.0f) whole = w.g;
        } else {
          w.u = race<false>(r, limit, least, false, first, s, all, all);
          w = exchange(w, r, s, cluster, turn);
        }
        winner = place_of(w.l, place_index(w.u));
        if (top_p >= 1.0f && r.weight(w.l) >= min_p) break;
        const Message b = before(r, winner, s, cluster, turn);
        if (r.weight(w.l) >= min_p && (top_p >= 1.0f || static_cast<double>(b.f) < static_cast<double>(top_p) * whole)) break;
        limit = winner;
        left = b.c;
        gather = left <= kList;
        if (gather) break;
        if (round >= kRounds) {
          uint64_t lo = limit, hi = place_of(r.top, 0);  // the cut lies between these places
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
          w = none;
          w.u = race<false>(r, limit, -INFINITY, false, first, s, all, all);
          w = exchange(w, r, s, cluster, turn);
          winner = place_of(w.l, place_index(w.u));
          break;
        }
      }
    }
    if (gather) {
      // ---- what is left goes to rank 0: counted first, so that each thread knows its place in the list
      if (mine < 0) {
        m = none;
        for (int i = r.begin + static_cast<int>(threadIdx.x); i < r.end; i += kThreads) m.c += in(i, r.logit(i));
        mine = m.c;
        exchange(m, r, s, cluster, turn, prior);
      }
      int upto = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, upto, o);
        if ((threadIdx.x & 31) >= o) upto += y;
      }
      int at = prior + upto - mine;
      for (int i = 0; i < static_cast<int>(threadIdx.x >> 5); ++i) at += s.warp[i].c;
      if (mine > 0) {
        uint64_t* list = cluster.map_shared_rank(&s.list[0], 0);
        for (int i = r.begin + static_cast<int>(threadIdx.x); i < r.end; i += kThreads) {
          const float l = r.logit(i);
          if (in(i, l) && at < kList) list[at++] = place_of(l, i);
        }
      }
      cluster.sync();
      if (rank == 0) {
        uint64_t hi = place_of(r.top, 0);
        if (cut.bin < kBins) {  // one bin more on both sides covers rounding
          if (tight && cut.bin > 1) hi = place_of(r.top - (cut.bin - 1) / kBinsPerUnit, 0);
          limit = static_cast<uint64_t>(order_key(r.top - (cut.bin + 2) / kBinsPerUnit)) << 32;
        }
        winner = finish(r, min(left, kList), top_k, limit, hi, top_p, min_p, whole, s);
      }
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    p.tokens[row] = empty ? -1 : place_index(winner);
    p.logprobs[row] = empty ? -INFINITY : (place_logit(winner) - r.top) - logf(raw);
  }
}

template <int kDtype, bool kResident>
int launch_sample(const SampleParams& p, int64_t rows, int ctas, cudaStream_t stream) {
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
                                                  cudaFuncAttributeMaxDynamicSharedMemorySize, kFixed + kSliceElems * 4 + 32),
                             "sample smem attribute"))
        return e;
      configured[dev] = 1;
    }
  }
  return cuda_check(launch_after(sample_kernel<kDtype, kResident>, dim3(static_cast<unsigned>(rows * ctas)), kThreads,
                                 kFixed + (kResident ? p.slice * 4 + 32 : 0), stream, static_cast<unsigned>(ctas), p),
                    "sample launch");
}

template <int kDtype>
int dispatch_sample(SampleParams p, int64_t rows, cudaStream_t stream) {
  // A row is split as far as keeps every CTA of all rows resident at once (a row alone is a chain of latencies, which
  // smaller slices shorten: 51866 logits, one row: 8 CTAs), and as far as its slices need to fit shared memory.
  const int64_t room = static_cast<int64_t>(sm_count() > 0 ? sm_count() : 148) * kCtasPerSm;
  int ctas = 1;
  while (ctas < kMaxCluster && ((p.vocab + ctas - 1) / ctas > kSliceElems ||
                                (p.vocab / (2 * ctas) >= kLeastSlice && rows * 2 * ctas <= room)))
    ctas *= 2;
  p.slice = ((p.vocab + ctas - 1) / ctas + 7) / 8 * 8;
  if (rows * ctas > (int64_t(1) << 31) - 1) return fail(WBK_ERR_UNSUPPORTED, "wbk_sample: too many rows");
  return p.slice <= kSliceElems ? launch_sample<kDtype, true>(p, rows, ctas, stream)
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
