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
// No sort: the winner of that race among all tokens (above top_k's threshold
// and min_p) is the answer if it is kept. If it is not, nothing after it in the
// order is kept either, so the race is run again among the tokens before it. Each
// round throws away a random share of what is left, so a few rounds are enough.
#include "wbk_common.cuh"
#include "wbk_kv8.cuh"

namespace wbk {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

struct SampleParams {
  const void* logits;
  int64_t logits_stride;
  const float* noise;
  int64_t noise_stride;
  const float *temperature, *top_p, *min_p;  // per row, or NULL: the numbers below
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int vocab;
  int64_t* tokens;
  float* logprobs;
};

// Logit as an ordered fp32: NaN is never drawn (-inf), +inf is the largest finite
// number, -0 is +0.
template <int kDtype>
__device__ __forceinline__ float load_logit(const void* row, int i) {
  float x;
  if constexpr (kDtype == WBK_DT_F32) x = static_cast<const float*>(row)[i];
  else if constexpr (kDtype == WBK_DT_F16) x = __half2float(static_cast<const __half*>(row)[i]);
  else x = __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
  return isnan(x) ? -INFINITY : fminf(x, 3.402823466e38f) + 0.0f;
}

// Order-preserving key of an fp32, and the place of token i in its row's order:
// larger is earlier.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t place_of(uint32_t key, int i) {
  return (static_cast<uint64_t>(key) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

// Block-wide sums and maxima in a fixed order, so equal inputs give equal bits.
struct Reduce {
  uint64_t u[kWarps];
  float f[kWarps];
  int c[kWarps];
};
__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, Reduce& r) {
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) r.u[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) v = max(v, r.u[i]);
  return v;
}
__device__ __forceinline__ float block_sum_f(float v, Reduce& r) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) r.f[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < kWarps; ++i) v += r.f[i];
  return v;
}
__device__ __forceinline__ int block_sum_i(int v, Reduce& r) {
  v = __reduce_add_sync(~0u, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) r.c[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < kWarps; ++i) v += r.c[i];
  return v;
}

// One CTA per row.
template <int kDtype>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  __shared__ Reduce red;
  const int64_t row = blockIdx.x;
  const int n = p.vocab;
  constexpr int kItem = kDtype == WBK_DT_F32 ? 4 : 2;
  const void* logits = static_cast<const uint8_t*>(p.logits) + row * p.logits_stride * kItem;
  const float* noise = p.noise + row * p.noise_stride;
  const float temperature = p.temperature != nullptr ? p.temperature[row] : p.temperature_all;
  const float top_p = p.top_p != nullptr ? p.top_p[row] : p.top_p_all;
  const float min_p = p.min_p != nullptr ? p.min_p[row] : p.min_p_all;
  const int top_k = p.top_k != nullptr ? p.top_k[row] : p.top_k_all;

  // the first token of the order
  uint64_t first = 0;
  for (int i = threadIdx.x; i < n; i += kThreads)
    first = max(first, place_of(order_key(load_logit<kDtype>(logits, i)), i));
  first = block_max_u64(first, red);
  const int first_i = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(first));
  const float top = load_logit<kDtype>(logits, first_i);
  if (top == -INFINITY) {  // nothing to draw
    if (threadIdx.x == 0) {
      p.tokens[row] = -1;
      p.logprobs[row] = -INFINITY;
    }
    return;
  }
  float raw = 0.0f;
  for (int i = threadIdx.x; i < n; i += kThreads) raw += expf(load_logit<kDtype>(logits, i) - top);
  raw = block_sum_f(raw, red);

  int winner = first_i;
  if (temperature > 0.0f) {
    // top_k: the key of the k-th token, by halving
    const bool some_k = top_k > 0 && top_k < n;
    uint32_t kth = 0;
    float kept_mass = 0.0f;
    if (some_k) {
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t tryk = kth | (1u << bit);
        int c = 0;
        for (int i = threadIdx.x; i < n; i += kThreads) c += order_key(load_logit<kDtype>(logits, i)) >= tryk;
        if (block_sum_i(c, red) >= top_k) kth = tryk;
      }
    }
    int above = 0;
    float tie = 0.0f;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float x = load_logit<kDtype>(logits, i);
      const uint32_t key = order_key(x);
      const float w = expf((x - top) / temperature);
      if (key > kth) kept_mass += w, ++above;
      else if (key == kth) tie = w;
    }
    kept_mass = block_sum_f(kept_mass, red);
    above = block_sum_i(above, red);
    if (some_k) kept_mass += (top_k - above) * __uint_as_float(static_cast<uint32_t>(block_max_u64(__float_as_uint(tie), red)));

    uint64_t limit = 0;  // the race is among the tokens placed before (above) this
    for (;;) {
      float best = -1.0f;
      int best_i = n;
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const float x = load_logit<kDtype>(logits, i);
        const uint32_t key = order_key(x);
        if (key < kth || place_of(key, i) <= limit || x == -INFINITY) continue;
        const float w = expf((x - top) / temperature);
        if (!(w >= min_p) && i != first_i) continue;
        const float score = w / fmaxf(noise[i], 1.17549435e-38f);
        if (score > best) best = score, best_i = i;
      }
      const uint64_t won = block_max_u64((static_cast<uint64_t>(order_key(best)) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(best_i)), red);
      winner = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(won));
      if (winner == first_i) break;
      const uint64_t place = place_of(order_key(load_logit<kDtype>(logits, winner)), winner);
      int before = 0;
      float mass = 0.0f;
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const float x = load_logit<kDtype>(logits, i);
        if (place_of(order_key(x), i) > place) ++before, mass += expf((x - top) / temperature);
      }
      before = block_sum_i(before, red);
      mass = block_sum_f(mass, red);
      if ((!some_k || before < top_k) && (top_p >= 1.0f || static_cast<double>(mass) < static_cast<double>(top_p) * kept_mass))
        break;
      limit = place;
    }
  }
  if (threadIdx.x == 0) {
    p.tokens[row] = winner;
    p.logprobs[row] = (load_logit<kDtype>(logits, winner) - top) - logf(raw);
  }
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
  const unsigned grid = static_cast<unsigned>(rows);
  if (dtype == WBK_DT_F16) sample_kernel<WBK_DT_F16><<<grid, kThreads, 0, st>>>(p);
  else if (dtype == WBK_DT_BF16) sample_kernel<WBK_DT_BF16><<<grid, kThreads, 0, st>>>(p);
  else sample_kernel<WBK_DT_F32><<<grid, kThreads, 0, st>>>(p);
  return cuda_check(cudaGetLastError(), "sample launch");
}

}  // extern "C"
