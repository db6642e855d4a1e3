// The 8-bit key/value cache of a decoder: appending new tokens to its pages.
//
// A page holds `block` tokens of one KV head as fp8 codes with one fp32 scale, a
// power of two. Scales are powers of two so that a page whose scale grows (a
// later token is larger than all before it) is re-coded by an exact shift of
// exponents: only values that fall into the format's subnormal range round a
// second time. What a sequence's cache holds then depends on its tokens and
// hardly on how they were split into appends, and a scale grows rarely.
#include <algorithm>

#include "wbk_kv8.cuh"

namespace wbk {

int kv8_check_pages(const char* what, const void* k_cache, const void* v_cache, const float* k_scale,
                    const float* v_scale, int64_t pages, int64_t kv_heads, int64_t block, int64_t head_dim, int fmt,
                    const int32_t* block_table, int64_t max_blocks, int64_t table_stride, const int32_t* seq_lens) {
  if (k_cache == nullptr || v_cache == nullptr || k_scale == nullptr || v_scale == nullptr || block_table == nullptr ||
      seq_lens == nullptr)
    return fail(WBK_ERR_INVALID_ARG, "%s: null pointer", what);
  if (fmt != WBK_FMT_E4M3 && fmt != WBK_FMT_E5M2) return fail(WBK_ERR_INVALID_ARG, "%s: unknown format %d", what, fmt);
  if (head_dim != 64 && head_dim != 128)
    return fail(WBK_ERR_UNSUPPORTED, "%s: head_dim %lld (64 or 128)", what, (long long)head_dim);
  if (block != 16 && block != 32 && block != 64 && block != 128)
    return fail(WBK_ERR_UNSUPPORTED, "%s: block %lld (16, 32, 64 or 128 tokens per page)", what, (long long)block);
  if (pages < 1 || kv_heads < 1 || max_blocks < 1 || table_stride < max_blocks)
    return fail(WBK_ERR_INVALID_ARG, "%s: bad cache size (pages %lld, kv_heads %lld, max_blocks %lld, table stride %lld)",
                what, (long long)pages, (long long)kv_heads, (long long)max_blocks, (long long)table_stride);
  if (pages > (int64_t(1) << 31) - 1 || kv_heads > 65535 || max_blocks * block > (int64_t(1) << 30))
    return fail(WBK_ERR_UNSUPPORTED, "%s: cache too large (pages %lld, kv_heads %lld, max_blocks %lld)", what,
                (long long)pages, (long long)kv_heads, (long long)max_blocks);
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16))
    return fail(WBK_ERR_UNSUPPORTED, "%s: cache pointers must be 16-byte aligned", what);
  if (!aligned(k_scale, 4) || !aligned(v_scale, 4) || !aligned(block_table, 4) || !aligned(seq_lens, 4))
    return fail(WBK_ERR_INVALID_ARG, "%s: misaligned scale, block table or length pointer", what);
  return WBK_OK;
}

Kv8Pages kv8_pages(int64_t pages, int64_t kv_heads, int64_t block, const int32_t* block_table, int64_t max_blocks,
                   int64_t table_stride) {
  Kv8Pages c{};
  c.pages = pages;
  c.kv_heads = static_cast<int>(kv_heads);
  c.block = static_cast<int>(block);
  c.block_log2 = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7;
  c.table = block_table;
  c.table_stride = table_stride;
  c.max_blocks = static_cast<int>(max_blocks);
  return c;
}

int64_t kv8_ticket_bytes() {
  const int sms = sm_count();
  return (static_cast<int64_t>(sms > 0 ? sms : 148) * kKv8TicketsPerSm * 4 + 255) / 256 * 256;
}

namespace {

// ------------------------------------------------------------------ append
//
// What bounds it: each new value is read once (2 bytes) and written once (1 byte), so
// HBM. A page and head is one CTA's work, held in registers between the maximum and
// the codes. The chain length -> page -> values -> maximum -> codes is all latency, so
// where there are enough CTAs to fill the SMs one takes several heads of its page, with
// the next head's values on their way meanwhile.
//
// Measured: 64 sequences of 1500 tokens, 20 heads of 64 (737 MB moved) 131 to 134 us,
// 5.5 to 5.6 TB/s, 0.85 of a plain copy's rate; one head per CTA, a page in two passes
// through shared memory: 146. 16 sequences of up to 1021 tokens, 8 heads of 128, into half-full
// pages (64 MB) 16 us, 4.0 TB/s. One token for each of 64 sequences 4.5 us, launch and
// that chain. The maximum is taken on 16-bit pairs as they are (exact), and a value's
// code is its one rounding: fp16 / bf16 times a power of two is exact in fp32.

struct AppendSide {
  const void* x;         // new keys or values, [batch, kv_heads, tokens, head_dim] view
  int64_t sb, sh, ss;    // its element strides
  uint8_t* cache;
  float* scale;
};

struct AppendParams {
  AppendSide side[2];
  Kv8Pages c;
  const int32_t* lens;
  const int32_t* fresh;  // new tokens of each sequence, or NULL: all
  int tokens;
  int heads_per_cta;
};

constexpr int kAppendVecs = 4;  // 16-byte vectors per thread, at most (8 KB per 128 threads)

// Larger of two packed pairs, lane by lane; NaN where both are.
template <int kDtype>
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (kDtype == WBK_DT_F16) asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int kDtype>
__device__ __forceinline__ float half_word_value(uint32_t bits) {
  return pair_to_float2<kDtype>(bits & 0xFFFFu).x;
}

// One CTA per touched page and heads_per_cta KV heads, for the keys or the values
// (blockIdx.y: heads, blockIdx.z: batch * 2 + side); kThreads threads hold a page of kThreads * kVec 16-byte vectors.
template <int kFmt, int kDtype, int kD, int kThreads, int kVec>
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(const AppendParams p) {
  constexpr int kWarps = kThreads / 32;
  griddep_launch_dependents();
  griddep_wait();
  const int b = blockIdx.z >> 1;
  const AppendSide& s = p.side[blockIdx.z & 1];
  const int len = kv8_len(p.lens, b, p.c);
  const int n = p.fresh != nullptr ? min(max(p.fresh[b], 0), p.tokens) : p.tokens;
  const int block = p.c.block;
  const int blk = (len >> p.c.block_log2) + blockIdx.x;
  const int start = blk << p.c.block_log2;                   // first position of the page
  const int slot0 = max(len - start, 0);                     // old tokens in it
  const int slot1 = static_cast<int>(min(static_cast<int64_t>(block), static_cast<int64_t>(len) + n - start));
  if (slot1 <= slot0) return;
  const int64_t page = kv8_page(p.c, b, blk);
  if (page < 0) return;
  const int h0 = blockIdx.y * p.heads_per_cta, h1 = min(h0 + p.heads_per_cta, p.c.kv_heads);
  constexpr int kPer = kD / 8;  // vectors per token
  const int vecs = (slot1 - slot0) * kPer;
  const uint16_t* x = static_cast<const uint16_t*>(s.x) + b * s.sb + static_cast<int64_t>(start + slot0 - len + threadIdx.x / kPer) * s.ss +
                      (threadIdx.x % kPer) * 8;
  const int64_t step = static_cast<int64_t>(kThreads / kPer) * s.ss;  // a thread's vectors lie in the same column
  auto load = [&](uint4 (&v)[kVec], int h) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (static_cast<int>(threadIdx.x) + i * kThreads < vecs) v[i] = ld_stream16(x + h * s.sh + i * step);
    }
  };
  __shared__ uint32_t red[2][kWarps];
  uint4 v[kVec];
  load(v, h0);
  for (int h = h0; h < h1; ++h) {
    const int64_t ph = page * p.c.kv_heads + h;
    const float old = slot0 > 0 ? s.scale[ph] : 0.0f;
    // ---- largest |x|: as 16-bit patterns, whose order is that of the values; NaN is passed over
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      top = pair_max<kDtype>(top, v[i].x & 0x7FFF7FFFu);
      top = pair_max<kDtype>(top, v[i].y & 0x7FFF7FFFu);
      top = pair_max<kDtype>(top, v[i].z & 0x7FFF7FFFu);
      top = pair_max<kDtype>(top, v[i].w & 0x7FFF7FFFu);
    }
    const int turn = (h - h0) & 1;
    top = warp_max_u32(max(top & 0xFFFFu, top >> 16));
    if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) top = max(top, red[turn][i]);
    float amax = half_word_value<kDtype>(top);
    if (isinf(amax)) {  // infinities do not count: again, without them (the same way in all threads)
      amax = 0.0f;
      for (int i = 0; i < kVec; ++i) {
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        for (int j = 0; j < 4; ++j) {
          const float2 f = pair_to_float2<kDtype>(w[j]);
          if (isfinite(f.x)) amax = fmaxf(amax, fabsf(f.x));
          if (isfinite(f.y)) amax = fmaxf(amax, fabsf(f.y));
        }
      }
      const uint32_t bits = warp_max_u32(__float_as_uint(amax));
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = bits;
      __syncthreads();
      for (int i = 0; i < kWarps; ++i) amax = fmaxf(amax, __uint_as_float(red[turn][i]));
    }
    // ---- the page's scale; older codes follow it where it grows
    uint8_t* codes = s.cache + ph * block * kD;
    int e = kv8_scale_exp<kFmt>(amax);
    float scale = kv8_pow2(e), inv = kv8_pow2(-e);
    if (slot0 > 0) {
      if (scale > old) {
        const float shift = old * inv;
        for (int i = threadIdx.x; i < slot0 * kD / 4; i += kThreads) {
          uint32_t* at = reinterpret_cast<uint32_t*>(codes) + i;
          const uint32_t w = *at;
          const float2 f = __half22float2(kv8_half2<kFmt>(w)), g = __half22float2(kv8_half2<kFmt>(w >> 16));
          *at = kv8_codes2<kFmt>(f.x * shift, f.y * shift) | (kv8_codes2<kFmt>(g.x * shift, g.y * shift) << 16);
        }
      } else {
        scale = old;
        inv = 1.0f / old;
      }
    }
    // ---- codes; the next head's values take the registers as they become free
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int id = threadIdx.x + i * kThreads;
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      uint32_t q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = f2_mul(pair_to_float2<kDtype>(w[j]), make_float2(inv, inv));
        q[j] = kv8_codes2<kFmt>(f.x, f.y);
      }
      if (id < vecs) {
        *reinterpret_cast<uint2*>(codes + slot0 * kD + id * 8) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
        if (h + 1 < h1) v[i] = ld_stream16(x + (h + 1) * s.sh + i * step);
      }
    }
    // with old tokens every thread has read the old scale: the sums' barrier lies in between
    if (threadIdx.x == 0) s.scale[ph] = scale;
  }
}

template <int kFmt, int kDtype, int kD>
int launch_append(const AppendParams& p, dim3 grid, cudaStream_t stream) {
  cudaError_t e;
  switch (p.c.block * kD / 8 / 128) {
    case 1: e = launch_after(kv8_append_kernel<kFmt, kDtype, kD, 128, 1>, grid, 128, 0, stream, 1, p); break;
    case 2: e = launch_after(kv8_append_kernel<kFmt, kDtype, kD, 128, 2>, grid, 128, 0, stream, 1, p); break;
    case 4: e = launch_after(kv8_append_kernel<kFmt, kDtype, kD, 128, kAppendVecs>, grid, 128, 0, stream, 1, p); break;
    case 8: e = launch_after(kv8_append_kernel<kFmt, kDtype, kD, 256, kAppendVecs>, grid, 256, 0, stream, 1, p); break;
    default: e = launch_after(kv8_append_kernel<kFmt, kDtype, kD, 256, 8>, grid, 256, 0, stream, 1, p); break;
  }
  return cuda_check(e, "kv8 append launch");
}

template <int kFmt>
int dispatch_append(const AppendParams& p, int dtype, int head_dim, dim3 grid, cudaStream_t stream) {
  if (dtype == WBK_DT_F16)
    return head_dim == 64 ? launch_append<kFmt, WBK_DT_F16, 64>(p, grid, stream) : launch_append<kFmt, WBK_DT_F16, 128>(p, grid, stream);
  return head_dim == 64 ? launch_append<kFmt, WBK_DT_BF16, 64>(p, grid, stream) : launch_append<kFmt, WBK_DT_BF16, 128>(p, grid, stream);
}

}  // namespace
}  // namespace wbk

using namespace wbk;

extern "C" {

int wbk_kv8_append(const void* k, const void* v, int dtype, int64_t batch, int64_t kv_heads, int64_t tokens,
                   int64_t head_dim, const int64_t* strides, int fmt, void* k_cache, void* v_cache, float* k_scale,
                   float* v_scale, int64_t pages, int64_t block, const int32_t* block_table, int64_t max_blocks,
                   int64_t table_stride, const int32_t* seq_lens, const int32_t* new_lens, wbk_stream_t stream) {
  if (batch < 0 || kv_heads < 0 || tokens < 0)
    return fail(WBK_ERR_INVALID_ARG, "wbk_kv8_append: negative size");
  if (dtype != WBK_DT_F16 && dtype != WBK_DT_BF16)
    return fail(WBK_ERR_INVALID_ARG, "wbk_kv8_append: dtype %d (WBK_DT_F16 or WBK_DT_BF16)", dtype);
  if (batch == 0 || kv_heads == 0 || tokens == 0) return WBK_OK;
  if (k == nullptr || v == nullptr || strides == nullptr)
    return fail(WBK_ERR_INVALID_ARG, "wbk_kv8_append: null pointer");
  if (int e = kv8_check_pages("wbk_kv8_append", k_cache, v_cache, k_scale, v_scale, pages, kv_heads, block, head_dim, fmt,
                              block_table, max_blocks, table_stride, seq_lens))
    return e;
  if (batch > 32767 || tokens > (1 << 30))
    return fail(WBK_ERR_UNSUPPORTED, "wbk_kv8_append: batch %lld (at most 32767) or %lld tokens", (long long)batch,
                (long long)tokens);
  if (new_lens != nullptr && !aligned(new_lens, 4))
    return fail(WBK_ERR_INVALID_ARG, "wbk_kv8_append: new_lens misaligned");
  if (!aligned(k, 16) || !aligned(v, 16))
    return fail(WBK_ERR_UNSUPPORTED, "wbk_kv8_append: k and v must be 16-byte aligned");
  for (int i = 0; i < 6; ++i)
    if (!kv8_stride_ok(strides[i]))
      return fail(WBK_ERR_UNSUPPORTED, "wbk_kv8_append: stride[%d] = %lld is not a multiple of 8 elements", i,
                  (long long)strides[i]);
  AppendParams p{};
  p.side[0] = {k, strides[0], strides[1], strides[2], static_cast<uint8_t*>(k_cache), k_scale};
  p.side[1] = {v, strides[3], strides[4], strides[5], static_cast<uint8_t*>(v_cache), v_scale};
  p.c = kv8_pages(pages, kv_heads, block, block_table, max_blocks, table_stride);
  p.lens = seq_lens;
  p.fresh = new_lens;
  p.tokens = static_cast<int>(tokens);
  // a run of `tokens` positions touches at most this many pages
  const int64_t touched = std::min<int64_t>((tokens + block - 2) / block + 1, max_blocks);
  // several heads per CTA once that still leaves the SMs two rounds of CTAs
  const int64_t units = touched * kv_heads * batch * 2, room = static_cast<int64_t>(sm_count() > 0 ? sm_count() : 148) * 16 * 2;
  p.heads_per_cta = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kv_heads, units / room)));
  const dim3 grid(static_cast<unsigned>(touched), static_cast<unsigned>((kv_heads + p.heads_per_cta - 1) / p.heads_per_cta),
                  static_cast<unsigned>(batch * 2));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return fmt == WBK_FMT_E4M3 ? dispatch_append<WBK_FMT_E4M3>(p, dtype, static_cast<int>(head_dim), grid, st)
                             : dispatch_append<WBK_FMT_E5M2>(p, dtype, static_cast<int>(head_dim), grid, st);
}

}  // extern "C"
