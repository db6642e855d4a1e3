// Arithmetic of the 8-bit key/value cache shared by the kernels that write it
// and the kernels that read it: 16-bit inputs as fp32, the power-of-two scale of
// a page and head, and codes to and from fp32 / fp16.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "wbk_common.cuh"

struct CUtensorMap_st;

namespace wbk {

// Smallest scale exponent: a page of zeros (or of values too small to matter)
// has scale 2^-64, so 1 / scale and products of two scales stay normal fp32.
constexpr int kKv8MinExp = -64;

// Pages of one cache: codes [pages, kv_heads, block, head_dim], scales
// [pages, kv_heads], and the block table of a batch (row b names the pages of
// sequence b in order).
struct Kv8Pages {
  int64_t pages;
  int kv_heads;
  int block;  // tokens per page, a power of two 16..128
  int block_log2;
  const int32_t* table;
  int64_t table_stride;  // elements between rows of the table
  int max_blocks;
};

// The page that holds position `blk * block ...` of sequence b; -1 when the table
// does not reach so far or names no page of the pool.
__device__ __forceinline__ int64_t kv8_page(const Kv8Pages& c, int b, int blk) {
  if (blk < 0 || blk >= c.max_blocks) return -1;
  const int64_t page = c.table[b * c.table_stride + blk];
  return page >= 0 && page < c.pages ? page : -1;
}

// Exponent E of the page scale 2^E: the least E >= kKv8MinExp with
// amax <= max_fp8 * 2^E. max_fp8 is 1.75 * 2^8 (E4M3) or 1.75 * 2^15 (E5M2), so
// this is a comparison of the significand of amax with 1.75 -- exact, without
// a division or a logarithm. amax is finite and >= 0.
template <int kFmt>
__device__ __forceinline__ int kv8_scale_exp(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>(bits >> 23) - 127 - (kFmt == WBK_FMT_E4M3 ? 8 : 15) + ((bits & 0x7FFFFFu) > 0x600000u);
  return e > kKv8MinExp ? e : kKv8MinExp;
}

// 2^e as fp32, e in [-126, 127].
__device__ __forceinline__ float kv8_pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

template <int kFmt>
__device__ __forceinline__ constexpr __nv_fp8_interpretation_t kv8_interp() {
  return kFmt == WBK_FMT_E4M3 ? __NV_E4M3 : __NV_E5M2;
}

// Two fp32 values, already divided by the scale -> two codes (low byte first),
// rounded to nearest even, saturated to +-max_fp8. NaN becomes -max_fp8, as in
// every quantiser of this library (fmaxf returns the operand that is not NaN).
template <int kFmt>
__device__ __forceinline__ uint32_t kv8_codes2(float a, float b) {
  constexpr float mx = kFmt == WBK_FMT_E4M3 ? 448.0f : 57344.0f;
  return __nv_cvt_float2_to_fp8x2(make_float2(fmaxf(a, -mx), fmaxf(b, -mx)), __NV_SATFINITE, kv8_interp<kFmt>());
}

// Two codes (low byte first) -> packed fp16 pair; exact for both formats.
template <int kFmt>
__device__ __forceinline__ __half2 kv8_half2(uint32_t codes) {
  return __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes & 0xFFFFu), kv8_interp<kFmt>()));
}

// Four codes -> two packed fp16 pairs (exact).
template <int kFmt>
__device__ __forceinline__ uint2 kv8_half4(uint32_t codes) {
  uint2 r;
  if constexpr (kFmt == WBK_FMT_E4M3)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(r.x), "=r"(r.y) : "r"(codes));
  else
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e5m2x2 %0, l;\n\tcvt.rn.f16x2.e5m2x2 %1, h;\n\t}"
        : "=r"(r.x), "=r"(r.y) : "r"(codes));
  return r;
}

// log2 of a scale, exact for powers of two.
__device__ __forceinline__ float kv8_log2(float s) {
  const int e = static_cast<int>(__float_as_uint(s) >> 23) - 127;
  return (__float_as_uint(s) & 0x7FFFFFu) == 0 ? static_cast<float>(e) : log2f(s);
}

// A packed pair of the 16-bit input type as fp32.
template <int kDtype>
__device__ __forceinline__ float2 pair_to_float2(uint32_t w) {
  if constexpr (kDtype == WBK_DT_F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// fp32 pair -> packed pair of the 16-bit output type, rounded to nearest even.
template <int kDtype>
__device__ __forceinline__ uint32_t float2_to_pair(float a, float b) {
  if constexpr (kDtype == WBK_DT_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Softmax weights are held relative to 2^(m - kKv8Lift), m the row's running maximum, which is passed by 2^8 at most:
// the largest is 2^15, the top of fp16's range. Rounded to fp16 a weight is then off by at most 2^-11 of itself and, below
// fp16's normal range, 2^-25 * 2^-7 of the largest. Sums and totals carry the same factor.
constexpr float kKv8Lift = 7.0f;

// Length of sequence b, held to what the block table can address.
__device__ __forceinline__ int kv8_len(const int32_t* lens, int b, const Kv8Pages& c) {
  const int64_t cap = static_cast<int64_t>(c.max_blocks) * c.block;
  const int64_t n = lens[b];
  return static_cast<int>(n < 0 ? 0 : n < cap ? n : cap);
}

// A call of attention over the cache, checked.
struct Kv8Attention {
  const void* q;
  void* out;
  int64_t q_sb, q_sh, q_ss, o_sb, o_sh, o_ss;  // element strides: sequence, head, position
  Kv8Pages c;
  const void *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int32_t* lens;
  const int32_t* q_lens;  // or NULL
  int batch, group, queries, head_dim;  // group: query heads per KV head
  int fmt, causal, bf16;
  float scale_log2;  // scale * log2(e)
};

// A workspace begins with tickets, zero between calls, as many as the SMs can have CTAs or a CTA 32-row parts; partial
// results follow. Both kernels of attention keep to this, so one workspace serves calls of either.
constexpr int kKv8TicketsPerSm = 8;
int64_t kv8_ticket_bytes();

// Attention for many query rows per KV head (wbk_kv8_prompt.cu), its workspace and its device error word.
int kv8_prompt_attention(const Kv8Attention& a, void* workspace, cudaStream_t stream);
int64_t kv8_prompt_ws_bytes(int64_t head_dim);
// A tensor map of pages (channel, head * block + token, page) with boxes of at most `tile` tokens of one page and head,
// swizzled over the row length or not.
int kv8_make_tmap(CUtensorMap_st* map, const void* base, const Kv8Attention& a, int tile, bool swizzle);

// Host: the checks of cache geometry that the cache's entry points share.
int kv8_check_pages(const char* what, const void* k_cache, const void* v_cache, const float* k_scale,
                    const float* v_scale, int64_t pages, int64_t kv_heads, int64_t block, int64_t head_dim, int fmt,
                    const int32_t* block_table, int64_t max_blocks, int64_t table_stride, const int32_t* seq_lens);
// Element stride of a batch, head or position: TMA and 16-byte accesses need multiples of 8.
inline bool kv8_stride_ok(int64_t s) { return s >= 0 && s % 8 == 0 && s < (int64_t(1) << 40); }
Kv8Pages kv8_pages(int64_t pages, int64_t kv_heads, int64_t block, const int32_t* block_table, int64_t max_blocks,
                   int64_t table_stride);

}  // namespace wbk
