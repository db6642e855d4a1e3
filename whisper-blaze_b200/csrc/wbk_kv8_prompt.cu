// Attention over the 8-bit key/value cache for many query rows per KV head (a
// prompt, or a chunk of one) on the tcgen05 tensor cores.
//
// What bounds it: 4 * head_dim operations per query row and visible token on the
// tensor cores, and 128 * 128 exponentials per tile of scores; the codes are read
// from L2 as a rule.
//
//   * Codes cannot meet fp16 queries in one tcgen05.mma, so each 128-token tile of
//     codes is converted once per CTA, by a warpgroup of its own, into fp16
//     (keys: the queries' type, exact for both) in the swizzled layout that
//     the products read, and serves two tiles of 128 query rows: 1/16 of an
//     instruction per product of the tensor cores.
//   * Rows of a tile are (position, query head of the group), position first, so
//     the query heads that share a KV head share its tiles, and a causal tile ends
//     where its last position does.
//   * The work is the list of 128-token tiles of all (sequence, block of
//     positions, KV head) items; every CTA (one per SM) takes an equal, contiguous
//     share of it, so causal triangles, ragged lengths and few long items fill the
//     SMs alike. An item that lies in several CTAs is joined by the last of them,
//     per 32 rows, in the order of the list.
//   * Up to 128 rows (one query tile per item): a CTA takes two shares of the list, one
//     for each of its softmax warpgroups, whose tiles come in turn. (16 sequences of
//     up to 16384 tokens, 8 KV heads, 64 rows, head size 64 / 128: 155 / 184 us; one share
//     with one warpgroup 192 / 209; the shares' keys and values in plain order, so that
//     one share's keys wait for the other's products: 193 / 248.)
//   * Warps 0-3 and 4-7: softmax of one query tile each, a row per thread; 8: TMA
//     producer; 9 and 14: tcgen05 issuers, one per query tile; 10-13: converters.
//   * Scores are computed for 64 tokens at a time, in two sets of TMEM columns per
//     query tile, and the weights replace their scores there. While a softmax warpgroup
//     works on one half of a tile, the tensor cores finish the other half's product and
//     then bring its next scores (the order of products with different accumulators is
//     not guaranteed, so the issuer waits for the first).
//
// Measured: 2011 queries of 32 heads (8 KV heads) of 128 behind 16000 cached tokens (0.49
// TFLOP) 546 to 575 us, 0.86 to 0.90 PFLOP/s, 0.52 to 0.55 of the rate of a plain bf16 product. The
// tensor pipe is busy 47 % of an SM's time, the exponentials' unit 48 %, issue slots 53 %:
// a softmax warp waits for its own chain of loads, maxima, exponentials and stores.
// Whole 128-token score tiles took 660 us; part of the exponentials as polynomials gave
// nothing. 8 prompts of 223 tokens, 20 heads of 64:
// 22 us (two tiles of work per SM; launch, set-up and join are most of it).
//
// The softmax is that of the few-rows kernel: running maximum of
// log2(e) * scale * q.k + log2(value scale), raised when it is passed by 2^8, and
// weights 2^7 larger than relative to it.
//
// Every mbarrier wait is bounded; one that runs out records WBK_ERR_DEVICE_TIMEOUT,
// raises the CTA's abort flag and every role leaves its loop; copies and products
// in flight are waited for (with a limit) before TMEM is freed. No warp waits
// at a block-wide barrier in between.
#include <algorithm>
#include <mutex>
#include <vector>

#include "wbk_kv8.cuh"
#include "wbk_sm100.cuh"

namespace wbk {
namespace {

constexpr int kTile = 128;  // tokens per tile, and rows of a query tile
constexpr int kTileLog2 = 7;
constexpr int kGroups = kTile / 16;
constexpr int kHalf = kTile / 2;      // tokens of one score product
constexpr int kThreads = 480;
constexpr int kConvThreads = 128;
constexpr int kConvWarp = 10;  // the first of them
constexpr int kStages = 2;       // converted tiles of keys, and of values
// Slots of per-tile factors. The producer writes a tile's factors before it asks for its codes, and nothing tells it that
// a slot is free: there are more than it can be ahead of the softmax. With R units in the ring of codes:
//   * One share. At tile i the values of tile i - 1 have been asked for, so those of i - 1 - R / 2 have been converted, so the
//     product that had their stage, of tile i - 1 - R / 2 - kStages, is done, and the softmax of that tile.
//   * Two shares, each with half of the slots and one stage, values one tile behind keys. At tile i of a share
//     its values of tile i - 2 have been asked for. The other share's codes lie in between, so those of i - 3 have been
//     converted, and the product of i - 4 is done: tiles i - 3 to i may be in use, four slots. A share whose
//     neighbour has ended would need one more from its second lone tile on, if that is tile 4 or later. There is none such: where
//     both have tiles they differ by one at most (shares of one list), and where one has none the list is short,
//     total / 2 shares of 2 or 3 tiles.
constexpr int kFactors = 8;
constexpr int kBlockBytes = kTile * 128;  // 64 channels of a 16-bit tile
constexpr uint32_t kTmemCols = 512;
constexpr float kRaise = 8.0f;   // log2 units
constexpr uint64_t kDrainNs = 100000000ull;  // least limit of the waits for what is in flight at the end
constexpr int kTickets = 8;      // per CTA: one for each 32 rows
static_assert(kTickets <= kKv8TicketsPerSm, "workspace layout");
enum : uint32_t {
  PSITE_PRODUCER = 51,
  PSITE_CONVERT = 52,
  PSITE_MMA = 53,
  PSITE_SOFTMAX = 54,
  PSITE_DRAIN = 55,
};

template <int kD>
struct Cfg {
  static constexpr int kRawUnits = kD == 64 ? 4 : 2;  // tiles of codes: keys and values in turn
  static constexpr int kRawBytes = kTile * kD;
  static constexpr int kBlocks = kD / 64;
  static constexpr int kTileBytes = kBlocks * kBlockBytes;
  static_assert(kFactors > kRawUnits / 2 + kStages && kFactors / 2 > 3 && kRawUnits <= 4, "a slot would be overwritten in use");
};
// TMEM columns: scores, then weights, of half h of query tile t; sums of query tile t.
__device__ __forceinline__ uint32_t s_col(int t, int h) { return static_cast<uint32_t>(t * 128 + h * 64); }
__device__ __forceinline__ uint32_t o_col(int t) { return static_cast<uint32_t>(256 + t * 128); }

template <int kD>
struct PromptSmem {
  uint8_t q[2][Cfg<kD>::kTileBytes];  // 1024-byte aligned
  uint8_t k[kStages][Cfg<kD>::kTileBytes];
  uint8_t v[kStages][Cfg<kD>::kTileBytes];
  uint8_t raw[Cfg<kD>::kRawUnits][Cfg<kD>::kRawBytes];
  float4 factor[kFactors][kGroups];  // of 16 tokens: key factor, log2 of the value scale, its inverse (0: not there)
  int limit[kFactors];               // tokens of the tile that the sequence has
  uint32_t holes[kFactors];          // groups below the limit whose page is outside the pool
  uint64_t q_full[2], q_empty[2], raw_full[Cfg<kD>::kRawUnits], raw_empty[Cfg<kD>::kRawUnits];
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], factor_full[kFactors];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], o_free[2], drain[2];  // [query tile][half]
  uint32_t tmem_base;
  int abort_flag;
};

struct PromptParams {
  Kv8Attention a;
  int tile_pos;     // query positions per 128-row tile: 128 / group
  int tiles_q;      // query tiles per item, 1 or 2
  int pos_blocks;   // items per sequence and KV head
  uint32_t idesc_s, idesc_o;
  uint32_t* tickets;
  float* parts;
  uint64_t timeout_ns;
};

// Partial result of an item: sums as [head_dim / 4][256 rows] float4, maxima [256], totals [256].
__host__ __device__ constexpr int64_t part_floats(int d) { return 256 * static_cast<int64_t>(d) + 512; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ void tma_load_5d(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int y, int z, int u,
                                            int w) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(u), "r"(w)
      : "memory");
}

// D[tmem] (+)= A[smem] . B[smem] and A[tmem] . B[smem], 16-bit operands. Issued by one
// elected lane of a converged warp from values that the compiler knows to be the same in
// all its lanes: issued by a lone thread, each product costs about 148 clocks of moves
// into uniform registers, whatever its size; so issued, 128 x 128 x 16 takes its 64.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
// A value that is the same in all lanes, in a form that the compiler knows it to be.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(~0u, x, 0); }

// The first 16 of r.
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Descriptor of the value tile as the B operand (N = channels contiguous): 128-byte rows of 64 channels per token,
// 8-token swizzle atoms 1024 bytes apart, 64-channel blocks kBlockBytes apart.
__device__ __forceinline__ uint64_t value_desc(const void* p) {
  const uint32_t addr = smem_u32(p);
  uint64_t d = static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(kBlockBytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// A wait of a whole warp with one result for all lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t timeout_ns,
                                          uint32_t site) {
  return __all_sync(~0u, mbar_wait(bar, parity, abort_flag, timeout_ns, site));
}

// One item of the work list: query positions pos0 .. of sequence b, KV head h.
struct Item {
  int b, pb, h;
  int len, n;  // tokens that its last row sees, real query positions
  int tiles;   // at least 1
};

__device__ __forceinline__ int tiles_of(const PromptParams& p, int unit, int& len, int& n) {
  const int b = unit / p.pos_blocks, pb = unit - b * p.pos_blocks;
  const int per = p.tile_pos * p.tiles_q;
  len = kv8_len(p.a.lens, b, p.a.c);
  n = p.a.q_lens != nullptr ? min(max(p.a.q_lens[b], 0), p.a.queries) : p.a.queries;
  if (pb * per >= n) len = 0;
  else if (p.a.causal) len = max(len - n + min(n, (pb + 1) * per), 0);
  return max((len + kTile - 1) >> kTileLog2, 1);
}

__device__ __forceinline__ int64_t total_tiles(const PromptParams& p) {
  int64_t sum = 0;
  int len, n;
  for (int u = threadIdx.x & 31; u < p.a.batch * p.pos_blocks; u += 32) sum += tiles_of(p, u, len, n);
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  return sum * p.a.c.kv_heads;
}

// The item and tile at place x of the list, by a converged warp.
__device__ __forceinline__ Item locate(const PromptParams& p, int64_t x, int& tile) {
  const int lane = threadIdx.x & 31, units = p.a.batch * p.pos_blocks;
  const int64_t heads = p.a.c.kv_heads;
  Item it{};
  for (int u0 = 0;; u0 += 32) {
    int len = 0, n = 0;
    const int t = u0 + lane < units ? tiles_of(p, u0 + lane, len, n) : 0;
    int64_t upto = t;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += y;
    }
    const uint32_t past = __ballot_sync(~0u, upto * heads > x);
    if (past == 0 && u0 + 32 < units) {
      x -= __shfl_sync(~0u, upto, 31) * heads;
      continue;
    }
    const int src = past != 0 ? __ffs(past) - 1 : 31;
    x -= __shfl_sync(~0u, upto - t, src) * heads;
    it.b = (u0 + src) / p.pos_blocks;
    it.pb = (u0 + src) - it.b * p.pos_blocks;
    it.len = __shfl_sync(~0u, len, src);
    it.n = __shfl_sync(~0u, n, src);
    it.tiles = __shfl_sync(~0u, t, src);
    it.h = static_cast<int>(x / it.tiles);
    tile = static_cast<int>(x - static_cast<int64_t>(it.h) * it.tiles);
    return it;
  }
}

__device__ __forceinline__ void next_item(const PromptParams& p, Item& it) {
  if (++it.h < p.a.c.kv_heads) return;
  it.h = 0;
  const int unit = it.b * p.pos_blocks + it.pb + 1;
  it.b = unit / p.pos_blocks;
  it.pb = unit - it.b * p.pos_blocks;
  if (it.b < p.a.batch) it.tiles = tiles_of(p, unit, it.len, it.n);
}

// A lane's page of 32 consecutive pages, with its scales.
struct PageLane {
  int64_t page;
  float ks, vs;
};
__device__ __forceinline__ PageLane fetch_page(const PromptParams& p, const Item& it, int blk) {
  PageLane r{-1, 0.0f, 1.0f};
  if ((static_cast<int64_t>(blk) << p.a.c.block_log2) < it.len) r.page = kv8_page(p.a.c, it.b, blk);
  if (r.page >= 0) {
    const int64_t ph = r.page * p.a.c.kv_heads + it.h;
    r.ks = p.a.k_scale[ph];
    r.vs = p.a.v_scale[ph];
  }
  return r;
}

// 16 codes -> 16 values of the 16-bit type, in order.
template <int kFmt, bool kBf16>
__device__ __forceinline__ void convert16(const uint4& u, uint4& a, uint4& b) {
  uint32_t w[8];
  const uint32_t in[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint2 h = kv8_half4<kFmt>(in[i]);
    w[2 * i] = h.x;
    w[2 * i + 1] = h.y;
  }
  if constexpr (kBf16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      w[i] = float2_to_pair<WBK_DT_BF16>(f.x, f.y);  // exact: at most 4 significant bits
    }
  }
  a = make_uint4(w[0], w[1], w[2], w[3]);
  b = make_uint4(w[4], w[5], w[6], w[7]);
}

// One arrival for a warp, after what all its lanes did.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// One tile of codes [128][kD] -> the 16-bit swizzled tile; `raw_empty` is given back as soon as the codes are read.
// `clear`: tokens at or after `limit`, or in groups that are not there, become 0.
template <int kFmt, int kD, bool kBf16>
__device__ __forceinline__ void convert_tile(const uint8_t* raw, uint8_t* dst, uint64_t* raw_empty, bool clear,
                                             const float4* factor, int limit) {
  const int tid = static_cast<int>(threadIdx.x) - kConvWarp * 32;
  constexpr int kPer = kD / 16;                     // 16-byte pieces per token, and per thread
  constexpr int kStep = kConvThreads / kPer;        // tokens from one piece of a thread to its next
  const int token = tid / kPer, piece = tid % kPer;
  uint4 u[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) u[i] = *reinterpret_cast<const uint4*>(raw + (tid + i * kConvThreads) * 16);
  if (clear) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (token + i * kStep >= limit || factor[(token + i * kStep) >> 4].z == 0.0f) u[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  warp_arrive(raw_empty);
  // 8 lanes store to 8 different 16-byte columns: those of the second 64 channels start with the odd one
  const int j = (piece & 3) * 2, sw = token & 7;  // kStep is a multiple of 8
  const bool odd = piece >= 4;
  uint8_t* row = dst + (piece >> 2) * kBlockBytes + token * 128;
  uint8_t* one = row + (((j + odd) ^ sw) << 4);
  uint8_t* two = row + (((j + !odd) ^ sw) << 4);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    uint4 a, b;
    convert16<kFmt, kBf16>(u[i], a, b);
    *reinterpret_cast<uint4*>(one + i * kStep * 128) = odd ? b : a;
    *reinterpret_cast<uint4*>(two + i * kStep * 128) = odd ? a : b;
  }
}

// Scores of 32 columns that are not to count: at or after `lim`, or in one of the two groups that `holes` names.
__device__ __forceinline__ void hide(uint32_t (&y)[32], int lim, uint32_t holes) {
#pragma unroll
  for (int k = 0; k < 32; ++k)
    if (k >= lim || (holes >> (k >> 4) & 1u)) y[k] = 0xFF800000u;  // -inf
}
// The largest x + log2 vs of 32 columns.
__device__ __forceinline__ float largest(const uint32_t (&y)[32], const float4* factor) {
  float mx = -INFINITY;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float* v = reinterpret_cast<const float*>(y) + 16 * h;
    const float a = max3(v[0], v[1], v[2]), b = max3(v[3], v[4], v[5]), c = max3(v[6], v[7], v[8]);
    const float d = max3(v[9], v[10], v[11]), e = max3(v[12], v[13], v[14]);
    const float4 f = factor[h];
    mx = fmaxf(mx, fmaf(fmaxf(max3(a, b, c), max3(d, e, v[15])), f.x, f.y));
  }
  return mx;
}
// The weights of 32 columns relative to 2^ref, as fp16 pairs in y[0 .. 15]; returns their sum over the value scales, of
// the fp32 weights (as fp16 those of a page of small value scale may be 0).
__device__ __forceinline__ float weights(uint32_t (&y)[32], const float4* factor, float ref) {
  float sum = 0.0f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float4 f = factor[h];
    const float2 mul = make_float2(f.x, f.x), off = make_float2(f.y - ref, f.y - ref);
    float2 rs = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float2 x = f2_fma(make_float2(__uint_as_float(y[16 * h + 2 * k]), __uint_as_float(y[16 * h + 2 * k + 1])), mul, off);
      const float2 w = make_float2(ex2(x.x), ex2(x.y));
      y[8 * h + k] = pack_half2(w.x, w.y);
      rs = f2_add(rs, w);
    }
    sum = fmaf(rs.x + rs.y, f.z, sum);
  }
  return sum;
}

template <int kFmt, int kD, bool kBf16, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
kv8_prompt_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                  const __grid_constant__ CUtensorMap tmap_v, const PromptParams p) {
  using C = Cfg<kD>;
  extern __shared__ uint8_t smem_raw[];
  PromptSmem<kD>& s = *reinterpret_cast<PromptSmem<kD>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort_flag;
  const int nq = kSplit ? 2 : p.tiles_q;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s.q_full[t], 1);
      mbar_init(&s.q_empty[t], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&s.s_full[t][h], 1);
        mbar_init(&s.p_full[t][h], 4);  // one arrival per warp
        mbar_init(&s.pv_done[t][h], 1);
      }
      mbar_init(&s.o_free[t], 4);
      mbar_init(&s.drain[t], 1);
    }
    for (int i = 0; i < C::kRawUnits; ++i) {
      mbar_init(&s.raw_full[i], 1);
      mbar_init(&s.raw_empty[i], kConvThreads / 32);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.k_full[i], kConvThreads / 32);
      mbar_init(&s.k_empty[i], kSplit ? 1u : static_cast<uint32_t>(nq));  // one per issuer that uses it
      mbar_init(&s.v_full[i], kConvThreads / 32);
      mbar_init(&s.v_empty[i], kSplit ? 1u : static_cast<uint32_t>(nq));
    }
    for (int i = 0; i < kFactors; ++i) mbar_init(&s.factor_full[i], 1);
    s.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  if (warp == 9) {
    tmem_alloc(&s.tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  griddep_launch_dependents();
  griddep_wait();  // nothing above reads or writes memory that the kernel before may still use

  // this CTA's share of the list, or where the query tiles split it (kSplit) that of each, as of twice as many CTAs
  const int64_t total = total_tiles(p);
  const int owners = static_cast<int>(gridDim.x) * (kSplit ? 2 : 1);
  const int64_t active = max(min(static_cast<int64_t>(owners), total / 2), static_cast<int64_t>(1));
  auto owner_of = [&](int t) { return static_cast<int>(blockIdx.x) + (kSplit ? t * static_cast<int>(gridDim.x) : 0); };
  auto share = [&](int owner) { return owner < active ? owner * total / active : total; };  // its start
  // Place of a query tile's i-th tile in the rings: its own count where they share all tiles, else in turn.
  auto slot_of = [](uint32_t i, int t) { return kSplit ? 2 * i + static_cast<uint32_t>(t) : i; };

  if (warp == 8 || warp == 9 || warp == 14) {
    if (warp == 8) {
      // -------------------------------------------------------- producer
      const int sub = min(p.a.c.block_log2, kTileLog2);  // log2 of tokens per TMA box
      const int cover = 32 << p.a.c.block_log2;          // tokens that 32 pages hold
      constexpr int kStreams = kSplit ? 2 : 1;  // kSplit: the two shares' tiles in turn
      uint32_t unit = 0, tiles[kStreams] = {}, q_loads[2] = {0, 0};
      bool ok = true;
      Item its[kStreams];
      int64_t xs[kStreams], ends[kStreams];
      int ts[kStreams], t1s[kStreams], blk0s[kStreams], tes[kStreams];
      PageLane held[kStreams];
#pragma unroll
      for (int u = 0; u < kStreams; ++u) {
        xs[u] = share(owner_of(u)), ends[u] = share(owner_of(u) + 1);
        if (owner_of(u) >= active) ends[u] = xs[u];
        ts[u] = t1s[u] = 0;
        if (xs[u] < ends[u]) {
          its[u] = locate(p, xs[u], ts[u]);
          t1s[u] = static_cast<int>(min(static_cast<int64_t>(its[u].tiles), ts[u] + (ends[u] - xs[u])));
          tes[u] = ts[u];
        }
      }
      bool fresh[kStreams] = {};  // a segment's first tile is done: its queries are loaded
      // kSplit: values go one tile behind, so that no share's next keys wait for the other's products
      bool vload[kStreams] = {};
      uint32_t vbytes[kStreams] = {};
      int vy[kStreams], vpage[kStreams];
      auto issue = [&](const CUtensorMap* map, bool load, uint32_t bytes, int y, int page) {
        const int r = static_cast<int>(unit % C::kRawUnits);
        ok = warp_wait(&s.raw_empty[r], ((unit / C::kRawUnits) & 1u) ^ 1u, abort_flag, p.timeout_ns, PSITE_PRODUCER);
        if (!ok) return;
        if (lane == 0) mbar_arrive_expect_tx(&s.raw_full[r], bytes);
        __syncwarp();
        if (load) tma_load_3d(map, &s.raw_full[r], s.raw[r] + lane * 16 * kD, 0, y, page);
        ++unit;
      };
      bool behind[kStreams] = {};  // kSplit: the last values are still to come
      while (ok && (xs[0] < ends[0] || xs[kStreams - 1] < ends[kStreams - 1] || behind[0] || behind[kStreams - 1])) {
#pragma unroll
        for (int u = 0; u < kStreams; ++u) {
          if (!ok) break;
          if (xs[u] >= ends[u]) {
            if (behind[u]) issue(&tmap_v, vload[u], vbytes[u], vy[u], vpage[u]);
            behind[u] = false;
            continue;
          }
          Item& it = its[u];
          PageLane& pages = held[u];
          const int t = ts[u];
          if (t == tes[u]) {
            blk0s[u] = (t * kTile) >> p.a.c.block_log2;
            pages = fetch_page(p, it, blk0s[u] + lane);
            tes[u] = ((blk0s[u] << p.a.c.block_log2) + cover) >> kTileLog2;
          }
          // ---- the tile's factors, before its codes
          const int slot = static_cast<int>(slot_of(tiles[u], u) % kFactors);
          const int pos = t * kTile + (lane & (kGroups - 1)) * 16;
          const int from = ((pos >> p.a.c.block_log2) - blk0s[u]) & 31;
          const int64_t page = __shfl_sync(~0u, pages.page, from);
          const float ks = __shfl_sync(~0u, pages.ks, from), vs = __shfl_sync(~0u, pages.vs, from);
          const bool there = page >= 0 && pos < it.len;
          // the factor stays above 0, so that a masked -inf stays -inf
          if (lane < kGroups)
            s.factor[slot][lane] = make_float4(fmaxf(ks * p.a.scale_log2, 1.17549435e-38f), kv8_log2(vs), there ? 1.0f / vs : 0.0f, 0.0f);
          const uint32_t holes = __ballot_sync(~0u, lane < kGroups && pos < it.len && !there);
          if (lane == 0) {
            s.limit[slot] = it.len - t * kTile;
            s.holes[slot] = holes;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.factor_full[slot]);
          // ---- keys, then values: one box per page, which the page's first group in the tile stands for
          const bool load = lane < kGroups && there && (lane & ((1 << (sub - 4)) - 1)) == 0;
          const uint32_t bytes = __popc(__ballot_sync(~0u, load)) * (static_cast<uint32_t>(kD) << sub);
          const int y = (it.h << p.a.c.block_log2) + (pos & (p.a.c.block - 1));
          if constexpr (kSplit) {
            issue(&tmap_k, load, bytes, y, static_cast<int>(page));
            if (ok && tiles[u] > 0) issue(&tmap_v, vload[u], vbytes[u], vy[u], vpage[u]);
            vload[u] = load, vbytes[u] = bytes, vy[u] = y, vpage[u] = static_cast<int>(page);
          } else {
#pragma unroll 1
            for (int kv = 0; kv < 2 && ok; ++kv) issue(kv == 0 ? &tmap_k : &tmap_v, load, bytes, y, static_cast<int>(page));
          }
          if (!ok) break;
          ++tiles[u];
          behind[u] = kSplit;
          // ---- queries, behind the item's first codes
          if (!fresh[u]) {
            fresh[u] = true;
            for (int qt = kSplit ? u : 0; qt < (kSplit ? u + 1 : nq); ++qt) {
              ok = warp_wait(&s.q_empty[qt], (q_loads[qt] & 1u) ^ 1u, abort_flag, p.timeout_ns, PSITE_PRODUCER);
              if (!ok) break;
              if (lane == 0) {
                mbar_arrive_expect_tx(&s.q_full[qt], static_cast<uint32_t>(p.tile_pos * p.a.group * kD * 2));
                for (int i = 0; i < C::kBlocks; ++i)
                  tma_load_5d(&tmap_q, &s.q_full[qt], s.q[qt] + i * kBlockBytes, i * 64, 0,
                              (kSplit ? it.pb : it.pb * nq + qt) * p.tile_pos, it.h, it.b);
              }
              __syncwarp();
              ++q_loads[qt];
            }
          }
          ++xs[u];
          if (++ts[u] == t1s[u] && xs[u] < ends[u]) {
            next_item(p, it);
            ts[u] = tes[u] = 0;
            t1s[u] = static_cast<int>(min(static_cast<int64_t>(it.tiles), ends[u] - xs[u]));
            fresh[u] = false;
          }
        }
      }
      // The CTA ends only when what was issued has landed and been used: every unit and query tile given back.
      if (lane == 0) {
        int dummy = 0;
        const uint64_t limit = max(p.timeout_ns, kDrainNs);
        for (uint32_t i = unit > C::kRawUnits ? unit - C::kRawUnits : 0; i < unit; ++i)
          mbar_wait(&s.raw_full[i % C::kRawUnits], (i / C::kRawUnits) & 1u, &dummy, limit, PSITE_DRAIN);
        for (int qt = 0; qt < nq; ++qt)
          if (q_loads[qt] > 0) mbar_wait(&s.q_full[qt], (q_loads[qt] - 1) & 1u, &dummy, limit, PSITE_DRAIN);
        if (ok) {  // and no commit to these barriers is still on its way
          for (int qt = 0; qt < nq; ++qt)
            if (q_loads[qt] > 0) mbar_wait(&s.q_empty[qt], (q_loads[qt] - 1) & 1u, abort_flag, limit, PSITE_DRAIN);
#pragma unroll
          for (int u = 0; u < kStreams; ++u)
            for (uint32_t i = tiles[u] > kStages / kStreams ? tiles[u] - kStages / kStreams : 0; i < tiles[u]; ++i) {
              const uint32_t g = slot_of(i, u);
              mbar_wait(&s.k_empty[g % kStages], (g / kStages) & 1u, abort_flag, limit, PSITE_DRAIN);
              mbar_wait(&s.v_empty[g % kStages], (g / kStages) & 1u, abort_flag, limit, PSITE_DRAIN);
            }
        }
      }
    } else {
      // ------------------------------------- MMA issuers: warp 9 query tile 0, warp 14 query tile 1
      const int t = warp == 9 ? 0 : 1;
      uint32_t g = 0, ui = 0;
      bool ok = t < nq && owner_of(t) < active;
      int tile = 0;
      int64_t x = share(owner_of(t));
      const int64_t x1 = share(owner_of(t) + 1);
      Item it{};
      if (ok) it = locate(p, x, tile);
      const uint32_t tm = static_cast<uint32_t>(uniform(static_cast<int>(tmem)));
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok) ok = warp_wait(bar, parity, abort_flag, p.timeout_ns, PSITE_MMA);
        return ok;
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) umma_commit(bar);
        __syncwarp();
      };
      const int qt = uniform(t);
      auto issue_s = [&](int h, uint32_t gj) {
        const int st = uniform(static_cast<int>(slot_of(gj, t) % kStages)), qh = uniform(h);
        if (elect_one()) {
          const uint32_t d = tm + s_col(qt, qh);
#pragma unroll
          for (int i = 0; i < C::kBlocks; ++i) {
            const uint64_t qd = make_sw128_desc(s.q[qt] + i * kBlockBytes);
            const uint64_t kd = make_sw128_desc(s.k[st] + i * kBlockBytes + qh * (kHalf * 128));
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) mma_ss(d, qd + kk * 2, kd + kk * 2, p.idesc_s, i > 0 || kk > 0 ? 1u : 0u);
          }
          umma_commit(&s.s_full[qt][qh]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int h, uint32_t gj, bool first) {
        const int st = uniform(static_cast<int>(slot_of(gj, t) % kStages)), qh = uniform(h);
        const uint32_t onto = static_cast<uint32_t>(uniform(first ? 0 : 1));
        if (elect_one()) {
          const uint64_t vd = value_desc(s.v[st] + qh * (kHalf * 128));
          const uint32_t d = tm + o_col(qt), a = tm + s_col(qt, qh);
#pragma unroll
          for (int kk = 0; kk < kHalf / 16; ++kk)
            mma_ts(d, a + kk * 8, vd + kk * (2048 >> 4), p.idesc_o, kk == 0 ? onto : 1u);
          umma_commit(&s.pv_done[qt][qh]);
        }
        __syncwarp();
      };
      while (x < x1 && ok) {
        const int t1 = static_cast<int>(min(static_cast<int64_t>(it.tiles), tile + (x1 - x)));
        const int n = t1 - tile;
        wait(&s.q_full[t], ui & 1u);
        // Half by half: the output product of tile j, then the scores of tile j + 1, which replace the weights that it
        // read. Tile -1 has no product: the item's first scores follow the item before.
#pragma unroll 1
        for (int j = -1; j < n && ok; ++j) {
          const uint32_t gj = g + static_cast<uint32_t>(j), gn = gj + 1;
          const uint32_t sj = slot_of(gj, t), sn = slot_of(gn, t);
          if (j >= 0) wait(&s.v_full[sj % kStages], (sj / kStages) & 1u);
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            if (j >= 0) {
              wait(&s.p_full[t][h], gj & 1u);
              if (j == 0 && h == 0) wait(&s.o_free[t], (ui & 1u) ^ 1u);
              if (!ok) break;
              tc_fence_after();
              issue_pv(h, gj, j == 0 && h == 0);
            }
            if (j + 1 < n) {
              if (h == 0) wait(&s.k_full[sn % kStages], (sn / kStages) & 1u);
              if (gn > 0) wait(&s.pv_done[t][h], gj & 1u);
              if (!ok) break;
              tc_fence_after();
              issue_s(h, gn);
            }
          }
          if (!ok) break;
          if (j >= 0) commit(&s.v_empty[sj % kStages]);
          if (j + 1 < n) {
            commit(&s.k_empty[sn % kStages]);
            if (j + 2 == n) commit(&s.q_empty[t]);  // the item's last scores are issued
          }
        }
        g += static_cast<uint32_t>(n);
        ++ui;
        x += n;
        tile = 0;
        if (x < x1) next_item(p, it);
      }
      // TMEM and the barriers are in use until every product issued has finished.
      commit(&s.drain[t]);
      int dummy = 0;
      mbar_wait(&s.drain[t], 0, &dummy, max(p.timeout_ns, kDrainNs), PSITE_DRAIN);
    }
  } else if (warp >= 10) {
    // ---------------------------------------------------------- converters
    uint32_t unit = 0;
    bool ok = true;
    int64_t mine[2] = {0, 0};
    for (int u = 0; u < (kSplit ? 2 : 1); ++u)
      if (owner_of(u) < active) mine[u] = share(owner_of(u) + 1) - share(owner_of(u));
    // kSplit: of each share in turn the next keys, then values; otherwise keys and values in turn
    const int64_t rounds = kSplit ? 2 * (max(mine[0], mine[1]) + 1) : mine[0];
    for (int64_t i = 0; i < rounds && ok; ++i) {
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        const int64_t own = kSplit ? (i >> 1) - kv : i;  // tile of the share
        if (kSplit && (own < 0 || own >= mine[i & 1])) continue;
        const uint32_t g = kSplit ? slot_of(static_cast<uint32_t>(own), static_cast<int>(i & 1)) : static_cast<uint32_t>(i);
        const int st = static_cast<int>(g % kStages), slot = static_cast<int>(g % kFactors);
        const uint32_t empty = ((g / kStages) & 1u) ^ 1u;
        if (kSplit || kv == 0) ok = warp_wait(&s.factor_full[slot], (g / kFactors) & 1u, abort_flag, p.timeout_ns, PSITE_CONVERT);
        const int u = static_cast<int>(unit % C::kRawUnits);
        if (ok) ok = warp_wait(&s.raw_full[u], (unit / C::kRawUnits) & 1u, abort_flag, p.timeout_ns, PSITE_CONVERT);
        if (ok) ok = warp_wait(kv == 0 ? &s.k_empty[st] : &s.v_empty[st], empty, abort_flag, p.timeout_ns, PSITE_CONVERT);
        if (!ok) break;
        const bool clear = kv == 1 && (s.limit[slot] < kTile || s.holes[slot] != 0);
        uint8_t* to = kv == 0 ? s.k[st] : s.v[st];
        if (kBf16 && kv == 0) convert_tile<kFmt, kD, kBf16>(s.raw[u], to, &s.raw_empty[u], false, s.factor[slot], 0);
        else convert_tile<kFmt, kD, false>(s.raw[u], to, &s.raw_empty[u], clear, s.factor[slot], s.limit[slot]);
        fence_async_smem();
        warp_arrive(kv == 0 ? &s.k_full[st] : &s.v_full[st]);
        ++unit;
      }
    }
  } else {
    // ------------------------------------------------------------- softmax
    const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    uint32_t g = 0;
    bool ok = t < nq && owner_of(t) < active;
    int tile = 0;
    int64_t x = share(owner_of(t));
    const int64_t x1 = share(owner_of(t) + 1);
    Item it{};
    if (ok) it = locate(p, x, tile);
    while (x < x1 && ok) {
      const int t1 = static_cast<int>(min(static_cast<int64_t>(it.tiles), tile + (x1 - x)));
      const int i = (kSplit ? it.pb : it.pb * nq + t) * p.tile_pos + r / p.a.group, gi = r % p.a.group;  // query position and head
      const bool real = r < p.tile_pos * p.a.group && i < p.a.queries;
      const int seq = kv8_len(p.a.lens, it.b, p.a.c);
      const int vis = i >= it.n ? 0 : p.a.causal ? max(seq - it.n + i + 1, 0) : seq;
      float m = -INFINITY, l = 0.0f;
      for (int hh = 2 * tile; hh < 2 * t1; ++hh) {  // 64 tokens at a time
        const uint32_t place = slot_of(g, t);
        const int h = hh & 1, slot = static_cast<int>(place % kFactors);
        if ((h == 0 && !warp_wait(&s.factor_full[slot], (place / kFactors) & 1u, abort_flag, p.timeout_ns, PSITE_SOFTMAX)) ||
            !warp_wait(&s.s_full[t][h], g & 1u, abort_flag, p.timeout_ns, PSITE_SOFTMAX)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sa = lane_addr + s_col(t, h);
        uint32_t ya[32], yb[32];
        tmem_ld_32x32b_x32(sa, ya);
        tmem_ld_32x32b_x32(sa + 32, yb);
        const uint32_t holes = s.holes[slot] >> (4 * h);
        const int lim = vis - hh * kHalf;
        const bool edge = holes != 0 || __any_sync(~0u, lim < kHalf);
        const float4* fac = s.factor[slot] + 4 * h;
        tmem_ld_wait(ya);
        tmem_ld_wait(yb);
        if (edge) {
          hide(ya, lim, holes);
          hide(yb, lim - 32, holes >> 2);
        }
        // ---- the row's largest x + log2 vs: factors are positive, so that of a group is that of its largest score
        const float mx = fmaxf(largest(ya, fac), largest(yb, fac + 2));
        float alpha = 1.0f;
        if (mx > m + kRaise) {
          alpha = ex2(m - mx);
          m = mx;
        }
        l *= alpha;
        const float ref = m == -INFINITY ? 0.0f : m - kKv8Lift;
        // ---- weights, in place of their scores
        l += weights(ya, fac, ref);
        tmem_st_x16(sa, ya);
        l += weights(yb, fac + 2, ref);
        tmem_st_x16(sa + 16, yb);
        if (hh > 2 * tile && __any_sync(~0u, alpha != 1.0f)) {
          // the sums are free once the previous half's product is done
          if (!warp_wait(&s.pv_done[t][h ^ 1], (h == 1 ? g : g - 1) & 1u, abort_flag, p.timeout_ns, PSITE_SOFTMAX)) {
            tmem_st_wait();
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < kD / 32; ++c) {
            const uint32_t oa = lane_addr + o_col(t) + c * 32;
            tmem_ld_32x32b_x32(oa, yb);
            tmem_ld_wait(yb);
#pragma unroll
            for (int k = 0; k < 32; ++k) yb[k] = __float_as_uint(__uint_as_float(yb[k]) * alpha);
            tmem_st_x32(oa, yb);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        warp_arrive(&s.p_full[t][h]);
        if (h == 1) ++g;
      }
      if (!ok) break;
      // ---- the item's rows: output, or this CTA's part of it
      if (!warp_wait(&s.pv_done[t][1], (g - 1) & 1u, abort_flag, p.timeout_ns, PSITE_SOFTMAX)) break;
      tc_fence_after();
      const bool whole = tile == 0 && t1 == it.tiles;
      const int row = t * kTile + r;
      uint16_t* dst = static_cast<uint16_t*>(p.a.out) + it.b * p.a.o_sb + (static_cast<int64_t>(it.h) * p.a.group + gi) * p.a.o_sh +
                      i * p.a.o_ss;
      float* part = p.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (tile == 0 ? 1 : 0)) * part_floats(kD);
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
      for (int c = 0; c < kD / 32; ++c) {
        uint32_t orr[32];
        tmem_ld_32x32b_x32(lane_addr + o_col(t) + c * 32, orr);
        tmem_ld_wait(orr);
        if (c == kD / 32 - 1) {  // read to the end: the next item's first product may overwrite it
          tc_fence_before();
          warp_arrive(&s.o_free[t]);
        }
        const float* o = reinterpret_cast<const float*>(orr);
        if (!whole) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            reinterpret_cast<float4*>(part)[(c * 8 + k) * 256 + row] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        } else if (real) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = float2_to_pair<kBf16 ? WBK_DT_BF16 : WBK_DT_F16>(o[8 * k + 2 * e] * inv, o[8 * k + 2 * e + 1] * inv);
            reinterpret_cast<uint4*>(dst + c * 32)[k] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (!whole) {
        part[256 * kD + row] = m;
        part[256 * kD + 256 + row] = l;
        // the shares that this item lies in; the last of them to finish these 32 rows joins them
        const int64_t begin = x - tile, end = begin + it.tiles;
        const int first = static_cast<int>(((begin + 1) * active - 1) / total), last = static_cast<int>((end * active - 1) / total);
        __threadfence();
        __syncwarp();
        uint32_t before = 0;
        if (lane == 0) {
          uint32_t* ticket = &p.tickets[kSplit ? first * 4 + quarter : first * kTickets + warp];
          before = atomicAdd(ticket, 1u);
          if (before == static_cast<uint32_t>(last - first)) *ticket = 0u;
        }
        if (__shfl_sync(~0u, before, 0) == static_cast<uint32_t>(last - first)) {
          __threadfence();
          const int count = last - first + 1;
          // the part of the k-th share; in units of float4, a row's place in it is that of this thread's row
          auto at = [&](int k) {
            const int owner = first + k, cta = kSplit && owner >= static_cast<int>(gridDim.x) ? owner - gridDim.x : owner;
            return p.parts + (static_cast<int64_t>(cta) * 2 + (k == 0 ? 1 : 0)) * part_floats(kD);
          };
          auto row_in = [&](int k) { return kSplit ? r + (first + k >= static_cast<int>(gridDim.x) ? kTile : 0) : row; };
          float top = -INFINITY, tot = 0.0f;
          for (int k = 0; k < count; ++k) top = fmaxf(top, __ldcg(at(k) + 256 * kD + row_in(k)));
          for (int k = 0; k < count; ++k) {
            const float mk = __ldcg(at(k) + 256 * kD + row_in(k));
            tot = fmaf(mk == -INFINITY ? 0.0f : ex2(mk - top), __ldcg(at(k) + 256 * kD + 256 + row_in(k)), tot);
          }
          const float invt = tot == 0.0f ? 0.0f : 1.0f / tot;
#pragma unroll 1
          for (int c = 0; c < kD / 32; ++c) {
            float o[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0.0f;
            for (int k = 0; k < count; ++k) {
              const float mk = __ldcg(at(k) + 256 * kD + row_in(k)), f = mk == -INFINITY ? 0.0f : ex2(mk - top);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 y = __ldcg(reinterpret_cast<const float4*>(at(k)) + (c * 8 + e) * 256 + row_in(k));
                o[4 * e] = fmaf(f, y.x, o[4 * e]), o[4 * e + 1] = fmaf(f, y.y, o[4 * e + 1]);
                o[4 * e + 2] = fmaf(f, y.z, o[4 * e + 2]), o[4 * e + 3] = fmaf(f, y.w, o[4 * e + 3]);
              }
            }
            if (real) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  w[e] = float2_to_pair<kBf16 ? WBK_DT_BF16 : WBK_DT_F16>(o[8 * k + 2 * e] * invt, o[8 * k + 2 * e + 1] * invt);
                reinterpret_cast<uint4*>(dst + c * 32)[k] = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
          }
        }
      }
      x += t1 - tile;
      tile = 0;
      if (x < x1) next_item(p, it);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Queries as a 5-D tensor (channel, head of the group, position, KV head, sequence); a box is 64 channels of one tile's
// rows, swizzled.
int make_tmap_queries(CUtensorMap* map, const Kv8Attention& a, int tile_pos) {
  auto encode = get_encode_fn();
  if (encode == nullptr) return fail(WBK_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
  const auto stride = [&](int64_t s, int64_t size) { return static_cast<cuuint64_t>(size > 1 ? s * 2 : 16); };
  const int64_t heads = a.c.kv_heads;
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.group),
                              static_cast<cuuint64_t>(a.queries), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(a.batch)};
  const cuuint64_t strides[4] = {stride(a.q_sh, a.group), stride(a.q_ss, a.queries), stride(a.q_sh * a.group, heads),
                                 stride(a.q_sb, a.batch)};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(tile_pos), 1, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode(map, a.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                            const_cast<void*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(WBK_ERR_CUDA, "cuTensorMapEncodeTiled (queries) failed (%d)", static_cast<int>(r));
  return WBK_OK;
}

// tcgen05 instruction descriptor, kind::f16: D fp32 (bit 4), A and B fp16 (0) or bf16 (1) at bits 7 and 10, B
// major-ness at bit 16 (1 = N contiguous), N >> 3 at bit 17, M >> 4 at bit 24.
constexpr uint32_t instruction(int n, bool bf16, bool b_n_major) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_n_major ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}

int prompt_sms() {
  const int n = sm_count();
  return n > 0 ? n : 148;
}

template <int kFmt, int kD, bool kBf16, bool kSplit>
int launch_prompt(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PromptParams& p, int grid,
                  cudaStream_t stream) {
  constexpr size_t smem = sizeof(PromptSmem<kD>) + 1024;
  static_assert(smem <= 232448, "shared memory budget");
  static std::mutex mu;
  static std::vector<char> configured;
  const int dev = current_device();
  if (dev < 0) return fail(WBK_ERR_CUDA, "no current CUDA device");
  {
    std::lock_guard<std::mutex> lock(mu);
    if (static_cast<int>(configured.size()) <= dev) configured.resize(dev + 1, 0);
    if (!configured[dev]) {
      if (int e = cuda_check(cudaFuncSetAttribute(kv8_prompt_kernel<kFmt, kD, kBf16, kSplit>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                  static_cast<int>(smem)),
                             "kv8 prompt smem attribute"))
        return e;
      configured[dev] = 1;
    }
  }
  return cuda_check(launch_after(kv8_prompt_kernel<kFmt, kD, kBf16, kSplit>, dim3(grid), kThreads, smem, stream, 1, tq, tk, tv, p),
                    "kv8 prompt launch");
}

template <int kFmt, int kD>
int dispatch_type(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PromptParams& p, int grid,
                  cudaStream_t stream) {
  if (p.tiles_q == 1)
    return p.a.bf16 ? launch_prompt<kFmt, kD, true, true>(tq, tk, tv, p, grid, stream)
                    : launch_prompt<kFmt, kD, false, true>(tq, tk, tv, p, grid, stream);
  return p.a.bf16 ? launch_prompt<kFmt, kD, true, false>(tq, tk, tv, p, grid, stream)
                  : launch_prompt<kFmt, kD, false, false>(tq, tk, tv, p, grid, stream);
}

}  // namespace

int64_t kv8_prompt_ws_bytes(int64_t head_dim) {
  return kv8_ticket_bytes() + static_cast<int64_t>(prompt_sms()) * 2 * part_floats(static_cast<int>(head_dim)) * 4;
}

int kv8_prompt_attention(const Kv8Attention& a, void* workspace, cudaStream_t stream) {
  PromptParams p{};
  p.a = a;
  p.tile_pos = kTile / a.group;
  p.tiles_q = a.queries > p.tile_pos ? 2 : 1;
  const int64_t per = static_cast<int64_t>(p.tile_pos) * p.tiles_q;
  p.pos_blocks = static_cast<int>((a.queries + per - 1) / per);
  p.idesc_s = instruction(kHalf, a.bf16, false);
  p.idesc_o = instruction(a.head_dim, false, true);
  p.tickets = static_cast<uint32_t*>(workspace);
  p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kv8_ticket_bytes());
  p.timeout_ns = wait_timeout_ns();
  CUtensorMap tq, tk, tv;
  if (int e = make_tmap_queries(&tq, a, p.tile_pos)) return e;
  if (int e = kv8_make_tmap(&tk, a.k_cache, a, kTile, false)) return e;
  if (int e = kv8_make_tmap(&tv, a.v_cache, a, kTile, false)) return e;
  const int64_t most = static_cast<int64_t>(a.batch) * p.pos_blocks * a.c.kv_heads *
                       ((static_cast<int64_t>(a.c.max_blocks) * a.c.block + kTile - 1) / kTile);
  const int grid = static_cast<int>(std::min<int64_t>(prompt_sms(), std::max<int64_t>(most / 2, 1)));
  if (a.fmt == WBK_FMT_E4M3)
    return a.head_dim == 64 ? dispatch_type<WBK_FMT_E4M3, 64>(tq, tk, tv, p, grid, stream)
                            : dispatch_type<WBK_FMT_E4M3, 128>(tq, tk, tv, p, grid, stream);
  return a.head_dim == 64 ? dispatch_type<WBK_FMT_E5M2, 64>(tq, tk, tv, p, grid, stream)
                          : dispatch_type<WBK_FMT_E5M2, 128>(tq, tk, tv, p, grid, stream);
}

int kv8_prompt_read_device_error(uint32_t* v, bool clear) {
  if (int e = cuda_check(cudaMemcpyFromSymbol(v, g_device_error, sizeof(*v)), "kv8 prompt device error read")) return e;
  if (clear) {
    const uint32_t zero = 0;
    if (int e = cuda_check(cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero)), "kv8 prompt device error clear")) return e;
  }
  return WBK_OK;
}

}  // namespace wbk
