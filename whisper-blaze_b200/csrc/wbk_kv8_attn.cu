// Attention over the 8-bit key/value cache for few query rows per KV head (a
// decoder's step: one or a few tokens).
//
// What bounds it: 2 * head_dim bytes of codes per token and KV head, each used by
// group * queries rows only, so HBM; nothing else may wait.
//
//   * The work is the list of 64-token tiles of all (sequence, KV head, block of
//     rows) items, in that order. Every CTA takes an equal, contiguous share of the
//     list, whatever the lengths are -- they are read on the device -- so ragged
//     batches and one long sequence fill the SMs alike. An item that lies in several
//     CTAs is joined by the last of them to finish, in the order of the list.
//   * One producer warp per CTA keeps a ring of tiles in flight with TMA (swizzled,
//     so that the fragment loads below have no bank conflicts), looks pages and
//     scales up 32 at a time and one batch ahead, and hands each 16 tokens their
//     factors through shared memory.
//   * Four compute warps share a tile's 16-token groups and the rows' 16-row groups.
//     Scores and outputs are m16n8k16 fp16 products of the codes (exact in fp16)
//     with fp32 sums: with at most 64 rows a 128-row tcgen05 tile would
//     be mostly padding, and the tensor pipe is not what bounds this. The order of
//     the channels within a product is free, so a lane's fragments of K are 16 or 32
//     consecutive bytes of one token, and so are its outputs.
//
// Softmax in powers of two: with x_j = log2(e) * scale * q.k_j and a page's value
// scale vs, the weight that meets the codes of V is w_j = 2^(x_j + log2 vs - m),
// m a running maximum of x_j + log2 vs, at most 2^8 too small (raising it rescales
// the sums, so it is raised only when needed). The output is sum w_j code_j /
// sum (w_j / vs). So w_j, rounded to fp16, is relative to the largest product of
// weight and value scale, and pages of small scale lose nothing.
#include <algorithm>
#include <mutex>
#include <vector>

#include "wbk_kv8.cuh"
#include "wbk_sm100.cuh"

namespace wbk {
namespace {

constexpr int kTile = 64;          // tokens per ring stage
constexpr int kGroups = kTile / 16;
constexpr int kComputeWarps = 4;
constexpr int kStepThreads = kComputeWarps * 32 + 32;
constexpr int kMinTiles = 2;       // of a CTA's share, where the SMs are not full
constexpr float kRaise = 8.0f;     // log2 units
constexpr float kLog2e = 1.4426950408889634f;

constexpr uint64_t kDrainNs = 100000000ull;  // limit of the waits for copies in flight at a CTA's end

enum : uint32_t { KSITE_PRODUCER = 41, KSITE_COMPUTE = 42, KSITE_DRAIN = 43 };

struct Kv8AttnParams {
  const void* q;
  void* out;
  int64_t q_sb, q_sh, q_ss, o_sb, o_sh, o_ss;
  Kv8Pages c;
  const float *k_scale, *v_scale;
  const int32_t* lens;
  const int32_t* q_lens;
  int batch, group, queries, rows;  // rows = group * queries of one KV head
  int row_blocks;                   // blocks of 16 * kWR rows
  int causal, bf16;
  float scale_log2;  // scale * log2(e)
  uint32_t* tickets;
  float* parts;
  uint64_t timeout_ns;
};

template <int kD, int kWR>
struct StepCfg {
  static constexpr int kRows = 16 * kWR;
  static constexpr int kCtasPerSm = kD == 64 ? 3 : 2;  // what the registers of a lane's fragments allow
  static constexpr int kStages = kD == 64 ? 6 : kWR == 2 ? 5 : 6;  // and what then fits into shared memory
  static constexpr int kTileBytes = kTile * kD;
  static constexpr int kPartFloats = kRows * (kD + 2);  // one partial result: sums, maxima, totals
};

template <int kD, int kWR>
struct StepSmem {
  static constexpr int kStages = StepCfg<kD, kWR>::kStages;
  uint8_t k[kStages][kTile * kD];  // 1024-byte aligned (swizzle atoms)
  uint8_t v[kStages][kTile * kD];
  float4 factor[kStages][kGroups];  // of 16 tokens: key factor, log2 of the value scale, its inverse, 1 if there
  float sum[kWR < 4 ? 16 * kWR * kD : 4];  // joins the compute warps of one row group
  float max[kComputeWarps][16], total[kComputeWarps][16];
  uint64_t full[kStages], empty[kStages];
  int last;
  int abort_flag;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int kFmt>
__device__ __forceinline__ uint32_t half2_bits(uint32_t codes) {
  const __half2 h = kv8_half2<kFmt>(codes);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint2 lds8(const uint8_t* p) { return *reinterpret_cast<const uint2*>(p); }

__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kComputeWarps * 32) : "memory"); }

// One item of the work list: KV head h of sequence b, rows 16 * kWR * rb onwards.
struct Item {
  int b, h, rb;
  int len, n;  // cached tokens, real query rows
  int tiles;   // 64-token tiles, at least 1 (an item without tokens still writes its zeros)
};

__device__ __forceinline__ int tiles_of(const Kv8AttnParams& p, int b, int& len, int& n) {
  len = kv8_len(p.lens, b, p.c);
  n = p.q_lens != nullptr ? min(max(p.q_lens[b], 0), p.queries) : p.queries;
  if (n == 0) len = 0;
  return max((len + kTile - 1) / kTile, 1);
}

// Tiles of the whole list, by a converged warp.
__device__ __forceinline__ int64_t total_tiles(const Kv8AttnParams& p) {
  int64_t sum = 0;
  int len, n;
  for (int b = threadIdx.x & 31; b < p.batch; b += 32) sum += tiles_of(p, b, len, n);
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  return sum * p.c.kv_heads * p.row_blocks;
}

// The item and tile at place x of the list, by a converged warp.
__device__ __forceinline__ Item locate(const Kv8AttnParams& p, int64_t x, int& tile) {
  const int lane = threadIdx.x & 31;
  const int64_t per = static_cast<int64_t>(p.c.kv_heads) * p.row_blocks;
  Item it{};
  for (int b0 = 0;; b0 += 32) {
    int len = 0, n = 0;
    const int t = b0 + lane < p.batch ? tiles_of(p, b0 + lane, len, n) : 0;
    int64_t upto = t;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += y;
    }
    const uint32_t past = __ballot_sync(~0u, upto * per > x);
    if (past == 0 && b0 + 32 < p.batch) {
      x -= __shfl_sync(~0u, upto, 31) * per;
      continue;
    }
    const int src = past != 0 ? __ffs(past) - 1 : 31;
    x -= __shfl_sync(~0u, upto - t, src) * per;
    it.b = b0 + src;
    it.len = __shfl_sync(~0u, len, src);
    it.n = __shfl_sync(~0u, n, src);
    it.tiles = __shfl_sync(~0u, t, src);
    const int hr = static_cast<int>(x / it.tiles);
    tile = static_cast<int>(x - static_cast<int64_t>(hr) * it.tiles);
    it.h = hr / p.row_blocks;
    it.rb = hr - it.h * p.row_blocks;
    return it;
  }
}

__device__ __forceinline__ void next_item(const Kv8AttnParams& p, Item& it) {
  if (++it.rb < p.row_blocks) return;
  it.rb = 0;
  if (++it.h < p.c.kv_heads) return;
  it.h = 0;
  ++it.b;
  if (it.b < p.batch) it.tiles = tiles_of(p, it.b, it.len, it.n);
}

// A lane's page of a batch of 32 consecutive pages of an item, with its scales.
struct PageLane {
  int64_t page;
  float ks, vs;
};
__device__ __forceinline__ PageLane fetch_page(const Kv8AttnParams& p, const Item& it, int blk) {
  PageLane r{-1, 0.0f, 1.0f};
  if ((static_cast<int64_t>(blk) << p.c.block_log2) < it.len) r.page = kv8_page(p.c, it.b, blk);
  if (r.page >= 0) {
    const int64_t ph = r.page * p.c.kv_heads + it.h;
    r.ks = p.k_scale[ph];
    r.vs = p.v_scale[ph];
  }
  return r;
}

// log2, exact for powers of two.
__device__ __forceinline__ float log2_scale(float s) {
  const int e = static_cast<int>(__float_as_uint(s) >> 23) - 127;
  const uint32_t frac = __float_as_uint(s) & 0x7FFFFFu;
  return frac == 0 ? static_cast<float>(e) : log2f(s);
}

template <int kFmt, int kD, int kWR, bool kHalf>
__global__ void __launch_bounds__(kStepThreads, StepCfg<kD, kWR>::kCtasPerSm)
kv8_step_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                const Kv8AttnParams p) {
  using Cfg = StepCfg<kD, kWR>;
  using Smem = StepSmem<kD, kWR>;
  constexpr int kStages = Cfg::kStages;
  constexpr int kTG = kComputeWarps / kWR;   // warps that share a row group's tokens
  constexpr int kKSteps = kD / 16;
  constexpr int kNTiles = kD / 8;
  extern __shared__ uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort_flag;

  // this CTA's share [x0, x1) of the list
  const int64_t total = total_tiles(p);
  const int64_t active = max(min(static_cast<int64_t>(gridDim.x), total / kMinTiles), static_cast<int64_t>(1));
  if (blockIdx.x >= active) return;
  const int64_t x0 = blockIdx.x * total / active, x1 = (blockIdx.x + 1) * total / active;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], kComputeWarps);
    }
    s.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  int tile = 0;
  Item it = locate(p, x0, tile);

  if (warp == kComputeWarps) {
    // ---------------------------------------------------------- producer
    const int sub = p.c.block < kTile ? p.c.block_log2 : 6;          // log2 of tokens per TMA box
    const int boxes = kTile >> sub;                                  // per tile
    const int batch_tiles = p.c.block < kTile ? 32 / boxes : 32 << (p.c.block_log2 - 6);
    uint32_t g = 0;
    bool ok = true;
    int64_t x = x0;
    auto first_blk = [&](int t) { return (t * kTile) >> p.c.block_log2; };
    PageLane cur = fetch_page(p, it, first_blk(tile) + lane);
    while (x < x1 && ok) {
      const int t1 = static_cast<int>(min(static_cast<int64_t>(it.tiles), tile + (x1 - x)));
      Item nit = it;
      if (x + (t1 - tile) < x1) next_item(p, nit);
      for (int tb = tile; tb < t1 && ok;) {
        const int blk0 = first_blk(tb);
        const int te = min(t1, ((blk0 << p.c.block_log2) / kTile) + batch_tiles);  // tiles that cur covers
        const PageLane nxt = te < t1 ? fetch_page(p, it, first_blk(te) + lane) : fetch_page(p, nit, lane);
        for (int t = tb; t < te; ++t, ++g) {
          const int st = static_cast<int>(g % kStages);
          const uint32_t ph = (g / kStages) & 1u;
          ok = __all_sync(~0u, mbar_wait_inl(&s.empty[st], ph ^ 1u, abort_flag, p.timeout_ns, KSITE_PRODUCER));
          if (!ok) break;
          const int pos = t * kTile + (lane & 3) * 16;  // of 16-token group lane & 3
          const int from = ((pos >> p.c.block_log2) - blk0) & 31;
          const int64_t page = __shfl_sync(~0u, cur.page, from);
          const float ks = __shfl_sync(~0u, cur.ks, from), vs = __shfl_sync(~0u, cur.vs, from);
          const bool there = page >= 0 && pos < it.len;
          if (lane < kGroups)
            s.factor[st][lane] = make_float4(ks * p.scale_log2, log2_scale(vs), 1.0f / vs, there ? 1.0f : 0.0f);
          __syncwarp();
          // the first 16-token group of each box stands for it
          const bool load = lane < kGroups && there && (lane & ((1 << (sub - 4)) - 1)) == 0;
          const uint32_t loads = __popc(__ballot_sync(~0u, load));
          if (lane == 0) mbar_arrive_expect_tx(&s.full[st], loads * 2u * (static_cast<uint32_t>(kD) << sub));
          __syncwarp();
          if (load) {
            const int y = (it.h << p.c.block_log2) + (pos & (p.c.block - 1));
            tma_load_3d(&tmap_k, &s.full[st], s.k[st] + lane * 16 * kD, 0, y, static_cast<int>(page));
            tma_load_3d(&tmap_v, &s.full[st], s.v[st] + lane * 16 * kD, 0, y, static_cast<int>(page));
          }
        }
        tb = te;
        cur = nxt;
      }
      x += t1 - tile;
      tile = 0;
      it = nit;
    }
    // Every copy lands before the CTA ends, also when a compute warp gave up waiting.
    if (lane == 0) {
      int dummy = 0;
      for (uint32_t i = g > kStages ? g - kStages : 0; i < g; ++i)
        mbar_wait_inl(&s.full[i % kStages], (i / kStages) & 1u, &dummy, kDrainNs, KSITE_DRAIN);
    }
  } else {
    // ----------------------------------------------------------- compute
    const int wr = warp % kWR, tg = warp / kWR;  // row group, token group
    const int gid = lane >> 2, c = lane & 3;
    uint32_t g = 0;
    bool ok = true;
    int64_t x = x0;
    while (x < x1) {
      const int t1 = static_cast<int>(min(static_cast<int64_t>(it.tiles), tile + (x1 - x)));
      // ---- this lane's rows (gid and gid + 8 of the row group), their queries and how much they see
      uint32_t qf[kKSteps][4];
      float qfac[2];
      int vis[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = it.rb * Cfg::kRows + wr * 16 + gid + half * 8;
        vis[half] = INT_MAX;  // rows beyond the last hide nothing: their results are dropped
        qfac[half] = 1.0f;
        uint32_t w[kD / 8];
#pragma unroll
        for (int i = 0; i < kD / 8; ++i) w[i] = 0u;
        if ((!kHalf || half == 0) && r < p.rows) {
          const int gi = r / p.queries, i = r - gi * p.queries;
          vis[half] = i >= it.n ? 0 : p.causal ? max(it.len - it.n + i + 1, 0) : it.len;
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + it.b * p.q_sb +
                                                            (it.h * p.group + gi) * p.q_sh + i * p.q_ss + c * (kD / 4));
#pragma unroll
          for (int i4 = 0; i4 < kD / 32; ++i4) {
            const uint4 u = src[i4];
            w[4 * i4] = u.x, w[4 * i4 + 1] = u.y, w[4 * i4 + 2] = u.z, w[4 * i4 + 3] = u.w;
          }
        }
        if (p.bf16) {
          // bf16 -> fp16 times a power of two that puts the row's largest value into [2^14, 2^15): exact but for
          // values 2^-28 of the largest and below; the power comes back as a factor of the scores
          float amax = 0.0f;
#pragma unroll
          for (int i = 0; i < kD / 8; ++i) {
            const float2 f = pair_to_float2<WBK_DT_BF16>(w[i]);
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
          amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
          amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
          const int e = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -100), 127);
          const float up = kv8_pow2(14 - e);
          qfac[half] = kv8_pow2(min(e - 14, 126));
#pragma unroll
          for (int i = 0; i < kD / 8; ++i) {
            const float2 f = pair_to_float2<WBK_DT_BF16>(w[i]);
            w[i] = float2_to_pair<WBK_DT_F16>(f.x * up, f.y * up);
          }
        }
#pragma unroll
        for (int k = 0; k < kKSteps; ++k) qf[k][half] = w[2 * k], qf[k][half + 2] = w[2 * k + 1];
      }
      const int clear = __reduce_min_sync(~0u, min(vis[0], vis[1]));  // tokens that no row of this warp hides

      float o[kNTiles][4];
#pragma unroll
      for (int j = 0; j < kNTiles; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

      for (int t = tile; t < t1; ++t, ++g) {
        const int st = static_cast<int>(g % kStages);
        if (ok) ok = __all_sync(~0u, mbar_wait_inl(&s.full[st], (g / kStages) & 1u, abort_flag, p.timeout_ns, KSITE_COMPUTE));
        if (ok) {
#pragma unroll 1
          for (int gi = tg; gi < kGroups; gi += kTG) {
            const float4 fac = s.factor[st][gi];
            if (fac.w == 0.0f) continue;
            const uint8_t* kt = s.k[st];
            const uint8_t* vt = s.v[st];
            const int pos = t * kTile + gi * 16;
            // ---- scores of 16 tokens: tokens gid (first n-tile) and gid + 8 (second)
            float sc[2][4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
              const int tok = gi * 16 + nt * 8 + gid;
              sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
              if constexpr (kD == 64) {
                const uint4 u = lds16(kt + tok * 64 + ((c ^ ((tok >> 1) & 3)) << 4));
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  mma16816(sc[nt], qf[k], half2_bits<kFmt>(w[k]), half2_bits<kFmt>(w[k] >> 16));
              } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint4 u = lds16(kt + tok * 128 + (((2 * c + h) ^ (tok & 7)) << 4));
                  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    mma16816(sc[nt], qf[4 * h + k], half2_bits<kFmt>(w[k]), half2_bits<kFmt>(w[k] >> 16));
                }
              }
            }
            // ---- x + log2 vs, masked; raise the maximum where a weight would pass 2^8
            constexpr int kHalves = kHalf ? 1 : 2;
            const bool edge = pos + 16 > clear;
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
              const float km = fac.x * qfac[half];
#pragma unroll
              for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float v = fmaf(sc[nt][2 * half + e], km, fac.y);
                  if (edge && pos + nt * 8 + 2 * c + e >= vis[half]) v = -INFINITY;
                  sc[nt][2 * half + e] = v;
                  top[half] = fmaxf(top[half], v);
                }
            }
            if (__any_sync(~0u, top[0] > m[0] + kRaise || (!kHalf && top[1] > m[1] + kRaise))) {
#pragma unroll
              for (int half = 0; half < kHalves; ++half) {
                top[half] = fmaxf(top[half], __shfl_xor_sync(~0u, top[half], 1));
                top[half] = fmaxf(top[half], __shfl_xor_sync(~0u, top[half], 2));
                const float up = fmaxf(m[half], top[half]);
                const float alpha = up == -INFINITY ? 1.0f : ex2(m[half] - up);
                m[half] = up;
                l[half] *= alpha;
#pragma unroll
                for (int j = 0; j < kNTiles; ++j) o[j][2 * half] *= alpha, o[j][2 * half + 1] *= alpha;
              }
            }
            // ---- weights, as the A operand of the second product
            uint32_t pa[4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (half < kHalves) {
                const float ref = m[half] == -INFINITY ? 0.0f : m[half];
                float sum = 0.0f;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                  const float w0 = ex2(sc[nt][2 * half] - ref), w1 = ex2(sc[nt][2 * half + 1] - ref);
                  const __half2 h = __floats2half2_rn(w0, w1);
                  pa[2 * nt + half] = *reinterpret_cast<const uint32_t*>(&h);
                  sum += w0 + w1;
                }
                l[half] = fmaf(sum, fac.z, l[half]);
              } else {
                pa[1] = pa[3] = 0u;
              }
            }
            // ---- outputs: tokens 2c, 2c + 1 and 2c + 8, 2c + 9, channels gid * kD / 8 ..
            uint32_t va[4][kD / 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              // for head_dim 64 odd lanes of a quad take the two tokens of a pair in the other order (see below)
              const int e = kD == 64 ? (i & 1) ^ (c & 1) : i & 1;
              const int tok = gi * 16 + (i >> 1) * 8 + 2 * c + e;
              if constexpr (kD == 64) {
                const uint2 u = lds8(vt + tok * 64 + (((gid >> 1) ^ ((tok >> 1) & 3)) << 4) + (gid & 1) * 8);
                va[i][0] = u.x, va[i][1] = u.y;
              } else {
                const uint4 u = lds16(vt + tok * 128 + ((gid ^ (tok & 7)) << 4));
                va[i][0] = u.x, va[i][1] = u.y, va[i][2] = u.z, va[i][3] = u.w;
              }
              if (edge && t * kTile + tok >= it.len) {  // whatever lies there, a weight of 0 has to give 0
#pragma unroll
                for (int w = 0; w < kD / 32; ++w) va[i][w] = 0u;
              }
            }
            // bytes of a token pair side by side; with head_dim 64 the loads of a half-warp hit all banks once only
            // if even and odd lanes of a quad read different halves of the 128-byte lines, so the selector swaps back
            const uint32_t lo = kD == 64 && (c & 1) ? 0x1504u : 0x5140u, hi = kD == 64 && (c & 1) ? 0x3726u : 0x7362u;
#pragma unroll
            for (int w = 0; w < kD / 32; ++w) {
              const uint32_t a01 = __byte_perm(va[0][w], va[1][w], lo), a23 = __byte_perm(va[0][w], va[1][w], hi);
              const uint32_t b01 = __byte_perm(va[2][w], va[3][w], lo), b23 = __byte_perm(va[2][w], va[3][w], hi);
              mma16816(o[4 * w], pa, half2_bits<kFmt>(a01), half2_bits<kFmt>(b01));
              mma16816(o[4 * w + 1], pa, half2_bits<kFmt>(a01 >> 16), half2_bits<kFmt>(b01 >> 16));
              mma16816(o[4 * w + 2], pa, half2_bits<kFmt>(a23), half2_bits<kFmt>(b23));
              mma16816(o[4 * w + 3], pa, half2_bits<kFmt>(a23 >> 16), half2_bits<kFmt>(b23 >> 16));
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.empty[st]);
        }
      }

      // ---- join the warps that shared this row group's tokens, in order
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        l[half] += __shfl_xor_sync(~0u, l[half], 1);
        l[half] += __shfl_xor_sync(~0u, l[half], 2);
        if (kTG > 1 && c == 0) s.max[warp][gid + 8 * half] = m[half];
      }
      if constexpr (kTG > 1) {
        compute_barrier();
        float fac[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < kTG; ++i) top = fmaxf(top, s.max[wr + i * kWR][gid + 8 * half]);
          fac[half] = m[half] == -INFINITY ? 0.0f : ex2(m[half] - top);
          m[half] = top;
          if (c == 0) s.total[warp][gid + 8 * half] = l[half] * fac[half];
        }
        for (int turn = 0; turn < kTG; ++turn) {
          if (turn == tg) {
#pragma unroll
            for (int half = 0; half < (kHalf ? 1 : 2); ++half) {
              float4* dst = reinterpret_cast<float4*>(&s.sum[(wr * 16 + gid + 8 * half) * kD + c * (kD / 4)]);
#pragma unroll
              for (int j = 0; j < kNTiles; j += 4) {  // column pair e of n-tile j is channel e * kD / 8 + j of the lane
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float4 v = make_float4(o[j][2 * half + e] * fac[half], o[j + 1][2 * half + e] * fac[half],
                                         o[j + 2][2 * half + e] * fac[half], o[j + 3][2 * half + e] * fac[half]);
                  float4& at = dst[(e * (kD / 8) + j) / 4];
                  if (turn > 0) v.x += at.x, v.y += at.y, v.z += at.z, v.w += at.w;
                  at = v;
                  o[j][2 * half + e] = v.x, o[j + 1][2 * half + e] = v.y;
                  o[j + 2][2 * half + e] = v.z, o[j + 3][2 * half + e] = v.w;
                }
              }
            }
          }
          compute_barrier();
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          l[half] = 0.0f;
#pragma unroll
          for (int i = 0; i < kTG; ++i) l[half] += s.total[wr + i * kWR][gid + 8 * half];
        }
      }

      // ---- the row groups' last warps hold the sums: write the output, or this CTA's part of it
      const bool whole = tile == 0 && t1 == it.tiles;
      const int slot = tile == 0 ? 1 : 0;
      float* part = p.parts + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * Cfg::kPartFloats;
      if (tg == kTG - 1) {
#pragma unroll
        for (int half = 0; half < (kHalf ? 1 : 2); ++half) {
          const int rl = wr * 16 + gid + 8 * half, r = it.rb * Cfg::kRows + rl;
          if (r >= p.rows) continue;
          if (whole) {
            const int gi = r / p.queries, i = r - gi * p.queries;
            const float inv = l[half] == 0.0f ? 0.0f : 1.0f / l[half];
            uint16_t* dst = static_cast<uint16_t*>(p.out) + it.b * p.o_sb + (it.h * p.group + gi) * p.o_sh + i * p.o_ss +
                            c * (kD / 4);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int j = 0; j < kNTiles; j += 8) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const float a = o[j + 2 * k][2 * half + e] * inv, b = o[j + 2 * k + 1][2 * half + e] * inv;
                  w[k] = p.bf16 ? float2_to_pair<WBK_DT_BF16>(a, b) : float2_to_pair<WBK_DT_F16>(a, b);
                }
                *reinterpret_cast<uint4*>(dst + e * (kD / 8) + j) = make_uint4(w[0], w[1], w[2], w[3]);
              }
          } else {
            float4* dst = reinterpret_cast<float4*>(part + rl * kD + c * (kD / 4));
#pragma unroll
            for (int j = 0; j < kNTiles; j += 4)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                dst[(e * (kD / 8) + j) / 4] = make_float4(o[j][2 * half + e], o[j + 1][2 * half + e],
                                                         o[j + 2][2 * half + e], o[j + 3][2 * half + e]);
            if (c == 0) {
              part[Cfg::kRows * kD + rl] = m[half];
              part[Cfg::kRows * (kD + 1) + rl] = l[half];
            }
          }
        }
      }
      if (!whole) {
        // the CTAs of this item: first .. last of the list's shares that reach into it
        const int64_t begin = x - tile, end = begin + it.tiles;
        const int first = static_cast<int>(((begin + 1) * active - 1) / total);
        const int last = static_cast<int>((end * active - 1) / total);
        __threadfence();
        compute_barrier();
        if (threadIdx.x == 0) {
          const uint32_t before = atomicAdd(&p.tickets[first], 1u);
          s.last = before == static_cast<uint32_t>(last - first);
          if (s.last) p.tickets[first] = 0u;
        }
        compute_barrier();
        if (s.last) {
          __threadfence();
          const int rows = min(Cfg::kRows, p.rows - it.rb * Cfg::kRows);
          const int64_t stride = 2 * Cfg::kPartFloats;
          // part of CTA i: its slot 0, but slot 1 for the first
          const float* base = p.parts + static_cast<int64_t>(first) * stride;
          const int parts = last - first + 1;
          for (int idx = threadIdx.x; idx < rows * (kD / 4); idx += kComputeWarps * 32) {
            const int rl = idx / (kD / 4), d4 = idx % (kD / 4);
            float top = -INFINITY;
            for (int i = 0; i < parts; ++i)
              top = fmaxf(top, __ldcg(base + i * stride + (i == 0 ? Cfg::kPartFloats : 0) + Cfg::kRows * kD + rl));
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float tot = 0.0f;
            for (int i = 0; i < parts; ++i) {
              const float* q = base + i * stride + (i == 0 ? Cfg::kPartFloats : 0);
              const float mi = __ldcg(q + Cfg::kRows * kD + rl);
              const float f = mi == -INFINITY ? 0.0f : ex2(mi - top);
              const float4 v = __ldcg(reinterpret_cast<const float4*>(q + rl * kD) + d4);
              tot = fmaf(f, __ldcg(q + Cfg::kRows * (kD + 1) + rl), tot);
              sum.x = fmaf(f, v.x, sum.x), sum.y = fmaf(f, v.y, sum.y);
              sum.z = fmaf(f, v.z, sum.z), sum.w = fmaf(f, v.w, sum.w);
            }
            const float inv = tot == 0.0f ? 0.0f : 1.0f / tot;
            const int r = it.rb * Cfg::kRows + rl, gi = r / p.queries, i = r - gi * p.queries;
            uint16_t* dst = static_cast<uint16_t*>(p.out) + it.b * p.o_sb + (it.h * p.group + gi) * p.o_sh + i * p.o_ss;
            uint2 w;
            if (p.bf16) {
              w.x = float2_to_pair<WBK_DT_BF16>(sum.x * inv, sum.y * inv);
              w.y = float2_to_pair<WBK_DT_BF16>(sum.z * inv, sum.w * inv);
            } else {
              w.x = float2_to_pair<WBK_DT_F16>(sum.x * inv, sum.y * inv);
              w.y = float2_to_pair<WBK_DT_F16>(sum.z * inv, sum.w * inv);
            }
            *reinterpret_cast<uint2*>(dst + d4 * 4) = w;
          }
        }
      }
      x += t1 - tile;
      tile = 0;
      if (x < x1) next_item(p, it);
    }
  }
}

// Pages as a 3-D tensor (channel, head * block + token, page) of bytes; a box is one page's tokens of one head, at
// most a tile of them, swizzled over its row length.
int make_tmap_pages(CUtensorMap* map, const void* base, int64_t pages, int64_t kv_heads, int64_t block, int64_t d) {
  auto encode = get_encode_fn();
  if (encode == nullptr) return fail(WBK_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(kv_heads * block),
                              static_cast<cuuint64_t>(pages)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(kv_heads * block * d)};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(d), static_cast<cuuint32_t>(std::min<int64_t>(block, kTile)), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE,
                            d == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(WBK_ERR_CUDA, "cuTensorMapEncodeTiled (kv8 pages) failed (%d)", static_cast<int>(r));
  return WBK_OK;
}

int step_sms() {
  const int n = sm_count();
  return n > 0 ? n : 148;
}

// Row groups (of 16) that share a CTA's tiles: as many as the rows need, up to 4.
int row_groups(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

// Tickets first (one per CTA), then two partial results per CTA.
int64_t step_ctas(int64_t head_dim) {
  return static_cast<int64_t>(step_sms()) * (head_dim == 64 ? StepCfg<64, 1>::kCtasPerSm : StepCfg<128, 1>::kCtasPerSm);
}
int64_t ticket_bytes(int64_t head_dim) { return (step_ctas(head_dim) * 4 + 255) / 256 * 256; }

template <int kFmt, int kD, int kWR, bool kHalf>
int launch_step(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int grid, cudaStream_t stream) {
  constexpr size_t smem = sizeof(StepSmem<kD, kWR>) + 1024;
  static_assert((smem + 1024) * StepCfg<kD, kWR>::kCtasPerSm <= 233472, "shared memory budget");
  static std::mutex mu;
  static std::vector<char> configured;
  const int dev = current_device();
  if (dev < 0) return fail(WBK_ERR_CUDA, "no current CUDA device");
  {
    std::lock_guard<std::mutex> lock(mu);
    if (static_cast<int>(configured.size()) <= dev) configured.resize(dev + 1, 0);
    if (!configured[dev]) {
      if (int e = cuda_check(cudaFuncSetAttribute(kv8_step_kernel<kFmt, kD, kWR, kHalf>,
                                                  cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)),
                             "kv8 attention smem attribute"))
        return e;
      configured[dev] = 1;
    }
  }
  kv8_step_kernel<kFmt, kD, kWR, kHalf><<<grid, kStepThreads, smem, stream>>>(tk, tv, p);
  return cuda_check(cudaGetLastError(), "kv8 attention launch");
}

template <int kFmt, int kD>
int dispatch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int grid, cudaStream_t stream) {
  if (p.rows <= 8) return launch_step<kFmt, kD, 1, true>(tk, tv, p, grid, stream);
  switch (row_groups(p.rows)) {
    case 1: return launch_step<kFmt, kD, 1, false>(tk, tv, p, grid, stream);
    case 2: return launch_step<kFmt, kD, 2, false>(tk, tv, p, grid, stream);
    default: return launch_step<kFmt, kD, 4, false>(tk, tv, p, grid, stream);
  }
}

}  // namespace

int kv8_read_device_error(uint32_t* v, bool clear) {
  if (int e = cuda_check(cudaMemcpyFromSymbol(v, g_device_error, sizeof(*v)), "kv8 device error read")) return e;
  if (clear) {
    const uint32_t zero = 0;
    if (int e = cuda_check(cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero)), "kv8 device error clear")) return e;
  }
  return WBK_OK;
}

}  // namespace wbk

using namespace wbk;

extern "C" {

int64_t wbk_attention_kv8_ws_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t queries, int64_t head_dim) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || queries <= 0 || head_dim <= 0) return 0;
  const int64_t rows = 16 * row_groups(heads / kv_heads * queries);
  return ticket_bytes(head_dim) + step_ctas(head_dim) * 2 * rows * (head_dim + 2) * 4;
}

int wbk_attention_kv8(const void* q, void* out, int dtype, int64_t batch, int64_t heads, int64_t kv_heads,
                      int64_t queries, int64_t head_dim, const int64_t* strides, int fmt, const void* k_cache,
                      const void* v_cache, const float* k_scale, const float* v_scale, int64_t pages, int64_t block,
                      const int32_t* block_table, int64_t max_blocks, int64_t table_stride, const int32_t* seq_lens,
                      const int32_t* q_lens, int causal, float scale, void* workspace, int64_t workspace_bytes,
                      wbk_stream_t stream) {
  if (batch < 0 || heads < 0 || kv_heads < 0 || queries < 0)
    return fail(WBK_ERR_INVALID_ARG, "wbk_attention_kv8: negative size");
  if (dtype != WBK_DT_F16 && dtype != WBK_DT_BF16)
    return fail(WBK_ERR_INVALID_ARG, "wbk_attention_kv8: dtype %d (WBK_DT_F16 or WBK_DT_BF16)", dtype);
  if (batch == 0 || heads == 0 || queries == 0) return WBK_OK;
  if (q == nullptr || out == nullptr || strides == nullptr)
    return fail(WBK_ERR_INVALID_ARG, "wbk_attention_kv8: null pointer");
  if (int e = kv8_check_pages("wbk_attention_kv8", k_cache, v_cache, k_scale, v_scale, pages, kv_heads, block, head_dim,
                              fmt, block_table, max_blocks, table_stride, seq_lens))
    return e;
  if (heads % kv_heads != 0)
    return fail(WBK_ERR_INVALID_ARG, "wbk_attention_kv8: %lld query heads do not share %lld KV heads evenly",
                (long long)heads, (long long)kv_heads);
  if (batch > 32767 || heads > 65535 || queries > (1 << 14))
    return fail(WBK_ERR_UNSUPPORTED, "wbk_attention_kv8: size beyond batch 32767, heads 65535, queries 16384");
  if (q_lens != nullptr && !aligned(q_lens, 4))
    return fail(WBK_ERR_INVALID_ARG, "wbk_attention_kv8: q_lens misaligned");
  if (!aligned(q, 16) || !aligned(out, 16))
    return fail(WBK_ERR_UNSUPPORTED, "wbk_attention_kv8: q and out must be 16-byte aligned");
  for (int i = 0; i < 6; ++i)
    if (!kv8_stride_ok(strides[i]))
      return fail(WBK_ERR_UNSUPPORTED, "wbk_attention_kv8: stride[%d] = %lld is not a multiple of 8 elements", i,
                  (long long)strides[i]);
  const int64_t need = wbk_attention_kv8_ws_bytes(batch, heads, kv_heads, queries, head_dim);
  if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256))
    return fail(WBK_ERR_INVALID_ARG, "wbk_attention_kv8: needs a 256-byte aligned workspace of %lld bytes", (long long)need);

  Kv8AttnParams p{};
  p.q = q;
  p.out = out;
  p.q_sb = strides[0], p.q_sh = strides[1], p.q_ss = strides[2];
  p.o_sb = strides[3], p.o_sh = strides[4], p.o_ss = strides[5];
  p.c = kv8_pages(pages, kv_heads, block, block_table, max_blocks, table_stride);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.lens = seq_lens;
  p.q_lens = q_lens;
  p.batch = static_cast<int>(batch);
  p.group = static_cast<int>(heads / kv_heads);
  p.queries = static_cast<int>(queries);
  p.rows = p.group * p.queries;
  const int rb = 16 * row_groups(p.rows);
  p.row_blocks = (p.rows + rb - 1) / rb;
  p.causal = causal;
  p.bf16 = dtype == WBK_DT_BF16;
  p.scale_log2 = scale * kLog2e;
  p.tickets = static_cast<uint32_t*>(workspace);
  p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ticket_bytes(head_dim));
  p.timeout_ns = wait_timeout_ns();
  CUtensorMap tk, tv;
  if (int e = make_tmap_pages(&tk, k_cache, pages, kv_heads, block, head_dim)) return e;
  if (int e = make_tmap_pages(&tv, v_cache, pages, kv_heads, block, head_dim)) return e;
  // the lengths are on the device: as many CTAs as the table could need, at most what the SMs hold
  const int64_t most = batch * kv_heads * p.row_blocks * ((max_blocks * block + kTile - 1) / kTile);
  const int grid = static_cast<int>(std::min<int64_t>(step_ctas(head_dim), std::max<int64_t>(most / kMinTiles, 1)));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (fmt == WBK_FMT_E4M3)
    return head_dim == 64 ? dispatch_rows<WBK_FMT_E4M3, 64>(tk, tv, p, grid, st)
                          : dispatch_rows<WBK_FMT_E4M3, 128>(tk, tv, p, grid, st);
  return head_dim == 64 ? dispatch_rows<WBK_FMT_E5M2, 64>(tk, tv, p, grid, st)
                        : dispatch_rows<WBK_FMT_E5M2, 128>(tk, tv, p, grid, st);
}

}  // extern "C"
