// Attention over the 8-bit key/value cache for few query rows per KV head (a
// decoder's step: one or a few tokens).
//
// What bounds it: 2 * head_dim bytes of codes per token and KV head, each used by
// group * queries rows only, so HBM; nothing else may wait.
//
//   * The work is the list of 32-token tiles of all (sequence, KV head, block of 8
//     rows) items, in that order. Every warp takes an equal, contiguous share of the
//     list, whatever the lengths are -- they are read on the device -- so ragged
//     batches and one long sequence fill the SMs alike. Warps share nothing but the
//     items that lie in several of them: such an item is joined first by the last warp
//     of a CTA to finish, through shared memory, then by the last of its CTAs, through
//     global memory, always in the order of the list. CTAs split an item only if it has
//     more tiles than min(a CTA's share, kWhole).
//   * Each warp keeps a ring of tiles in flight with TMA (swizzled, so that the
//     fragment loads below have no bank conflicts) and looks pages and scales up 32
//     at a time and one batch ahead.
//   * Scores and outputs are m16n8k16 fp16 products of the codes (exact in fp16) with
//     fp32 sums, transposed: tokens (then channels) are the 16 rows, queries the 8
//     columns. With 8 columns a 128-row tcgen05 tile would be mostly padding, and the
//     tensor pipe is not what bounds this. The order of the channels within a
//     product is free, so a lane's fragments are consecutive bytes of one token.
//
// Softmax in powers of two: with x_j = log2(e) * scale * q.k_j and a page's value
// scale vs, the weight that meets the codes of V is w_j = 2^(x_j + log2 vs - m + 7),
// m a running maximum of x_j + log2 vs, at most 2^8 too small (raising it rescales
// the sums, so it is raised only when needed). The output is sum w_j code_j /
// sum (w_j / vs). So w_j, rounded to fp16, is relative to the largest product of
// weight and value scale, and pages of small scale lose nothing. The rounding, as fp16
// codes need fp16 weights, is an error of 2^-11 of each weight and of 2^-32 of the
// largest product; totals take the fp32 weights. Queries in bf16 become fp16 by an exact power of two per row.
//
// Measured, head size 64: 64 sequences of 1500 tokens, 20 heads, one query (246 MB) 55 us:
// the first tiles are there at 5 to 11 us, half of the warps have done their last by 42 us
// (HBM's rate in between), the others by 51, and joins end at 53. The same with 45 to 448 tokens (41 MB)
// 21 us; one sequence of 224 tokens 7.4 us (launch, lengths, pages, codes, join: each
// waits for the one before). Head size 128: 16 sequences of up to 32768 tokens, 8 KV heads for
// 32 query heads (738 MB) 135 us, 5.5 TB/s, 0.84 of a plain copy's rate. Longer shares
// for the CTAs that an SM gets first, which end first, gave nothing (54.4 -> 55.2 to
// 57.5 us): HBM is busy meanwhile.
#include <algorithm>
#include <climits>
#include <mutex>
#include <vector>

#include "wbk_kv8.cuh"
#include "wbk_sm100.cuh"

namespace wbk {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;          // tokens per ring stage
constexpr int kTileLog2 = 5;
constexpr int kGroups = kTile / 16;
constexpr int kRows = 8;           // query rows per item
constexpr int kSlots = 6;          // partial results that the warps of a CTA can have for one another
constexpr int kMaxStages = 4;
constexpr int kMinShare = 8;
constexpr int kWhole = 16;         // tiles of an item that is not split between CTAs
constexpr float kRaise = 8.0f;     // log2 units
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint64_t kDrainNs = 100000000ull;  // limit of the waits for copies in flight after a wait gave up

enum : uint32_t { KSITE_TILE = 41, KSITE_DRAIN = 42 };

struct Kv8AttnParams : Kv8Attention {
  int rows;        // group * queries of one KV head
  int row_blocks;  // blocks of kRows rows
  int part_rows;   // rows of a partial result: min(rows, kRows)
  int stages;      // of a warp's ring
  uint32_t* tickets;
  float* parts;
  uint64_t timeout_ns;
};

// Shared memory: the rings (kWarps * stages tiles, 1024-byte aligned for the swizzle),
// then this, then kSlots partial results.
struct StepSmem {
  float4 factor[kWarps][kMaxStages][kGroups];  // of 16 tokens: key factor, log2 of the value scale, its inverse, 1 if there
  uint64_t full[kWarps][kMaxStages];
  uint32_t tickets[kWarps];
  int abort_flag;
};
// A partial result: sums [part_rows][kD], then maxima and totals [part_rows], in whole 16-byte units.
__host__ __device__ constexpr int part_floats(int rows, int d) { return rows * d + (2 * rows + 3) / 4 * 4; }

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

__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint2 lds8(const uint8_t* p) { return *reinterpret_cast<const uint2*>(p); }

// The transposed 8 x 8 matrix of 16-bit values (row lane / 4, columns 2 * (lane % 4) and the next).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// A try_wait may suspend for longer than a tile takes to come, so a limit below kFineTimeoutNs goes without.
__device__ __forceinline__ bool tile_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t timeout_ns) {
  if (timeout_ns >= kFineTimeoutNs && mbar_try_wait(bar, parity)) return true;
  return mbar_wait_slow(bar, parity, abort_flag, timeout_ns, KSITE_TILE);
}

// Tiles of a CTA's share, at least, where the SMs are not full: two per warp, and more for long items. An item of L
// tiles in P parts takes about a * L / P + b * P, with a the time of a tile in a CTA and b that of joining a part
// (0.18 and 0.45 us), least at a share of L / P = sqrt(L * b / a).
__device__ __forceinline__ int least_share(int total, int items) {
  return max(kMinShare, static_cast<int>(1.6f * sqrtf(static_cast<float>(total) / items)));
}

// One item of the work list: KV head h of sequence b, rows kRows * rb onwards.
struct Item {
  int b, h, rb;
  int len, n;  // cached tokens, real query rows
  int tiles;   // at least 1 (an item without tokens still writes its zeros)
};

__device__ __forceinline__ int tiles_of(const Kv8AttnParams& p, int b, int& len, int& n) {
  len = kv8_len(p.lens, b, p.c);
  n = p.q_lens != nullptr ? min(max(p.q_lens[b], 0), p.queries) : p.queries;
  if (n == 0) len = 0;
  return max((len + kTile - 1) >> kTileLog2, 1);
}

// Tiles of the whole list, by a converged warp. (The host keeps the list below 2^31 tiles.)
__device__ __forceinline__ int total_tiles(const Kv8AttnParams& p) {
  int sum = 0, len, n;
  for (int b = threadIdx.x & 31; b < p.batch; b += 32) sum += tiles_of(p, b, len, n);
  return __reduce_add_sync(~0u, sum) * p.c.kv_heads * p.row_blocks;
}

// 32 sequences of the list, one per lane of a converged warp.
struct Scan {
  int b0 = -1, base;     // the first of them, places of the list before it
  int len, n, t, upto;   // of this lane's sequence: as in Item; places up to its end, from base
  __device__ __forceinline__ void load(const Kv8AttnParams& p, int first, int places) {
    const int lane = threadIdx.x & 31;
    b0 = first;
    base = places;
    len = n = t = 0;
    if (b0 + lane < p.batch) t = tiles_of(p, b0 + lane, len, n);
    upto = t * p.c.kv_heads * p.row_blocks;
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += y;
    }
  }
};

// The item and tile at place x of the list, by a converged warp; `s` keeps what it looked at for the next place.
__device__ __forceinline__ Item locate(const Kv8AttnParams& p, int x, int& tile, Scan& s) {
  if (s.b0 < 0 || x < s.base) s.load(p, 0, 0);
  uint32_t past;
  while ((past = __ballot_sync(~0u, s.base + s.upto > x)) == 0 && s.b0 + 32 < p.batch)
    s.load(p, s.b0 + 32, s.base + __shfl_sync(~0u, s.upto, 31));
  const int src = past != 0 ? __ffs(past) - 1 : 31;
  Item it{};
  it.b = s.b0 + src;
  it.len = __shfl_sync(~0u, s.len, src);
  it.n = __shfl_sync(~0u, s.n, src);
  it.tiles = __shfl_sync(~0u, s.t, src);
  x -= s.base + __shfl_sync(~0u, s.upto, src) - it.tiles * p.c.kv_heads * p.row_blocks;
  const int hr = x / it.tiles;
  tile = x - hr * it.tiles;
  it.h = hr / p.row_blocks;
  it.rb = hr - it.h * p.row_blocks;
  return it;
}

// `total` places dealt to n owners in contiguous shares, the first `r` of them one longer.
struct Split {
  int q, r;
  __device__ __forceinline__ Split(int total, int n) : q(total / n), r(total - total / n * n) {}
  __device__ __forceinline__ int start(int k) const { return k * q + min(k, r); }
  __device__ __forceinline__ int owner(int x) const {
    const int longer = r * (q + 1);
    return x < longer ? x / (q + 1) : r + (x - longer) / q;
  }
};

// Whether CTAs may split an item of so many tiles. Joining the parts takes a CTA about 4 us, whatever their size, and
// not splitting leaves the shares uneven by half an item: 0.37 us for two tiles where all SMs read at HBM's rate.
__device__ __forceinline__ bool splits(int tiles, int share) { return tiles > min(share, kWhole); }

// Where CTA k's share begins: at the nearer end of an item that is not to be split.
__device__ __forceinline__ int share_start(const Kv8AttnParams& p, const Split& split, int k, int ctas, int total, Scan& s) {
  if (k == 0 || k == ctas) return k == 0 ? 0 : total;
  int tile;
  const int x = split.start(k);
  const Item it = locate(p, x, tile, s);
  if (splits(it.tiles, split.q)) return x;
  return 2 * tile < it.tiles ? x - tile : x - tile + it.tiles;
}

__device__ __forceinline__ void next_item(const Kv8AttnParams& p, Item& it) {
  if (++it.rb < p.row_blocks) return;
  it.rb = 0;
  if (++it.h < p.c.kv_heads) return;
  it.h = 0;
  ++it.b;
  if (it.b < p.batch) it.tiles = tiles_of(p, it.b, it.len, it.n);
}

// A lane's page of a batch of 32 consecutive pages of an item, with its scales; `factors` turns these into what they
// are to the softmax. Apart, so that the page's codes can be asked for before its scales have come.
struct PageLane {
  int page;           // -1: not there
  float ks, vs;       // scales
  float log2v, inv;   // after factors(): log2 of the value scale, its inverse; ks is the factor of the scores
  __device__ __forceinline__ void factors(const Kv8AttnParams& p) {
    ks *= p.scale_log2;
    log2v = kv8_log2(vs);
    inv = 1.0f / vs;
  }
};
__device__ __forceinline__ PageLane fetch_page(const Kv8AttnParams& p, const Item& it, int blk) {
  PageLane r{-1, 0.0f, 1.0f, 0.0f, 0.0f};
  if ((static_cast<int64_t>(blk) << p.c.block_log2) < it.len) r.page = static_cast<int>(kv8_page(p.c, it.b, blk));
  if (r.page >= 0) {
    const int64_t ph = static_cast<int64_t>(r.page) * p.c.kv_heads + it.h;
    r.ks = p.k_scale[ph];
    r.vs = p.v_scale[ph];
  }
  return r;
}

// A warp's loads: the place in its share that the next tile comes from, and the pages there.
struct Loader {
  Item it;
  int tile, t1;       // next tile of the item, end of this warp's tiles of it
  int blk0, te;       // cur covers the tiles up to te; its first page
  int x, x1;          // place in the list, end of the share
  PageLane cur, nxt;  // this batch of 32 pages and, if `ahead`, the next
  bool ahead;

  __device__ __forceinline__ int first_blk(const Kv8AttnParams& p, int t) const { return (t * kTile) >> p.c.block_log2; }
  __device__ __forceinline__ void take(const Kv8AttnParams& p, const PageLane& pages) {
    cur = pages;
    ahead = false;
    blk0 = first_blk(p, tile);
    te = min(t1, ((blk0 + 32) << p.c.block_log2) >> kTileLog2);
  }
  __device__ __forceinline__ void look_ahead(const Kv8AttnParams& p) {
    const int lane = threadIdx.x & 31;
    if (ahead) return;
    ahead = true;
    if (te < t1) {
      nxt = fetch_page(p, it, first_blk(p, te) + lane);
    } else if (x + (t1 - tile) < x1) {
      Item n = it;
      next_item(p, n);
      nxt = fetch_page(p, n, lane);
    }
  }
  __device__ __forceinline__ void start(const Kv8AttnParams& p, const Item& first, int t, int begin, int end) {
    it = first;
    tile = t;
    x = begin;
    x1 = end;
    t1 = min(it.tiles, tile + (x1 - x));
    nxt = PageLane{-1, 0.0f, 1.0f, 0.0f, 0.0f};
    take(p, fetch_page(p, it, first_blk(p, tile) + (threadIdx.x & 31)));
  }
  // The 16-token group of this lane (of kGroups) in a tile of the item: its first position, the lane of cur that has its
  // page, and whether it is there.
  __device__ __forceinline__ bool group_of(const Kv8AttnParams& p, int t, int& pos, int& page, int& from) const {
    pos = t * kTile + (threadIdx.x & (kGroups - 1)) * 16;
    from = ((pos >> p.c.block_log2) - blk0) & 31;
    page = __shfl_sync(~0u, cur.page, from);
    return page >= 0 && pos < it.len;
  }
  // Asks for the codes of tile t.
  template <int kD>
  __device__ __forceinline__ void codes(const Kv8AttnParams& p, int t, const CUtensorMap* tk, const CUtensorMap* tv,
                                        uint8_t* stage, uint64_t* full) const {
    const int lane = threadIdx.x & 31;
    int pos, page, from;
    const bool there = group_of(p, t, pos, page, from);
    // one box per page of the tile; the first 16-token group of it stands for it
    const int sub = min(p.c.block_log2, kTileLog2);
    const bool load = lane < kGroups && there && (lane & ((1 << (sub - 4)) - 1)) == 0;
    const uint32_t loads = __popc(__ballot_sync(~0u, load));
    if (lane == 0) mbar_arrive_expect_tx(full, loads * 2u * (static_cast<uint32_t>(kD) << sub));
    __syncwarp();
    if (load) {
      const int y = (it.h << p.c.block_log2) + (pos & (p.c.block - 1));
      tma_load_3d(tk, full, stage + lane * 16 * kD, 0, y, page);
      tma_load_3d(tv, full, stage + (kTile + lane * 16) * kD, 0, y, page);
    }
  }
  // Writes what the softmax needs for tile t.
  __device__ __forceinline__ void factors(const Kv8AttnParams& p, int t, float4* factor) const {
    int pos, page, from;
    const bool there = group_of(p, t, pos, page, from);
    const float key = __shfl_sync(~0u, cur.ks, from), log2v = __shfl_sync(~0u, cur.log2v, from);
    const float inv = __shfl_sync(~0u, cur.inv, from);
    if ((threadIdx.x & 31) < kGroups) factor[threadIdx.x & 31] = make_float4(key, log2v, there ? inv : 0.0f, 0.0f);
  }
  // n tiles on, none of them beyond te.
  __device__ __forceinline__ void advance(const Kv8AttnParams& p, int n) {
    tile += n;
    x += n;
    if (x < x1 && tile == te) {
      look_ahead(p);
      if (tile == t1) {
        next_item(p, it);
        tile = 0;
        t1 = min(it.tiles, x1 - x);
      }
      nxt.factors(p);
      take(p, nxt);
    }
  }
};

// Where a row's output goes; r counts the rows of one KV head.
__device__ __forceinline__ uint16_t* out_row(const Kv8AttnParams& p, const Item& it, int r) {
  const int gi = r / p.queries, i = r - gi * p.queries;
  return static_cast<uint16_t*>(p.out) + it.b * p.o_sb + (it.h * p.group + gi) * p.o_sh + i * p.o_ss;
}

// Joins `count` partial results (`at(i)`: the i-th, in the order of the list) and writes the rows: to the output, or,
// where `part` is given, to a partial result.
template <int kD, bool kShared, class At>
__device__ __forceinline__ void join(const Kv8AttnParams& p, const Item& it, const At& at, int count, int rows, float* part) {
  constexpr int kV = kD / 32;                  // channels per lane
  constexpr int kAtOnce = kShared ? kWarps : 8;  // parts in flight
  const int lane = threadIdx.x & 31, r = lane & (kRows - 1), q = lane / kRows;
  const auto load = [](const float* x) { return kShared ? *x : __ldcg(x); };
  // maxima and totals: lane (r, q) looks at row r of every 4th part
  float top = -INFINITY, total = 0.0f;
  if (r < rows) {
#pragma unroll 4
    for (int i = q; i < count; i += 4) top = fmaxf(top, load(at(i) + p.part_rows * kD + r));
  }
  top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
  top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
  const float ref = top == -INFINITY ? 0.0f : top;  // a part that saw nothing has -inf, and factor 0
  if (r < rows) {
#pragma unroll 4
    for (int i = q; i < count; i += 4) {
      const float* src = at(i) + p.part_rows * kD + r;
      total = fmaf(ex2(load(src) - ref), load(src + p.part_rows), total);
    }
  }
  total += __shfl_xor_sync(~0u, total, 8);
  total += __shfl_xor_sync(~0u, total, 16);
  if (part != nullptr && lane < rows) {
    part[p.part_rows * kD + lane] = top;
    part[p.part_rows * (kD + 1) + lane] = total;
  }
#pragma unroll 1
  for (int rl = 0; rl < rows; ++rl) {
    float sum[kV];
#pragma unroll
    for (int v = 0; v < kV; ++v) sum[v] = 0.0f;
    const float peak = __shfl_sync(~0u, ref, rl), li = __shfl_sync(~0u, total, rl);
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += kAtOnce) {
      float x[kAtOnce][kV];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const float* y = at(min(i0 + k, count - 1)) + rl * kD + lane * kV;
        if constexpr (kV == 2) {
          const float2 z = kShared ? *reinterpret_cast<const float2*>(y) : __ldcg(reinterpret_cast<const float2*>(y));
          x[k][0] = z.x, x[k][1] = z.y;
        } else {
          const float4 z = kShared ? *reinterpret_cast<const float4*>(y) : __ldcg(reinterpret_cast<const float4*>(y));
          x[k][0] = z.x, x[k][1] = z.y, x[k][2] = z.z, x[k][3] = z.w;
        }
      }
      float f = 0.0f;  // of part i0 + lane
      if (lane < kAtOnce && i0 + lane < count) f = ex2(load(at(i0 + lane) + p.part_rows * kD + rl) - peak);
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const float fk = __shfl_sync(~0u, f, k);  // 0 past the last part
#pragma unroll
        for (int v = 0; v < kV; ++v) sum[v] = fmaf(fk, x[k][v], sum[v]);
      }
    }
    if (part != nullptr) {
      float* dst = part + rl * kD + lane * kV;
      if constexpr (kV == 2) *reinterpret_cast<float2*>(dst) = make_float2(sum[0], sum[1]);
      else *reinterpret_cast<float4*>(dst) = make_float4(sum[0], sum[1], sum[2], sum[3]);
      continue;
    }
    const float inv = li == 0.0f ? 0.0f : 1.0f / li;
    uint32_t w[kV / 2];
#pragma unroll
    for (int v = 0; v < kV / 2; ++v)
      w[v] = p.bf16 ? float2_to_pair<WBK_DT_BF16>(sum[2 * v] * inv, sum[2 * v + 1] * inv)
                    : float2_to_pair<WBK_DT_F16>(sum[2 * v] * inv, sum[2 * v + 1] * inv);
    uint16_t* dst = out_row(p, it, it.rb * kRows + rl) + lane * kV;
    if constexpr (kV == 2) *reinterpret_cast<uint32_t*>(dst) = w[0];
    else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  }
}

template <int kFmt, int kD>
__global__ void __launch_bounds__(kThreads, kD == 64 ? 4 : 3)
kv8_step_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                const Kv8AttnParams p) {
  constexpr int kMTiles = kD / 16;  // of an output product
  constexpr int kTileBytes = 2 * kTile * kD;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* rings = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  StepSmem& s = *reinterpret_cast<StepSmem*>(rings + kWarps * p.stages * kTileBytes);
  float* slots = reinterpret_cast<float*>(&s + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &s.abort_flag;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
    for (int i = 0; i < kWarps; ++i) {
      for (int j = 0; j < kMaxStages; ++j) mbar_init(&s.full[i][j], 1);
      s.tickets[i] = 0;
    }
    s.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  griddep_launch_dependents();
  __syncthreads();
  griddep_wait();  // nothing below the set-up reads or writes memory that the kernel before may still use
  // this CTA's share [c0, c1) of the list, and of it this warp's, [x0, x1)
  const int total = total_tiles(p), items = p.batch * p.c.kv_heads * p.row_blocks;
  const int ctas = min(static_cast<int>(gridDim.x), max(items, total / least_share(total, items)));
  if (blockIdx.x >= ctas) return;
  const Split split(total, ctas);
  Scan scan;
  const int c0 = share_start(p, split, blockIdx.x, ctas, total, scan), c1 = share_start(p, split, blockIdx.x + 1, ctas, total, scan);
  if (c0 == c1) return;
  const int warps = min(kWarps, c1 - c0);
  const Split own(c1 - c0, warps);
  if (warp >= warps) return;
  const int x0 = c0 + own.start(warp), x1 = c0 + own.start(warp + 1);

  int tile = 0;
  Item it = locate(p, x0, tile, scan);
  uint8_t* ring = rings + warp * p.stages * kTileBytes;
  Loader loader;
  loader.start(p, it, tile, x0, x1);
  {
    // the first page batch's codes as soon as its pages are known, and then their scales; the queries meanwhile
    const int n = min(p.stages, loader.te - loader.tile);
    for (int i = 0; i < n; ++i) loader.codes<kD>(p, tile + i, &tmap_k, &tmap_v, ring + i * kTileBytes, &s.full[warp][i]);
    const int r = it.rb * kRows + (lane >> 2);
    if (r < p.rows) {
      const int gi = r / p.queries;
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + it.b * p.q_sb + (it.h * p.group + gi) * p.q_sh + (r - gi * p.queries) * p.q_ss;
      asm volatile("prefetch.global.L1 [%0];" ::"l"(q + (lane & 3) * (kD / 4)));
    }
    loader.cur.factors(p);
    for (int i = 0; i < n; ++i) loader.factors(p, tile + i, s.factor[warp][i]);
    loader.advance(p, n);
    for (int i = n; i < p.stages && loader.x < x1; ++i) {
      loader.codes<kD>(p, loader.tile, &tmap_k, &tmap_v, ring + i * kTileBytes, &s.full[warp][i]);
      loader.factors(p, loader.tile, s.factor[warp][i]);
      loader.advance(p, 1);
    }
    if (loader.x < x1) loader.look_ahead(p);
    __syncwarp();
  }

  const int gid = lane >> 2, c = lane & 3;
  // Fragment addresses within a tile. Keys: 16 (or twice 16) bytes of token gid, channels c * kD / 4 .. Values: the
  // tokens 2c and 2c + 1, channels gid * kD / 8 .. With head_dim 64 the value loads of a half-warp hit all banks
  // once only if even and odd lanes of a quad read different halves of the 128-byte lines: odd c take
  // the pair in the other order, and the selectors that interleave the pair's bytes swap it back.
  const int koff = kD == 64 ? gid * 64 + ((c ^ (gid >> 1)) & 3) * 16 : gid * 128 + ((2 * c) ^ gid) * 16;
  const int khop = kD == 64 ? 0 : (((2 * c + 1) ^ gid) - ((2 * c) ^ gid)) * 16;
  const int pair = 2 * c + (kD == 64 ? c & 1 : 0);
  const int voff0 = kTile * kD + (kD == 64 ? pair * 64 + ((gid >> 1) ^ c) * 16 + (gid & 1) * 8 : pair * 128 + (gid ^ pair) * 16);
  const int voff1 = kTile * kD + (kD == 64 ? (pair ^ 1) * 64 + ((gid >> 1) ^ c) * 16 + (gid & 1) * 8
                                           : (pair ^ 1) * 128 + (gid ^ pair ^ 1) * 16);
  const uint32_t lo = kD == 64 && (c & 1) ? 0x1504u : 0x5140u, hi = kD == 64 && (c & 1) ? 0x3726u : 0x7362u;

  int st = 0;
  uint32_t phase = 0;
  int x = x0;
  while (x < x1) {
    const int t1 = min(it.tiles, tile + (x1 - x));
    // ---- queries: row gid, channels c * kD / 4 ..
    uint32_t qf[kD / 8];
    float qfac = 1.0f;
    {
      const int r = it.rb * kRows + gid;
#pragma unroll
      for (int i = 0; i < kD / 8; ++i) qf[i] = 0u;
      if (r < p.rows) {
        const int gi = r / p.queries, i = r - gi * p.queries;
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + it.b * p.q_sb +
                                                          (it.h * p.group + gi) * p.q_sh + i * p.q_ss + c * (kD / 4));
#pragma unroll
        for (int j = 0; j < kD / 32; ++j) {
          const uint4 u = src[j];
          qf[4 * j] = u.x, qf[4 * j + 1] = u.y, qf[4 * j + 2] = u.z, qf[4 * j + 3] = u.w;
        }
      }
      if (p.bf16) {
        // bf16 -> fp16 times a power of two that puts the row's largest value into [2^14, 2^15): exact but for values
        // 2^-28 of the largest and below; the power comes back as a factor of the scores
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < kD / 8; ++i) {
          const float2 f = pair_to_float2<WBK_DT_BF16>(qf[i]);
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
        amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
        const int e = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -100), 127);
        const float up = kv8_pow2(14 - e);
        qfac = kv8_pow2(min(e - 14, 126));
#pragma unroll
        for (int i = 0; i < kD / 8; ++i) {
          const float2 f = pair_to_float2<WBK_DT_BF16>(qf[i]);
          qf[i] = float2_to_pair<WBK_DT_F16>(f.x * up, f.y * up);
        }
      }
    }
    // ---- the columns of this lane's scores, rows 2c and 2c + 1: factor, and how many tokens they see
    float qcol[2];
    int vis[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      qcol[e] = __shfl_sync(~0u, qfac, (2 * c + e) * 4);
      const int r = it.rb * kRows + 2 * c + e, i = r % p.queries;
      // rows beyond the last hide nothing: their results are dropped
      vis[e] = r >= p.rows ? INT_MAX : i >= it.n ? 0 : p.causal ? max(it.len - it.n + i + 1, 0) : it.len;
    }
    const int clear = __reduce_min_sync(~0u, min(vis[0], vis[1]));  // tokens that no row hides

    float o[kMTiles][4];
#pragma unroll
    for (int j = 0; j < kMTiles; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (int t = tile; t < t1; ++t) {
      if (!__all_sync(~0u, tile_wait(&s.full[warp][st], phase, abort_flag, p.timeout_ns))) {
        // Give up: copies in flight land before the CTA ends (this tile's, and those of the stages after it).
        int dummy = 0;
        if (lane == 0) {
          const int left = loader.x - (x + (t - tile));
          for (int i = 0; i < left; ++i) {
            mbar_wait(&s.full[warp][st], phase, &dummy, kDrainNs, KSITE_DRAIN);
            if (++st == p.stages) st = 0, phase ^= 1u;
          }
        }
        return;
      }
      const uint8_t* stage = ring + st * kTileBytes;
      // ---- scores of 32 tokens: group gi holds tokens 16 gi + gid (sc 0, 1) and 16 gi + gid + 8 (sc 2, 3)
      float sc[kGroups][4];
#pragma unroll
      for (int gi = 0; gi < kGroups; ++gi) {
        sc[gi][0] = sc[gi][1] = sc[gi][2] = sc[gi][3] = 0.0f;
#pragma unroll
        for (int h = 0; h < kD / 64; ++h) {
          const uint8_t* at = stage + koff + gi * 16 * kD + (h == 0 ? 0 : khop);
          const uint4 u = lds16(at), v = lds16(at + 8 * kD);
          const uint32_t a[4] = {u.x, u.y, u.z, u.w}, b[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint2 fa = kv8_half4<kFmt>(a[k]), fb = kv8_half4<kFmt>(b[k]);
            const uint32_t frag[4] = {fa.x, fb.x, fa.y, fb.y};
            mma16816(sc[gi], frag, qf[8 * h + 2 * k], qf[8 * h + 2 * k + 1]);
          }
        }
      }
      // ---- x + log2 vs, masked; raise the maximum where a weight would pass 2^8
      float inv[kGroups];  // 0: no tokens there
      bool edge = (t + 1) * kTile > clear;
#pragma unroll
      for (int gi = 0; gi < kGroups; ++gi) {
        const float4 fac = s.factor[warp][st][gi];
        inv[gi] = fac.z;
        edge = edge || fac.z == 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[gi][e] = fmaf(sc[gi][e], fac.x * qcol[e & 1], fac.y);
      }
      if (edge) {
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (inv[gi] == 0.0f || t * kTile + gi * 16 + gid + (e >> 1) * 8 >= vis[e & 1]) sc[gi][e] = -INFINITY;
      }
      float top[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) top[e] = fmaxf(fmaxf(sc[0][e], sc[0][e + 2]), fmaxf(sc[1][e], sc[1][e + 2]));
      if (__any_sync(~0u, top[0] > m[0] + kRaise || top[1] > m[1] + kRaise)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], d));
          const float up = fmaxf(m[e], top[e]);
          const float alpha = up == -INFINITY ? 1.0f : ex2(m[e] - up);
          m[e] = up;
          l[e] *= alpha;
#pragma unroll
          for (int j = 0; j < kMTiles; ++j) o[j][e] *= alpha, o[j][e + 2] *= alpha;
        }
      }
      const float ref[2] = {m[0] == -INFINITY ? 0.0f : m[0] - kKv8Lift, m[1] == -INFINITY ? 0.0f : m[1] - kKv8Lift};
#pragma unroll
      for (int gi = 0; gi < kGroups; ++gi) {
        // ---- weights of 16 tokens, transposed: tokens 2c, 2c + 1 (pb0) and 8 further (pb1) of row gid
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = ex2(sc[gi][e] - ref[e & 1]);
        l[0] = fmaf(w[0] + w[2], inv[gi], l[0]);
        l[1] = fmaf(w[1] + w[3], inv[gi], l[1]);
        const uint32_t pb0 = transpose8x8(float2_to_pair<WBK_DT_F16>(w[0], w[1]));
        const uint32_t pb1 = transpose8x8(float2_to_pair<WBK_DT_F16>(w[2], w[3]));
        // ---- outputs: tokens 2c, 2c + 1 and 8 further, channels gid * kD / 8 ..
        uint32_t va[4][kD / 32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* at = stage + ((i & 1) ? voff1 : voff0) + (gi * 16 + (i >> 1) * 8) * kD;
          if constexpr (kD == 64) {
            const uint2 u = lds8(at);
            va[i][0] = u.x, va[i][1] = u.y;
          } else {
            const uint4 u = lds16(at);
            va[i][0] = u.x, va[i][1] = u.y, va[i][2] = u.z, va[i][3] = u.w;
          }
        }
        if (edge) {  // whatever lies at a place without a token, a weight of 0 has to give 0
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tok = t * kTile + gi * 16 + (i >> 1) * 8 + 2 * c + (kD == 64 ? (i & 1) ^ (c & 1) : i & 1);
            if (inv[gi] == 0.0f || tok >= it.len) {
#pragma unroll
              for (int k = 0; k < kD / 32; ++k) va[i][k] = 0u;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < kD / 32; ++k) {  // bytes of a token pair side by side: channels 4k .. 4k + 3
          const uint2 a01 = kv8_half4<kFmt>(__byte_perm(va[0][k], va[1][k], lo));
          const uint2 b01 = kv8_half4<kFmt>(__byte_perm(va[2][k], va[3][k], lo));
          const uint2 a23 = kv8_half4<kFmt>(__byte_perm(va[0][k], va[1][k], hi));
          const uint2 b23 = kv8_half4<kFmt>(__byte_perm(va[2][k], va[3][k], hi));
          const uint32_t f01[4] = {a01.x, a01.y, b01.x, b01.y}, f23[4] = {a23.x, a23.y, b23.x, b23.y};
          mma16816(o[2 * k], f01, pb0, pb1);
          mma16816(o[2 * k + 1], f23, pb0, pb1);
        }
      }
      __syncwarp();
      if (loader.x < x1) {
        loader.codes<kD>(p, loader.tile, &tmap_k, &tmap_v, ring + st * kTileBytes, &s.full[warp][st]);
        loader.factors(p, loader.tile, s.factor[warp][st]);
        loader.advance(p, 1);
        if (loader.x < x1) loader.look_ahead(p);
        __syncwarp();
      }
      if (++st == p.stages) st = 0, phase ^= 1u;
    }

#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(~0u, l[e], d);

    // ---- the warps and CTAs that this item lies in
    const int begin = x - tile, end = begin + it.tiles, cta = blockIdx.x;
    const int w0 = own.owner(max(begin, c0) - c0), w1 = own.owner(min(end, c1) - 1 - c0);
    const bool split_up = splits(it.tiles, split.q);
    const int first_cta = split_up ? split.owner(begin) : cta, last_cta = split_up ? split.owner(end - 1) : cta;
    const bool alone = w0 == w1, here = first_cta == last_cta;
    const int rows = min(kRows, p.rows - it.rb * kRows);
    const int floats = part_floats(p.part_rows, kD);
    float* part = here ? nullptr : p.parts + (static_cast<int64_t>(cta) * 2 + (first_cta == cta ? 1 : 0)) * floats;
    auto slot_of = [&](int w) {  // a warp's partial result of this item in shared memory
      return slots + (w == 0 ? 0 : w == kWarps - 1 ? kSlots - 1 : 2 * w - (w == w0 ? 0 : 1)) * floats;
    };
    float* mine = alone ? part : slot_of(warp);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rl = 2 * c + e;
      if (rl >= rows) continue;
      if (mine == nullptr) {
        const float invl = l[e] == 0.0f ? 0.0f : 1.0f / l[e];
        uint32_t w[kD / 16];
#pragma unroll
        for (int j = 0; j < kMTiles; ++j)
          w[j] = p.bf16 ? float2_to_pair<WBK_DT_BF16>(o[j][e] * invl, o[j][e + 2] * invl)
                        : float2_to_pair<WBK_DT_F16>(o[j][e] * invl, o[j][e + 2] * invl);
        uint4* dst = reinterpret_cast<uint4*>(out_row(p, it, it.rb * kRows + rl) + gid * (kD / 8));
#pragma unroll
        for (int j = 0; j < kMTiles / 4; ++j) dst[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
      } else {
        float4* dst = reinterpret_cast<float4*>(mine + rl * kD + gid * (kD / 8));
#pragma unroll
        for (int j = 0; j < kMTiles / 2; ++j)
          dst[j] = make_float4(o[2 * j][e], o[2 * j][e + 2], o[2 * j + 1][e], o[2 * j + 1][e + 2]);
        if (gid == 0) mine[p.part_rows * kD + rl] = m[e], mine[p.part_rows * (kD + 1) + rl] = l[e];
      }
    }
    bool holder = alone;  // this warp has the CTA's result of the item
    if (!alone) {
      __threadfence_block();
      __syncwarp();
      uint32_t before = 0;
      if (lane == 0) before = atomicAdd(&s.tickets[w0], 1u);
      holder = __shfl_sync(~0u, before, 0) == static_cast<uint32_t>(w1 - w0);
      if (holder) {
        __threadfence_block();
        join<kD, true>(p, it, [&](int i) { return static_cast<const float*>(slot_of(w0 + i)); }, w1 - w0 + 1, rows, part);
      }
    }
    if (holder && !here) {
      __threadfence();
      __syncwarp();
      uint32_t before = 0;
      if (lane == 0) {
        before = atomicAdd(&p.tickets[first_cta], 1u);
        if (before == static_cast<uint32_t>(last_cta - first_cta)) p.tickets[first_cta] = 0u;
      }
      if (__shfl_sync(~0u, before, 0) == static_cast<uint32_t>(last_cta - first_cta)) {
        __threadfence();
        const float* base = p.parts + static_cast<int64_t>(first_cta) * 2 * floats;
        join<kD, false>(p, it, [&](int i) { return base + (i == 0 ? 1 : 2 * static_cast<int64_t>(i)) * floats; },
                        last_cta - first_cta + 1, rows, nullptr);
      }
    }
    x += t1 - tile;
    tile = 0;
    if (x < x1) next_item(p, it);
  }
}

int step_sms() {
  const int n = sm_count();
  return n > 0 ? n : 148;
}

// How a launch divides an SM: CTAs on it and the stages of a warp's ring, from the
// registers (4 CTAs with head_dim 64, 3 with 128) and the shared memory that
// the partial results of `rows` rows leave. More warps before more stages, but two
// stages at least: one tile is computed on while another is on its way.
struct StepShape {
  int ctas_per_sm, stages;
  size_t smem;
};
StepShape step_shape(int64_t rows, int64_t d) {
  const int part_rows = static_cast<int>(std::min<int64_t>(rows, kRows));
  const size_t fixed = 1024 + sizeof(StepSmem) + static_cast<size_t>(kSlots) * part_floats(part_rows, static_cast<int>(d)) * 4;
  const size_t set = static_cast<size_t>(kWarps) * 2 * kTile * d;
  static_assert(4 <= kKv8TicketsPerSm, "workspace layout");
  for (int ctas = d == 64 ? 4 : 3;; --ctas) {
    const size_t room = 233472 / ctas - 1024;  // 228 KB per SM, 1 KB of it taken by each CTA
    const int stages = room > fixed ? static_cast<int>(std::min<size_t>((room - fixed) / set, kMaxStages)) : 0;
    if (stages >= 2 || ctas == 1) return {ctas, std::max(stages, 1), fixed + std::max(stages, 1) * set};
  }
}

// Two partial results per CTA, behind a ticket per CTA.
int64_t step_ctas(const StepShape& s) { return static_cast<int64_t>(step_sms()) * s.ctas_per_sm; }

// Many rows per KV head go to the kernel of wbk_kv8_prompt.cu, which converts each tile of codes once for up to 256 of
// them; the one here takes time for each 8. us for 24, 32, 48 and 64 rows, here / there: 16 sequences of up to 16384
// tokens, 8 KV heads, head size 64: 125 155 222 287 / 155 for each, head size 128: 186 237 339 453 / 184; 32 of up to
// 512: 28 30 32 34 / 28 and 28 32 39 47 / 35; 2 of up to 4096: 27 26 29 31 / 31 and 28 28 32 35 / 45.
bool prompt_kernel(int64_t group, int64_t queries) { return group <= 128 && group * queries > 32; }

template <int kFmt, int kD>
int launch_step(const CUtensorMap& tk, const CUtensorMap& tv, const Kv8AttnParams& p, int grid, size_t smem,
                cudaStream_t stream) {
  static std::mutex mu;
  static std::vector<char> configured;
  const int dev = current_device();
  if (dev < 0) return fail(WBK_ERR_CUDA, "no current CUDA device");
  {
    std::lock_guard<std::mutex> lock(mu);
    if (static_cast<int>(configured.size()) <= dev) configured.resize(dev + 1, 0);
    if (!configured[dev]) {
      if (int e = cuda_check(cudaFuncSetAttribute(kv8_step_kernel<kFmt, kD>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448),
                             "kv8 attention smem attribute"))
        return e;
      configured[dev] = 1;
    }
  }
  return cuda_check(launch_after(kv8_step_kernel<kFmt, kD>, dim3(grid), kThreads, smem, stream, 1, tk, tv, p), "kv8 attention launch");
}

}  // namespace

int kv8_make_tmap(CUtensorMap* map, const void* base, const Kv8Attention& a, int tile, bool swizzle) {
  auto encode = get_encode_fn();
  if (encode == nullptr) return fail(WBK_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
  const cuuint64_t d = static_cast<cuuint64_t>(a.head_dim), page_rows = static_cast<cuuint64_t>(a.c.kv_heads) * a.c.block;
  const cuuint64_t dims[3] = {d, page_rows, static_cast<cuuint64_t>(a.c.pages)};
  const cuuint64_t strides[2] = {d, page_rows * d};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(d), static_cast<cuuint32_t>(std::min(a.c.block, tile)), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE,
                            !swizzle ? CU_TENSOR_MAP_SWIZZLE_NONE : d == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(WBK_ERR_CUDA, "cuTensorMapEncodeTiled (kv8 pages) failed (%d)", static_cast<int>(r));
  return WBK_OK;
}

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
  const int64_t rows = heads / kv_heads * queries;
  const int64_t ctas = step_ctas(step_shape(rows, head_dim));
  const int64_t step =
      kv8_ticket_bytes() + ctas * 2 * part_floats(static_cast<int>(std::min<int64_t>(rows, kRows)), static_cast<int>(head_dim)) * 4;
  return prompt_kernel(heads / kv_heads, queries) ? std::max(step, kv8_prompt_ws_bytes(head_dim)) : step;
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
  if (!(scale >= 0.0f && scale <= 3.402823466e38f))
    return fail(WBK_ERR_INVALID_ARG, "wbk_attention_kv8: scale %g is negative or not finite", static_cast<double>(scale));
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
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.lens = seq_lens;
  p.q_lens = q_lens;
  p.batch = static_cast<int>(batch);
  p.group = static_cast<int>(heads / kv_heads);
  p.queries = static_cast<int>(queries);
  p.head_dim = static_cast<int>(head_dim);
  p.fmt = fmt;
  p.causal = causal;
  p.bf16 = dtype == WBK_DT_BF16;
  p.scale_log2 = scale * kLog2e;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // queries repeated by a stride of 0 cannot be described to TMA: the few-rows kernel loads them itself
  const bool repeated = (batch > 1 && p.q_sb == 0) || (heads > 1 && p.q_sh == 0) || (queries > 1 && p.q_ss == 0);
  if (prompt_kernel(p.group, queries) && !repeated) return kv8_prompt_attention(p, workspace, st);

  p.rows = p.group * p.queries;
  p.row_blocks = (p.rows + kRows - 1) / kRows;
  p.part_rows = std::min(p.rows, kRows);
  const StepShape shape = step_shape(p.rows, head_dim);
  p.stages = shape.stages;
  p.tickets = static_cast<uint32_t*>(workspace);
  p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kv8_ticket_bytes());
  p.timeout_ns = wait_timeout_ns();
  CUtensorMap tk, tv;
  if (int e = kv8_make_tmap(&tk, k_cache, p, kTile, true)) return e;
  if (int e = kv8_make_tmap(&tv, v_cache, p, kTile, true)) return e;
  // the lengths are on the device: as many CTAs as the table could need, at most what the SMs hold
  const int64_t items = batch * kv_heads * p.row_blocks, most = items * ((max_blocks * block + kTile - 1) / kTile);
  if (most > INT_MAX) return fail(WBK_ERR_UNSUPPORTED, "wbk_attention_kv8: more than 2^31 tiles of 32 tokens in one call");
  const int grid = static_cast<int>(std::min(step_ctas(shape), std::max<int64_t>(most / kMinShare, items)));
  if (fmt == WBK_FMT_E4M3)
    return head_dim == 64 ? launch_step<WBK_FMT_E4M3, 64>(tk, tv, p, grid, shape.smem, st)
                          : launch_step<WBK_FMT_E4M3, 128>(tk, tv, p, grid, shape.smem, st);
  return head_dim == 64 ? launch_step<WBK_FMT_E5M2, 64>(tk, tv, p, grid, shape.smem, st)
                        : launch_step<WBK_FMT_E5M2, 128>(tk, tv, p, grid, shape.smem, st);
}

}  // extern "C"
