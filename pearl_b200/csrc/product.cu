// product.cu -- int8 products with an epilogue: the linear layer
//   C = act(sA[m] * sB[n] * (A . B^T) + bias[n]) + residual
// and the experts' product of a MoE layer, whose rows are grouped by expert
// and multiplied by their expert's weights, with the group boundaries read on
// the device.
//
// A TMA thread fills a ring of 128-byte K stages, a thread issues the tcgen05
// int8 MMAs, and the epilogue warps turn accumulators into C: the grid is
// persistent and the accumulator double-buffered in tensor memory, or, for
// few tiles, each tile's K is split over a cluster (kOnce below).  int32 sums
// are exact; the epilogue works in f32 and rounds once.
//
// What bounds it.  Many rows: the tensor cores under the power cap, and
// beside them the 32 KB a CTA of a 256 x 256 pair tile loads per K block.
// 8192 x 14336 x 4096: 304 us in a burst (3.16 POPS), 356 in a long run at
// 1.32 GHz and 990 W; its MMAs alone 248 and 285, its loads alone 240.  Few
// rows: the weights' bytes (16 slots over 8 experts of 4096 x 14336: 63.5 us,
// 6.5 TB/s).  Few rows and few weights: start, join and end, about 5 us
// (1 x 4096 x 4096: 6.2 us with weights from HBM, whose bytes are 2.6 of them;
// 5.3 from L2).
#include <algorithm>
#include <atomic>
#include <cstring>

#include "pb2_epilogue.cuh"

namespace pb2 {
namespace {

constexpr int kCtaRows = 128;  // rows of C per CTA
constexpr int kTileK = 128;     // bytes of K per stage
// Epilogue warps: a persistent CTA's 16 hide each other's latency (eight took
// 5.7 kclocks for a tile of 128 x 256, twice its MMAs at K = 768); where two
// CTAs share an SM, eight fit.
constexpr int epi_warps(bool once) { return once ? 8 : 16; }
constexpr int product_threads(bool once) { return 32 * (2 + epi_warps(once)); }
constexpr int kMaxStages = 10;
constexpr int kBoxBytes = 32 * 64;  // an epilogue warp's 32 rows x 32 16-bit columns
constexpr int kMaxGroups = 256;

enum { kBiasNone = 0, kBiasF32 = 1, kBiasHalf = 2 };  // kBiasHalf: C's type

// Shared memory for the sums a CTA receives from the other split - 1 ranges.
__host__ __device__ constexpr int received_bytes(int rows, int tile_columns, int split) {
  return rows * tile_columns * 4 / split * (split - 1);
}

struct ProductArgs {
  CUtensorMap tmA;  // A (rows, K) int8, boxes of box_rows rows
  CUtensorMap tmB;  // B (N rows every b_rows, K) int8
  const float* sA;
  const float* sB;
  void* C;
  const void* bias;
  const void* residual;
  int c_f16, c_f32, bias_kind, act;  // C: bf16, f16 or, of groups only, f32
  int M, N, K;
  int tiles_m, tiles_n;    // of the whole product (tiles_m: without groups)
  int groups;              // 0: one product of M rows
  int b_rows;              // rows of B and column scales from one group's to the next's
  const int32_t* ends;     // groups: end row of each group
  const int32_t* c_rows;   // optional: row r of the product goes to row c_rows[r] of C
  int c_dst_rows;
  int tile_rows;           // rows of C per tile
  int box_rows, a_bytes;   // rows of an A load; A bytes of a stage
  int stages;
  int split;               // K ranges, one per CTA (pair) of the cluster
  int early;               // only A and sA come from the kernel before this one (see the start of the kernel)
  int zero_rest;           // groups: rows past the last group's end are zeros in C, not left as they are
  int vec;                 // rows of C and residual can be moved 16 bytes at a time
  SignalSync* sync;
  long long wait_budget;
  uint32_t wait_hint_ns;
};

struct ProductSmem {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t drain;
  uint64_t join;  // kOnce: the other K ranges' sums have arrived
  uint32_t tmem_base;
  int abort_flag;
  int tile0[kMaxGroups + 1];  // first tile of each group
  int row0[kMaxGroups + 1];   // first row of each group
  int tiles_m[kMaxGroups];    // row tiles of each group
  float scale[kCtaRows];      // kOnce: the rows' scales and places in C
  int dst[kCtaRows];
};

struct Tile {
  int group;  // of B and sB
  int row0;   // first row of A
  int rows;   // rows of the group from row0 on (may exceed the tile)
  int tn;
};

// Tile t, asked by a whole warp: groups follow one another; inside one,
// kRaster row tiles walk all column tiles before the next row tiles, so B
// tiles are read by neighbours.  Divisions are kept off the common path (a
// tile of few K blocks is over in 1500 clocks, and so was a binary search
// with four divisions).  8192 x 14336 x 4096 in a long run: 361 us with 16
// row tiles, 374 with 8, 367 with 32, 392 with 4.
constexpr int kRaster = 16;
template <bool kGrouped>
__device__ __forceinline__ Tile tile_at(const ProductArgs& a, const ProductSmem& S, int t) {
  int g = 0, first = 0, rows = a.M, lt = t, tiles_m = a.tiles_m;
  if constexpr (kGrouped) {
    // The last group whose first tile is <= t: by eights, then among eight.
    const int lane = threadIdx.x % 32;
    const bool by8 = 8 * lane < a.groups && S.tile0[8 * lane] <= t;
    const int base = 8 * (__popc(__ballot_sync(0xffffffffu, by8)) - 1);
    const bool by1 = lane < 8 && base + lane < a.groups && S.tile0[base + lane] <= t;
    g = base + __popc(__ballot_sync(0xffffffffu, by1)) - 1;
    first = S.row0[g];
    rows = S.row0[g + 1] - first;
    lt = t - S.tile0[g];
    tiles_m = S.tiles_m[g];
  }
  int m0 = 0, mm = min(kRaster, tiles_m), in = lt;
  if (in >= mm * a.tiles_n) {
    const int block = lt / (kRaster * a.tiles_n);
    m0 = block * kRaster;
    mm = min(kRaster, tiles_m - m0);
    in = lt - block * kRaster * a.tiles_n;
  }
  int tm = 0, tn = in;
  if (mm == kRaster) {
    tn = in / kRaster;
    tm = in % kRaster;
  } else if (mm > 1) {
    tn = in / mm;
    tm = in - tn * mm;
  }
  tm += m0;
  return Tile{g, first + tm * a.tile_rows, rows - tm * a.tile_rows, tn};
}

// The producer and the issuer are single threads whose loops bound short-tile
// products (a K stage of a 128-column tile is 256 clocks of MMA), so they keep
// to 32-bit shared addresses that only step: these are the barrier, TMA and
// MMA instructions on such addresses.
__device__ __forceinline__ bool bar_ready(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A box to `dst`, counted on `bar`; with kPair on the barrier at this offset
// in the pair's leader.
template <bool kPair>
__device__ __forceinline__ void load_box(const CUtensorMap* map, uint32_t bar, uint32_t dst, int x, int y) {
  if constexpr (kPair)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & 0xFEFFFFFFu), "r"(x), "r"(y)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
// One stage of int8 MMAs (128 bytes of K) and its commit; the 2-SM commit
// reaches the barrier in both CTAs of the pair.
template <bool kPair>
__device__ __forceinline__ void umma_i8_stage(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate,
                                              uint32_t bar, uint16_t pair_mask) {
  if constexpr (kPair) {
    umma_i8_2sm(d, ad, bd, idesc, accumulate);
#pragma unroll
    for (int i = 1; i < 4; ++i) umma_i8_2sm(d, ad + 2 * i, bd + 2 * i, idesc, 1);
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(pair_mask)
        : "memory");
  } else {
    umma_i8(d, ad, bd, idesc, accumulate);
#pragma unroll
    for (int i = 1; i < 4; ++i) umma_i8(d, ad + 2 * i, bd + 2 * i, idesc, 1);
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  }
}

// act(sum * row scale * column scale + bias) of 32 columns, cols holding
// {scale, bias} of each.
template <int kAct>
__device__ __forceinline__ void finish(uint32_t* v, float rs, const float2* cols) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const float4 c = *reinterpret_cast<const float4*>(cols + i);  // {scale, bias} of two columns
    v[i] = __float_as_uint(activate<kAct>(fmaf(float(int(v[i])) * rs, c.x, c.y)));
    v[i + 1] = __float_as_uint(activate<kAct>(fmaf(float(int(v[i + 1])) * rs, c.z, c.w)));
  }
}

__device__ __forceinline__ void cp_async16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ int4 ld_int4(const uint8_t* p) { return *reinterpret_cast<const int4*>(p); }
__device__ __forceinline__ int4 add4(int4 a, int4 b) { return make_int4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// `bytes` of this CTA's shared memory to the same place as `to` in the CTA of
// cluster rank `peer`, counted on its barrier `bar`.
__device__ __forceinline__ void copy_to_peer(const void* to, const void* from, uint32_t bytes, const uint64_t* bar, uint32_t peer) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   mapa(to, peer)),
               "r"(smem_u32(from)), "r"(bytes), "r"(mapa(bar, peer))
               : "memory");
}

template <int kAct>
__device__ __forceinline__ void activate8(float* f) {
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = activate<kAct>(f[j]);
}

// Eight 16-bit elements from element `at` on, of which the row has `left`.
__device__ __forceinline__ uint4 load8(const void* base, bool vec, int64_t at, int left) {
  const uint16_t* src = static_cast<const uint16_t*>(base) + at;
  if (vec) return *reinterpret_cast<const uint4*>(src);
  uint32_t e[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) e[j / 2] |= uint32_t(src[j]) << (16 * (j & 1));
  return make_uint4(e[0], e[1], e[2], e[3]);
}
__device__ __forceinline__ void store8(const ProductArgs& a, int64_t at, int left, uint4 val) {
  uint16_t* out = static_cast<uint16_t*>(a.C) + at;
  if (a.vec) {
    *reinterpret_cast<uint4*>(out) = val;
    return;
  }
  const uint32_t w[4] = {val.x, val.y, val.z, val.w};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) out[j] = uint16_t(w[j / 2] >> (16 * (j & 1)));
}
// Four f32 elements.
__device__ __forceinline__ void store4(const ProductArgs& a, int64_t at, int left, uint4 val) {
  uint32_t* out = static_cast<uint32_t*>(a.C) + at;
  if (a.vec) {
    *reinterpret_cast<uint4*>(out) = val;
    return;
  }
  const uint32_t w[4] = {val.x, val.y, val.z, val.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) out[j] = w[j];
}

// Group boundaries to shared memory: row0 and tile0 (exclusive prefix of the
// groups' tiles), by one warp, eight groups a lane.  Ends are clamped to
// [0, M] and made non-decreasing, so no table of boundaries leads outside A.
__device__ __forceinline__ void build_groups(const ProductArgs& a, ProductSmem& S) {
  constexpr int kPer = kMaxGroups / 32;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int end[kPer], tiles[kPer];
    int most = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = lane * kPer + i;
      end[i] = g < a.groups ? min(max(a.ends[g], 0), a.M) : 0;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) end[i] = most = max(most, end[i]);
    int before = most;  // running maximum over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before = max(before, v);
    }
    before = __shfl_up_sync(0xffffffffu, before, 1);
    if (lane == 0) before = 0;
    int sum = 0, begin = before;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      end[i] = max(end[i], before);
      tiles[i] = sum;
      const int tiles_m = (end[i] - begin + a.tile_rows - 1) / a.tile_rows;
      if (lane * kPer + i < a.groups) S.tiles_m[lane * kPer + i] = tiles_m;
      sum += tiles_m * a.tiles_n;
      begin = end[i];
    }
    int total = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, total, o);
      if (lane >= o) total += v;
    }
    const int base = total - sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = lane * kPer + i;
      if (g < a.groups) {
        S.tile0[g] = base + tiles[i];
        S.row0[g + 1] = end[i];
        if (g == a.groups - 1) S.tile0[a.groups] = i + 1 < kPer ? base + tiles[(i + 1) % kPer] : total;
      }
    }
    if (lane == 0) S.row0[0] = 0;
  }
  __syncthreads();
}

// kPair: a tile is worked on by two CTAs (2-SM MMAs, 128 rows of A and half
// of the tile's rows of B each), else by one.
//
// kOnce: for products of few tiles, one tile for each cluster, whose CTAs
// (pairs) take a.split ranges of its K and add their int32 sums up through
// distributed shared memory, each finishing its share of the columns: the
// weights are then read through all SMs.  int32 sums are exact, so C does not
// depend on the split.  Otherwise the grid is persistent and the accumulator double-buffered.
template <bool kPair, int kTN, bool kGrouped, bool kOnce>
__global__ void __launch_bounds__(product_threads(kOnce), kOnce ? 2 : 1) product_kernel(const __grid_constant__ ProductArgs a) {
  constexpr int kCtas = kPair ? 2 : 1;
  constexpr int kBRows = kTN / kCtas;  // rows of B this CTA loads
  constexpr int kBBytes = kBRows * kTileK;
  constexpr int kEpiWarps = epi_warps(kOnce);
  constexpr int kCols = kTN / (kEpiWarps / 4);  // columns of an epilogue warp
  constexpr uint32_t kIdesc = idesc_i8(kCtas * kCtaRows, kTN);
  // An MMA reads kCtaRows rows of A, however few the stage holds (at least
  // eight): the read must end inside the stage.  Pairs always hold them all.
  static_assert(kPair || 8 * kTileK + kBBytes >= kCtaRows * kTileK, "A operand would be read past the stage");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = a.a_bytes + kBBytes;
  uint8_t* boxes = ring + a.stages * stage_bytes;
  float2* col_mem = reinterpret_cast<float2*>(boxes + kEpiWarps * kBoxBytes);
  // kOnce has neither boxes nor column scales, but the sums it receives.
  uint8_t* received = boxes;
  ProductSmem& S = *reinterpret_cast<ProductSmem*>(kOnce ? received + received_bytes(a.a_bytes / kTileK, kTN, a.split)
                                                         : reinterpret_cast<uint8_t*>(col_mem + kEpiWarps * kCols));
  constexpr int kTmemCols = kOnce ? kTN : 2 * kTN;
  volatile int* abort_flag = &S.abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t crank = kPair || kOnce ? cluster_ctarank() : 0;
  const uint32_t rank = kPair ? crank & 1 : 0;  // 0 issues the pair's MMAs
  const uint32_t lead = crank - rank;           // its cluster rank
  const uint16_t pair_mask = uint16_t(0x3u << lead);
  const int split = kOnce ? a.split : 1;
  const int first = blockIdx.x / (kCtas * split), stride = gridDim.x / (kCtas * split);

  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(&S.full[i], 1);
      mbar_init(&S.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.acc_full[i], 1);
      mbar_init(&S.acc_empty[i], kCtas * kEpiWarps);
    }
    mbar_init(&S.drain, 1);
    mbar_init(&S.join, 1);
    S.abort_flag = 0;
    fence_barrier_init();
    tma_prefetch(&a.tmA);
    tma_prefetch(&a.tmB);
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_2sm(&S.tmem_base, kTmemCols);
      tmem_relinquish_2sm();
    } else {
      tmem_alloc(&S.tmem_base, kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  // Every CTA of the cluster runs, its barriers set up, before a remote
  // arrive, copy or 2-SM load.
  if constexpr (kPair || kOnce) cluster_sync_all();
  tc_fence_after();
  const int kblocks = (a.K + kTileK - 1) / kTileK;
  const int range = kOnce ? int(crank) / kCtas : 0;
  const int kb0 = range * kblocks / split, kb1 = (range + 1) * kblocks / split;
  if constexpr (kOnce && !kGrouped) {
    // The previous kernel is still running: ask L2 for the first stages of B
    // (a prefetch is coherent with whatever that kernel writes).
    if (warp == 0 && lane == 0) {
      const Tile w = tile_at<false>(a, S, first);
      for (int kb = kb0; kb < min(kb1, kb0 + a.stages); ++kb)
        tma_prefetch_l2_2d(&a.tmB, kb * kTileK, w.tn * kTN + int(rank) * kBRows);
    }
  }
  // Programmatic dependent launch: with a.early everything but A and sA was
  // complete before the kernel before this one could let it start (that
  // kernel waits for its own predecessors first), so the groups and the first
  // stages of B are read while it is still running.
  if (!kGrouped || !a.early) griddep_wait();
  griddep_launch_dependents();
  if constexpr (kGrouped) build_groups(a, S);
  const uint32_t tmem = S.tmem_base;
  const int tiles = kGrouped ? S.tile0[a.groups] : a.tiles_m * a.tiles_n;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    // The warp finds each tile; one thread issues its loads.
    const bool leader = elect_one();
    bool ok = true;
    const uint32_t full0 = smem_u32(S.full), empty0 = smem_u32(S.empty), ring0 = smem_u32(ring);
    const uint32_t past = 8 * a.stages;
    uint32_t at = 0, dst = ring0, phase = 1;  // of the stage: barrier offset, address, wait parity
    const int box_bytes = a.box_rows * kTileK;
    bool early = kGrouped && a.early;
    for (int t = first; t < tiles; t += stride) {
      const Tile w = tile_at<kGrouped>(a, S, t);
      if (leader && ok) {
        const int arow = w.row0 + int(rank) * kCtaRows;
        const int brow = w.group * a.b_rows + w.tn * kTN + int(rank) * kBRows;
        // Only loads of A with rows of this tile: the rest of the stage keeps
        // what it held, and rows past the tile's are never stored.
        auto boxes_of = [&](int r) {
          return (min(max(w.rows - r * kCtaRows, 0), min(kCtaRows, a.tile_rows)) + a.box_rows - 1) / a.box_rows;
        };
        const int mine = boxes_of(rank);
        const int bytes = kCtas * kBBytes + (boxes_of(0) + (kPair ? boxes_of(1) : 0)) * box_bytes;
        const int x1 = kb1 * kTileK;
        int x = kb0 * kTileK;
        auto load_a = [&](uint32_t bar, uint32_t to, int k) {
          if (mine == 1) {
            load_box<kPair>(&a.tmA, bar, to, k, arow);
          } else {
            for (int i = 0; i < mine; ++i) load_box<kPair>(&a.tmA, bar, to + i * box_bytes, k, arow + i * a.box_rows);
          }
        };
        if (kGrouped && early) {  // the ring is empty: B of its first round, then the wait, then A
          early = false;
          const int n = min(a.stages, kb1 - kb0);
          for (int i = 0; i < n; ++i) {
            if (rank == 0) bar_expect(full0 + 8 * i, bytes);
            load_box<kPair>(&a.tmB, full0 + 8 * i, ring0 + i * stage_bytes + a.a_bytes, x + i * kTileK, brow);
          }
          griddep_wait();
          for (int i = 0; i < n; ++i) load_a(full0 + 8 * i, ring0 + i * stage_bytes, x + i * kTileK);
          x += n * kTileK;
          at = 8 * n;
          dst = ring0 + n * stage_bytes;
          if (at == past) { at = 0; dst = ring0; phase ^= 1; }
        }
        for (; x < x1; x += kTileK) {
          if (!bar_ready(empty0 + at, phase) &&
              !(ok = mbar_wait(&S.empty[at / 8], phase, abort_flag, a.sync, a.wait_budget, a.wait_hint_ns)))
            break;
          // The pair leader's barrier counts both CTAs' bytes.
          if (rank == 0) bar_expect(full0 + at, bytes);
          load_box<kPair>(&a.tmB, full0 + at, dst + a.a_bytes, x, brow);
          load_a(full0 + at, dst, x);
          at += 8;
          dst += stage_bytes;
          if (at == past) { at = 0; dst = ring0; phase ^= 1; }
        }
      }
      __syncwarp();
    }
    if (leader) {
      // Every load in flight has landed and been consumed before the CTA ends
      // (bounded).  The next wait of each stage in turn is for just that; on a
      // stage that was never filled it returns at once.
      for (int i = 0; i < a.stages; ++i) {
        const long long t0 = clock64();
        while (!bar_ready(empty0 + at, phase) && clock64() - t0 < 100000000LL) {
        }
        at += 8;
        if (at == past) { at = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (the pair's leader)
    if (rank == 0 && elect_one()) {
      bool ok = true;
      int n = 0;
      const uint32_t full0 = smem_u32(S.full), empty0 = smem_u32(S.empty);
      const uint32_t past = 8 * a.stages;
      const uint64_t desc0 = sdesc_sw128(smem_u32(ring));  // address field: the low 14 bits, in 16 bytes
      const uint32_t step = stage_bytes >> 4, b_off = a.a_bytes >> 4;
      uint32_t at = 0, phase = 0;
      uint64_t ad = desc0;
      for (int t = first; t < tiles && ok; t += stride, ++n) {
        const int slot = n & 1;
        if (!(ok = mbar_wait(&S.acc_empty[slot], ((n >> 1) & 1) ^ 1, abort_flag, a.sync, a.wait_budget, a.wait_hint_ns)))
          break;
        tc_fence_after();
        const uint32_t d = tmem + slot * kTN;
        uint32_t accumulate = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!bar_ready(full0 + at, phase) &&
              !(ok = mbar_wait(&S.full[at / 8], phase, abort_flag, a.sync, a.wait_budget, a.wait_hint_ns)))
            break;
          tc_fence_after();
          umma_i8_stage<kPair>(d, ad, ad + b_off, kIdesc, accumulate, empty0 + at, pair_mask);
          accumulate = 1;
          at += 8;
          ad += step;
          if (at == past) { at = 0; ad = desc0; phase ^= 1; }
        }
        if (ok) {
          if constexpr (kPair) umma_commit_2sm(&S.acc_full[slot], pair_mask);
          else umma_commit(&S.acc_full[slot]);
        }
      }
      // Every MMA has retired before TMEM is released.
      if constexpr (kPair) umma_commit_2sm(&S.drain, uint16_t(1u << lead));
      else umma_commit(&S.drain);
      const long long t0 = clock64();
      while (!mbar_test(&S.drain, 0) && clock64() - t0 < 100000000LL) {
      }
    }
    __syncwarp();
  } else if constexpr (!kOnce) {
    // ------------------------------------------------------------ epilogue
    // Warp: TMEM lane quadrant q (32 rows), strip h of the tile's columns.
    const int q = warp & 3, ew = warp - 2, h = ew >> 2;
    uint8_t* box = boxes + ew * kBoxBytes;
    float2* cols = col_mem + ew * kCols;
    const bool f16 = a.c_f16;
    const int q0 = int(rank) * kCtaRows + 32 * q;  // the warp's first row in the tile
    const uint32_t leader_empty = kPair ? mapa(&S.acc_empty[0], lead) : 0;
    auto release = [&](int slot) {  // the warp's loads of the accumulator have completed (wait::ld)
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair) mbar_arrive_relaxed_cluster(leader_empty + 8 * slot);
        else mbar_arrive(&S.acc_empty[slot]);
      }
    };
    // What a tile needs beside its accumulator: the row's scale and place in
    // C (lane = row) and the columns' scales and biases.  Loaded a tile ahead:
    // with short K the round trip to memory would otherwise be most of a
    // tile's time.
    struct Meta {
      int tn;
      bool live;  // this warp has something to store
      float rs;
      int dst;
      float2 col[kCols / 32];
    };
    auto load_meta = [&](int t) {
      Meta m;
      m.live = false;
      m.tn = 0;
      m.rs = 0.f;
      m.dst = -1;
#pragma unroll
      for (int j = 0; j < kCols / 32; ++j) m.col[j] = make_float2(0.f, 0.f);
      if (t >= tiles) return m;
      const Tile w = tile_at<kGrouped>(a, S, t);
      m.tn = w.tn;
      const int c0 = w.tn * kTN + h * kCols;
      const int rows = min(w.rows, a.tile_rows);
      m.live = q0 < rows && c0 < a.N;
      if (!m.live) return m;
      if (q0 + lane < rows) {
        const int r = w.row0 + q0 + lane;
        m.rs = a.sA[r];
        m.dst = kGrouped && a.c_rows ? a.c_rows[r] : r;
      }
#pragma unroll
      for (int j = 0; j < kCols / 32; ++j) {
        const int c = c0 + 32 * j + lane;
        if (c < a.N) {
          m.col[j].x = a.sB[int64_t(w.group) * a.b_rows + c];
          if (!kGrouped && a.bias_kind)
            m.col[j].y = a.bias_kind == kBiasF32 ? static_cast<const float*>(a.bias)[c] : half_at(a.bias, c, f16);
        }
      }
      return m;
    };
    // Four lanes move one 64-byte row of a 32-column chunk, eight rows an
    // instruction, so loads of the residual and stores of C are whole sectors.
    // Rows change hands through the warp's box (16-byte piece j of row r at
    // j ^ (r / 2 % 4): no bank conflicts either way), into which the residual
    // is copied asynchronously while the accumulator is still being computed.
    const int piece = lane & 3, sub = lane >> 2;
    auto place = [&](int row, int j) { return box + row * 64 + ((j ^ ((row >> 1) & 3)) << 4); };
    bool ok = true;
    int n = 0;
    if (kGrouped && a.early) griddep_wait();
    Meta next = load_meta(first);
    for (int t = first; t < tiles && ok; t += stride, ++n) {
      const Meta m = next;
      const int slot = n & 1;
      const int c0 = m.tn * kTN + h * kCols;
      int dst[4];  // the rows of C this lane moves pieces of
      {
        const int mine = !kGrouped || m.dst < a.c_dst_rows ? m.dst : -1;
#pragma unroll
        for (int it = 0; it < 4; ++it) dst[it] = __shfl_sync(0xffffffffu, mine, 8 * it + sub);
      }
      auto fetch_residual = [&](int ch) {
        const int col = c0 + 32 * ch + 8 * piece;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          if (dst[it] >= 0 && col < a.N) {
            uint8_t* to = place(8 * it + sub, piece);
            const int64_t at = int64_t(dst[it]) * a.N + col;
            if (a.vec)
              cp_async16(to, static_cast<const uint16_t*>(a.residual) + at);
            else
              *reinterpret_cast<uint4*>(to) = load8(a.residual, false, at, a.N - col);
          }
        }
      };
      if (m.live) {
#pragma unroll
        for (int j = 0; j < kCols / 32; ++j) cols[32 * j + lane] = m.col[j];
        __syncwarp();
        if (!kGrouped && a.residual) fetch_residual(0);
      }
      next = load_meta(t + stride);
      if (!(ok = mbar_wait_warp(&S.acc_full[slot], (n >> 1) & 1, abort_flag, a.sync, a.wait_budget, a.wait_hint_ns)))
        break;
      tc_fence_after();
      const uint32_t taddr = tmem + slot * kTN + (uint32_t(32 * q) << 16) + h * kCols;
      if (!m.live) {
        release(slot);
        continue;
      }
#pragma unroll 1
      for (int ch = 0; ch < kCols / 32; ++ch) {
        uint32_t v[32];
        __syncwarp();
        tmem_ld32(taddr + 32 * ch, v);
        tmem_wait_ld_into(v);
        if (ch == kCols / 32 - 1) release(slot);  // the accumulator is free for the tile after next
        const float2* cc = cols + 32 * ch;
        switch (kGrouped ? PB2_ACT_NONE : a.act) {
          case PB2_ACT_RELU: finish<PB2_ACT_RELU>(v, m.rs, cc); break;
          case PB2_ACT_SILU: finish<PB2_ACT_SILU>(v, m.rs, cc); break;
          case PB2_ACT_GELU: finish<PB2_ACT_GELU>(v, m.rs, cc); break;
          case PB2_ACT_GELU_TANH: finish<PB2_ACT_GELU_TANH>(v, m.rs, cc); break;
          default: finish<PB2_ACT_NONE>(v, m.rs, cc);
        }
        if (!kGrouped && a.residual) {
          cp_async_wait();
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 r = *reinterpret_cast<const uint4*>(place(lane, j));
            const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              const float2 f = unpack_half2(rw[p], f16);
              v[8 * j + 2 * p] = __float_as_uint(__uint_as_float(v[8 * j + 2 * p]) + f.x);
              v[8 * j + 2 * p + 1] = __float_as_uint(__uint_as_float(v[8 * j + 2 * p + 1]) + f.y);
            }
          }
          __syncwarp();
        }
        if (kGrouped && a.c_f32) {
#pragma unroll
          for (int part = 0; part < 2; ++part) {  // 16 columns are a box's 64-byte rows
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<uint4*>(place(lane, j)) =
                  make_uint4(v[16 * part + 4 * j], v[16 * part + 4 * j + 1], v[16 * part + 4 * j + 2], v[16 * part + 4 * j + 3]);
            __syncwarp();
            const int col = c0 + 32 * ch + 16 * part + 4 * piece;
#pragma unroll
            for (int it = 0; it < 4; ++it) {
              const uint4 val = *reinterpret_cast<const uint4*>(place(8 * it + sub, piece));
              if (dst[it] >= 0 && col < a.N) store4(a, int64_t(dst[it]) * a.N + col, a.N - col, val);
            }
            __syncwarp();
          }
          continue;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t o[4];
#pragma unroll
          for (int p = 0; p < 4; ++p)
            o[p] = pack_half2(__uint_as_float(v[8 * j + 2 * p]), __uint_as_float(v[8 * j + 2 * p + 1]), f16);
          *reinterpret_cast<uint4*>(place(lane, j)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        __syncwarp();
        uint4 out[4];
#pragma unroll
        for (int it = 0; it < 4; ++it) out[it] = *reinterpret_cast<const uint4*>(place(8 * it + sub, piece));
        const int col = c0 + 32 * ch + 8 * piece;
        if (col < a.N) {
#pragma unroll
          for (int it = 0; it < 4; ++it)
            if (dst[it] >= 0) store8(a, int64_t(dst[it]) * a.N + col, a.N - col, out[it]);
        }
        __syncwarp();
        if (!kGrouped && a.residual && ch + 1 < kCols / 32) fetch_residual(ch + 1);
      }
    }
  }
  if constexpr (kOnce) {
    // ------------------------------------------------------------ join of the K ranges
    // A CTA finishes kTN / split of the tile's columns.  Its accumulator goes
    // to its own ring (idle by now) as [finisher][row][columns] int32, 16-byte
    // piece j of a row at j ^ (row & 7); one bulk copy a finisher takes its
    // share over, and the sums are local when the copies have arrived.  (With
    // a remote load per row, range and piece instead: 32 x 4096 x 4096 6.1 |
    // 6.9 us, 128 x 4096 x 14336 16.4 | 17.9, in pairs 256 x 4096 x 14336
    // 18.6 | 18.3, whose ring then has two stages more.)
    const bool has = first < tiles;
    const Tile w = has ? tile_at<kGrouped>(a, S, first) : Tile{0, 0, 0, 0};
    const int live = has ? min(max(min(w.rows, a.tile_rows) - int(rank) * kCtaRows, 0), kCtaRows) : 0;
    const bool f16 = a.c_f16;
    const int width = kTN / split, pieces = width / 8;  // 64 or 32 columns
    // A thread keeps its piece of eight columns over all its rows.
    const int et = threadIdx.x - 64, step = 32 * kEpiWarps / pieces;
    const int rows = a.a_bytes / kTileK;      // of a CTA's tile
    const uint32_t share = live * width * 4;  // bytes of a finisher's columns from one range
    const int r0 = et / pieces, lc = range * width + (et - r0 * pieces) * 8;
    const int col = w.tn * kTN + lc;
    const bool cols_in = et >= 0 && has && col < a.N;
    float sb[8], bias[8];
    auto load_residual = [&](int r) {
      const int dst = r < live && cols_in ? S.dst[r] : -1;
      return dst >= 0 ? load8(a.residual, a.vec, int64_t(dst) * a.N + col, a.N - col) : make_uint4(0u, 0u, 0u, 0u);
    };
    uint4 res;
    if (warp >= 2) {
      if (kGrouped && a.early) griddep_wait();
      // What does not wait for the products: scales, places, the residual.
      if (et < live) {
        const int row = w.row0 + int(rank) * kCtaRows + et;
        S.scale[et] = a.sA[row];
        int dst = row;
        if (kGrouped && a.c_rows) dst = a.c_rows[row] < a.c_dst_rows ? a.c_rows[row] : -1;
        S.dst[et] = dst;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sb[j] = bias[j] = 0.f;
      if (cols_in) {
        const float* p = a.sB + int64_t(w.group) * a.b_rows + col;
        if (a.vec) {
          *reinterpret_cast<float4*>(sb) = *reinterpret_cast<const float4*>(p);
          *reinterpret_cast<float4*>(sb + 4) = *reinterpret_cast<const float4*>(p + 4);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (col + j < a.N) sb[j] = p[j];
        }
        if (!kGrouped && a.bias_kind == kBiasF32) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (col + j < a.N) bias[j] = static_cast<const float*>(a.bias)[col + j];
        } else if (!kGrouped && a.bias_kind) {
          const uint4 u = load8(a.bias, a.vec, col, a.N - col);
          const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 g = unpack_half2(uw[j], f16);
            bias[2 * j] = g.x;
            bias[2 * j + 1] = g.y;
          }
        }
      }
      if (et == 0 && live > 0) mbar_arrive_expect_tx(&S.join, (split - 1) * share);
      named_barrier_sync(1, 32 * kEpiWarps);  // S.scale and S.dst are in
      if (!kGrouped && a.residual) {
        // The first row's residual, and the others' to L2, from where a load a
        // row ahead is in time (from HBM a round of four waited 1600 clocks,
        // 850 now; all of them in registers: 1 to 4% slower where rows are few).
        res = load_residual(r0);
        if (cols_in)
          for (int r = r0 + step; r < live; r += step)
            prefetch_l2(static_cast<const uint16_t*>(a.residual) + int64_t(S.dst[r]) * a.N + col);
      }
      const int q = warp & 3, h = (warp - 2) >> 2;
      const bool ok = has && mbar_wait_warp(&S.acc_full[0], 0, abort_flag, a.sync, a.wait_budget, a.wait_hint_ns);
      tc_fence_after();
      if (ok && 32 * q < live) {
#pragma unroll 1
        for (int ch = 0; ch < kCols / 32; ++ch) {
          uint32_t v[32];
          __syncwarp();
          tmem_ld32(tmem + (uint32_t(32 * q) << 16) + h * kCols + 32 * ch, v);
          tmem_wait_ld_into(v);
          const int r = 32 * q + lane;
          if (r < live) {
            const int c = h * kCols + 32 * ch, owner = c / width;  // width >= 32: a chunk has one finisher
            const int j0 = (c - owner * width) / 4;
            uint4* row = reinterpret_cast<uint4*>(ring + (owner * rows + r) * width * 4);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              row[(j0 + j) ^ (r & 7)] = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
        }
        fence_proxy_async_smem();
      }
      named_barrier_sync(1, 32 * kEpiWarps);
      if (live > 0 && !__any_sync(0xffffffffu, *abort_flag)) {
        if (et < split && et != range)  // the finisher keeps the other ranges' sums in their order
          copy_to_peer(received + (range - int(range > et)) * rows * width * 4, ring + et * rows * width * 4, share, &S.join,
                       et * kCtas + rank);
        mbar_wait_warp(&S.join, 0, abort_flag, a.sync, a.wait_budget, a.wait_hint_ns);
      }
      if (et == 0 && live > 0 && *abort_flag) {  // given up: no copy may still be on its way when the CTA ends (bounded)
        const long long t0 = clock64();
        while (!mbar_test(&S.join, 0) && clock64() - t0 < 100000000LL) {
        }
      }
    }
    if (cols_in && !*abort_flag) {
      const int own = range * rows * width * 4;
      // With 64 columns the upper half of a row's threads take their two pieces
      // in the other order: eight threads' loads then meet all banks once
      // (with the ranges' loads in flight together: 256 x 4096 x 14336 with a
      // residual 19.5 us, 21.0 before both and the prefetch).
      const int p4 = (lc - range * width) / 4, turn = (p4 >> 3) & 1;
      for (int r = r0; r < live; r += step) {
        const int dst = S.dst[r];
        const int x_at = r * width * 4 + (((p4 + turn) ^ (r & 7)) << 4), y_at = r * width * 4 + (((p4 + 1 - turn) ^ (r & 7)) << 4);
        int4 x = ld_int4(ring + own + x_at), y = ld_int4(ring + own + y_at);
        // split is 2 or 4: the loads of two ranges in flight.
        const int4 x1 = ld_int4(received + x_at), y1 = ld_int4(received + y_at);
        if (split == 4) {
          const uint8_t* more = received + rows * width * 4;
          const int4 x2 = ld_int4(more + x_at), y2 = ld_int4(more + y_at);
          const int4 x3 = ld_int4(more + rows * width * 4 + x_at), y3 = ld_int4(more + rows * width * 4 + y_at);
          x = add4(x, add4(x2, x3));
          y = add4(y, add4(y2, y3));
        }
        x = add4(x, x1);
        y = add4(y, y1);
        const int4 lo = turn ? y : x, hi = turn ? x : y;
        const int acc[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        const uint4 mine = res;
        if (!kGrouped && a.residual) res = load_residual(r + step);
        if (dst < 0) continue;
        const float rs = S.scale[r];
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = fmaf(float(acc[j]) * rs, sb[j], bias[j]);
        if constexpr (!kGrouped) {
          switch (a.act) {
            case PB2_ACT_RELU: activate8<PB2_ACT_RELU>(f); break;
            case PB2_ACT_SILU: activate8<PB2_ACT_SILU>(f); break;
            case PB2_ACT_GELU: activate8<PB2_ACT_GELU>(f); break;
            case PB2_ACT_GELU_TANH: activate8<PB2_ACT_GELU_TANH>(f); break;
            default: break;
          }
          if (a.residual) {
            const uint32_t rw[4] = {mine.x, mine.y, mine.z, mine.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 g = unpack_half2(rw[j], f16);
              f[2 * j] += g.x;
              f[2 * j + 1] += g.y;
            }
          }
        }
        if (kGrouped && a.c_f32) {
#pragma unroll
          for (int j = 0; j < 8; j += 4)
            if (col + j < a.N)
              store4(a, int64_t(dst) * a.N + col + j, a.N - col - j,
                     make_uint4(__float_as_uint(f[j]), __float_as_uint(f[j + 1]), __float_as_uint(f[j + 2]),
                                __float_as_uint(f[j + 3])));
          continue;
        }
        store8(a, int64_t(dst) * a.N + col, a.N - col,
               make_uint4(pack_half2(f[0], f[1], f16), pack_half2(f[2], f[3], f16), pack_half2(f[4], f[5], f16),
                          pack_half2(f[6], f[7], f16)));
      }
    }
  }
  if constexpr (kGrouped) {
    // Rows of no group (their expert is on another GPU): zeros, 16 bytes a
    // thread where rows allow it.  The kernel before may still read them.
    if (a.early) griddep_wait();
    for (int r = (a.zero_rest ? S.row0[a.groups] : a.M) + int(blockIdx.x); r < a.M; r += int(gridDim.x)) {
      const int dst = a.c_rows ? a.c_rows[r] : r;
      if (uint32_t(dst) >= uint32_t(a.c_dst_rows)) continue;
      const int size = a.c_f32 ? 4 : 2;
      uint8_t* row = static_cast<uint8_t*>(a.C) + int64_t(dst) * a.N * size;
      if (a.vec) {
        for (int64_t i = 16 * threadIdx.x; i < int64_t(a.N) * size; i += 16 * blockDim.x)
          *reinterpret_cast<uint4*>(row + i) = make_uint4(0u, 0u, 0u, 0u);
      } else {
        for (int64_t i = 2 * threadIdx.x; i < int64_t(a.N) * size; i += 2 * blockDim.x)
          *reinterpret_cast<uint16_t*>(row + i) = 0;
      }
    }
  }
  // No CTA leaves while another of its cluster can still address its
  // barriers, tensor memory or sums.
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair || kOnce) cluster_sync_all();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    if constexpr (kPair) tmem_dealloc_2sm(tmem, kTmemCols);
    else tmem_dealloc(tmem, kTmemCols);
  }
}

// ------------------------------------------------------------------ host
bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// CTA pairs of this kernel that can be resident at once (SM pairs of one GPC).
// Asked once a device and kernel; threads that ask together get the same.
int resident_pairs(std::atomic<int>& cached, int device, const void* kern, int smem) {
  int n = cached.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2, 1, 1);
    cfg.blockDim = dim3(product_threads(false), 1, 1);
    cfg.dynamicSmemBytes = size_t(smem);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) != cudaSuccess || clusters <= 0) {
      cudaGetLastError();
      clusters = std::max(1, sm_count(device) / 2);
    }
    n = clusters;
    cached.store(n, std::memory_order_relaxed);
  }
  return n;
}

// Shared memory of a CTA that leaves room for another on its SM: for short K
// ranges, so that the set-up of one product overlaps the end of the one before
// it (weights from HBM, half an SM | a full ring: 1 x 4096 x 4096 in ranges of
// 8 blocks 6.2 | 7.4 us, 16 x 2048 x 8192 in ranges of 16 8.4 | 8.2, 32 x 4096
// x 14336 in ranges of 28 15.5 | 13.7).  Tiles of more than 32 rows leave such
// a ring too few stages beside the sums they receive.
constexpr int kHalfSm = 115712;

template <bool kPair, int kTN, bool kGrouped, bool kOnce>
int launch_product(ProductArgs& a, const int8_t* A, const int8_t* B, int cta_rows, int device, cudaStream_t s) {
  constexpr int kCtas = kPair ? 2 : 1;
  constexpr int kBRows = kTN / kCtas;
  a.a_bytes = cta_rows * kTileK;
  a.tile_rows = kCtas * cta_rows;
  a.tiles_m = int((int64_t(a.M) + a.tile_rows - 1) / a.tile_rows);
  a.tiles_n = (a.N + kTN - 1) / kTN;
  int st;
  if ((st = make_tmap_2d(&a.tmA, A, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.M, kTileK, a.box_rows,
                         CU_TENSOR_MAP_SWIZZLE_128B)) ||
      (st = make_tmap_2d(&a.tmB, B, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, uint64_t(std::max(a.groups, 1) - 1) * a.b_rows + a.N,
                         kTileK, kBRows, CU_TENSOR_MAP_SWIZZLE_128B)))
    return st;
  const int fixed = 1024 + int(sizeof(ProductSmem)) +
                    (kOnce ? received_bytes(cta_rows, kTN, a.split) : epi_warps(false) * kBoxBytes + 4 * kTN * 8);
  const bool half = kOnce && cta_rows <= 32 && (a.K + kTileK - 1) / kTileK <= 8 * a.split;
  a.stages = std::min(kMaxStages, ((half ? kHalfSm : 232448) - fixed) / (a.a_bytes + kBRows * kTileK));
  // Whole loads of A in a stage, and with kOnce a tile's sums in the ring.
  if (cta_rows % a.box_rows || cta_rows > kCtaRows || (kPair && cta_rows != kCtaRows) ||
      (kOnce && ((a.split != 2 && a.split != 4) ||
                 cta_rows * kTN * 4 > a.stages * (a.a_bytes + kBRows * kTileK))))
    return PB2_ERR_UNSUPPORTED_CONFIG;
  a.wait_budget = wait_budget_cycles();
  a.wait_hint_ns = suspend_hint_ns(a.wait_budget);
  const int smem = fixed + a.stages * (a.a_bytes + kBRows * kTileK);
  auto kern = product_kernel<kPair, kTN, kGrouped, kOnce>;
  static std::atomic<bool> allowed[64];  // the attribute holds for the process: set once a device
  if (!allowed[device & 63].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess) return launch_status();
    allowed[device & 63].store(true, std::memory_order_relaxed);
  }
  // Row tiles: exact without groups; with them, whose sizes only the device
  // knows, at most one ragged tile a group beyond the whole ones.
  const int64_t tiles_m = kGrouped ? int64_t(a.M) / a.tile_rows + std::min(a.groups, a.M)
                                   : (int64_t(a.M) + a.tile_rows - 1) / a.tile_rows;
  int64_t clusters = tiles_m * a.tiles_n;
  if (clusters > INT32_MAX / 8) return PB2_ERR_INVALID_ARGUMENT;
  if (!kOnce) {
    static std::atomic<int> pairs[64];
    const int most = kPair ? resident_pairs(pairs[device & 63], device, reinterpret_cast<const void*>(kern), smem)
                           : std::max(1, sm_count(device));
    clusters = std::min<int64_t>(clusters, most);
  }
  const int cluster = kCtas * (kOnce ? a.split : 1);
  return launch_programmatic(kern, dim3(unsigned(clusters * cluster)), product_threads(kOnce), smem, s, cluster, a);
}

// The variant for a product is the one with the smallest estimate of its
// time, in us: a start and end, and for each K block of a CTA's tiles what a
// stage of that tile takes.  Fitted to products of 1 to 2048 rows, 300 to
// 14336 columns and 304 to 16384 of K with weights from HBM; the variant it
// takes was within 5% of the fastest for all 37 of them.
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int run_linear(ProductArgs& a, const int8_t* A, const int8_t* B, int device, cudaStream_t s) {
  const int64_t sms = std::max(1, sm_count(device)), pairs = std::max<int64_t>(1, sms / 2);
  const int64_t kblocks = ceil_div(a.K, kTileK), m = a.M, n = a.N;
  enum { kWide, kPairs, kSingle } kind = kSingle;
  double best = 1e30;
  int cta_rows = kCtaRows;
  auto offer = [&](double us, int k, int rows, int split) {
    if (us >= best) return;
    best = us;
    kind = static_cast<decltype(kind)>(k);
    cta_rows = rows;
    a.split = split;
  };
  // Persistent pairs with tiles of 256 x 256 and 256 x 128 (1024 x 4096 x
  // 4096: 18.7 | 19.5, single CTAs 20.7; 512 x 4096 x 14336: 41 | 28 | 32), or
  // with 256 x 128 and K in two ranges (256 x 4096 x 14336: 19, unsplit 25,
  // single CTAs with two ranges 21).
  if (m > kCtaRows) {
    offer(7.0 + 0.33 * double(ceil_div(ceil_div(m, 256) * ceil_div(n, 256), pairs) * kblocks), kWide, kCtaRows, 1);
    const int64_t tiles = ceil_div(m, 256) * ceil_div(n, 128);
    offer(5.0 + 0.20 * double(ceil_div(tiles, pairs) * kblocks), kPairs, kCtaRows, 1);
    if (tiles * 2 <= pairs && kblocks >= 4) offer(7.5 + 0.20 * double(ceil_div(kblocks, 2)), kPairs, kCtaRows, 2);
  }
  // Single CTAs.  Tiles of fewer rows start and end sooner and occupy more
  // SMs (200 x 2048 x 2048: 6.5 with 32 rows, 7.6 with 128; 200 x 1001 x 1040,
  // whose odd rows are stored in pieces: 6.2 | 14.5).  K is split over a
  // cluster of two or four CTAs (of eight, most have to wait for a second
  // round) while every one has an SM (1 x 4096 x 4096: 6.2, unsplit 9.0;
  // 100 x 1000 x 1008 with 32 rows: 4.8 | 5.3; 128 x 300 x 16384: 9.8 | 25).
  for (int rows = 32; rows <= kCtaRows; rows *= 2) {
    const int r = int(std::min<int64_t>(rows, ceil_div(m, 8) * 8));
    const int64_t tiles = ceil_div(m, r) * ceil_div(n, 128);
    const double block = 0.176 + 0.0005 * r;
    offer(3.85 + 0.002 * r + block * double(ceil_div(tiles, sms) * kblocks), kSingle, r, 1);
    for (int split = 2; split <= 4 && tiles * split <= sms && kblocks >= 2 * split; split *= 2)
      offer(3.2 + 0.024 * r + 0.0056 * double(tiles * split) + block * double(ceil_div(kblocks, split)), kSingle, r, split);
    if (r >= m) break;
  }
  a.box_rows = cta_rows;
  if (a.split > 1) {
    if (kind == kPairs) return launch_product<true, 128, false, true>(a, A, B, cta_rows, device, s);
    return launch_product<false, 128, false, true>(a, A, B, cta_rows, device, s);
  }
  if (kind == kSingle) return launch_product<false, 128, false, false>(a, A, B, cta_rows, device, s);
  if (kind == kPairs) return launch_product<true, 128, false, false>(a, A, B, cta_rows, device, s);
  return launch_product<true, 256, false, false>(a, A, B, cta_rows, device, s);
}

int run_grouped(ProductArgs& a, const int8_t* A, const int8_t* B, int device, cudaStream_t s) {
  const int64_t sms = std::max(1, sm_count(device));
  const int64_t kblocks = ceil_div(a.K, kTileK), average = a.M / a.groups;
  a.split = 1;
  // Groups of more rows than a CTA's tile: pairs (16 groups of 256 rows,
  // 4096 x 4096: 85, single CTAs 94; of 128 rows 64, single CTAs 62).
  if (average > kCtaRows + kCtaRows / 4) {
    a.box_rows = kCtaRows;
    return launch_product<true, 256, true, false>(a, A, B, kCtaRows, device, s);
  }
  // The weights bound what is left: a stage holds no more rows of A than
  // groups of this size need, so that more of it is weights in flight (60
  // groups of 22 rows: 34 with 64 rows a stage, 38 with 128).
  int cta_rows = average <= 16 ? 32 : average <= 64 ? 64 : kCtaRows;
  cta_rows = int(std::min<int64_t>(cta_rows, ceil_div(a.M, 8) * 8));
  a.box_rows = std::min(cta_rows, 32);
  cta_rows = int(ceil_div(cta_rows, a.box_rows)) * a.box_rows;
  const int64_t used = std::min<int64_t>(a.groups, a.M);
  const int64_t tiles_m = used + a.M / (2 * cta_rows);  // about
  const int64_t narrow = tiles_m * ceil_div(a.N, 128), broad = tiles_m * ceil_div(a.N, 256);
  while (narrow * 2 * a.split <= sms && 2 * a.split <= 4 && kblocks / (2 * a.split) >= 4) a.split *= 2;
  if (a.split > 1) return launch_product<false, 128, true, true>(a, A, B, cta_rows, device, s);
  // 128 columns a tile, or 256 with half the loads of A (128 groups of 128
  // rows: 63 | 55; 20 groups of one row or two, 2048 x 1408: 14.3 | 15.6).
  const double full = cta_rows == kCtaRows ? 1.0 : 0.9;
  if (0.22 * full * double(ceil_div(narrow, sms)) < 0.32 * double(ceil_div(broad, sms)))
    return launch_product<false, 128, true, false>(a, A, B, cta_rows, device, s);
  return launch_product<false, 256, true, false>(a, A, B, cta_rows, device, s);
}

// out[t] = residual[t] + sum_j w[t, j] * slots[t * top_k + j], f32 sums in
// slot order.  HBM-bound (4 top_k + 4 bytes a column of f32 slots, 2 top_k + 4
// of 16-bit ones): a block per token and 256 vectors of eight columns,
// kCombineBatch slots' loads in flight at a time with the residual's.  8192
// tokens of two slots of 4096: 67 us (6.0 TB/s), of bf16 slots 44 (6.1 TB/s;
// slot by slot 72, two vectors a thread 72).
struct CombineArgs {
  const void* slots;
  const float* weights;
  const void* residual;
  void* out;
  int top_k, n, f16, vec;
  int64_t out_n;  // columns from one row of residual and out to the next
  int round_f16;  // f32 slots: rounded to f16 where it holds them
};
constexpr int kCombineBatch = 4;
// Eight columns of a slot.
struct Eight {
  uint4 lo, hi;  // hi: of f32 slots
};

template <bool kSlotF32>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t t = blockIdx.x;
  const int col = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  if (col >= a.n) return;
  const int left = a.n - col;
  const bool f16 = a.f16;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  auto load_slot = [&](int64_t row) {
    Eight e;
    if constexpr (kSlotF32) {
      const uint32_t* p = static_cast<const uint32_t*>(a.slots) + row * a.n + col;
      if (a.vec) {
        e.lo = *reinterpret_cast<const uint4*>(p);
        e.hi = *reinterpret_cast<const uint4*>(p + 4);
      } else {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = j < left ? p[j] : 0u;
        e.lo = make_uint4(w[0], w[1], w[2], w[3]);
        e.hi = make_uint4(w[4], w[5], w[6], w[7]);
      }
    } else {
      e.lo = load8(a.slots, a.vec, row * a.n + col, left);
    }
    return e;
  };
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto add16 = [&](uint4 r, float w) {
    const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack_half2(rw[j], f16);
      acc[2 * j] = fmaf(w, f.x, acc[2 * j]);
      acc[2 * j + 1] = fmaf(w, f.y, acc[2 * j + 1]);
    }
  };
  auto add = [&](const Eight& e, float w) {
    if constexpr (kSlotF32) {
      const uint32_t x[8] = {e.lo.x, e.lo.y, e.lo.z, e.lo.w, e.hi.x, e.hi.y, e.hi.z, e.hi.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float v = __uint_as_float(x[j]);
        if (a.round_f16) {
          const float h = __half2float(__float2half_rn(v));
          v = isinf(h) ? v : h;
        }
        acc[j] = fmaf(w, v, acc[j]);
      }
    } else {
      add16(e.lo, w);
    }
  };
  const uint4 res = a.residual ? load8(a.residual, a.vec, t * a.out_n + col, left) : zero;
  for (int j0 = 0; j0 < a.top_k; j0 += kCombineBatch) {
    Eight r[kCombineBatch];
    float w[kCombineBatch];
#pragma unroll
    for (int j = 0; j < kCombineBatch; ++j) {
      const bool in = j0 + j < a.top_k;
      if (in) r[j] = load_slot(t * a.top_k + j0 + j);
      w[j] = in ? a.weights[t * a.top_k + j0 + j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kCombineBatch; ++j)
      if (w[j] != 0.f) add(r[j], w[j]);  // whatever a slot without weight holds does not count
  }
  if (a.residual) add16(res, 1.0f);
  uint16_t* o = static_cast<uint16_t*>(a.out) + t * a.out_n + col;
  if (a.vec) {
    *reinterpret_cast<uint4*>(o) = make_uint4(pack_half2(acc[0], acc[1], f16), pack_half2(acc[2], acc[3], f16),
                                              pack_half2(acc[4], acc[5], f16), pack_half2(acc[6], acc[7], f16));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) o[j] = half_bits(acc[j], f16);
  }
}

// Between its product and its combination gated_experts holds the slots'
// products in f32, so that a result is rounded once: of all columns where the
// workspace has room for them, else of half of them at a time (as many bytes
// as 16-bit products of all columns).  2048 tokens of 128 experts, 134 MB of
// f32: 103 us, in halves 112, with bf16 products 79 and 1.4 times the error
// against 64 bits; 8192 tokens of 8 wide experts 1038 | 1072 | 1002.
//
// f16 outputs of more than 32 MB of products keep the values that they have
// always had, those of gemm_grouped into f16 and combine_slots: each product
// is rounded to f16's eleven bits before its weight.  Held in f32, one beyond
// 65504 stays what it is: in f16 it was infinite, and so was its sum, however
// small its weight.
constexpr int64_t kSlotBytes = 32 << 20;
bool slots_fit(int64_t slots, int64_t hidden) { return slots * hidden * 4 <= kSlotBytes; }
int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }
// Workspace of f32 products of `columns` columns, and the least it may be.
int64_t workspace_bytes(int64_t slots, int64_t inner, int64_t columns) {
  return round256(slots * inner) + round256(slots * 4) + round256(slots * columns * 4);
}
int64_t least_columns(int64_t slots, int64_t hidden) {
  return slots_fit(slots, hidden) ? hidden : std::min(hidden, ((hidden + 1) / 2 + 7) / 8 * 8);
}

bool type16(int t) { return t == PB2_TYPE_BF16 || t == PB2_TYPE_F16; }

}  // namespace
}  // namespace pb2

extern "C" int pb2_gemm_epilogue(const pb2_gemm_epilogue_params* pp, void* stream) {
  pb2::NvtxRange nvtx_range("pb2_gemm_epilogue");
  using namespace pb2;
  if (!pp) return PB2_ERR_INVALID_ARGUMENT;
  const pb2_gemm_epilogue_params& p = *pp;
  if (p.m < 0 || p.n <= 0 || p.k <= 0 || p.m > INT32_MAX || p.n > INT32_MAX || p.k > INT32_MAX)
    return PB2_ERR_INVALID_ARGUMENT;
  if (!type16(p.c_type) || p.activation < PB2_ACT_NONE || p.activation > PB2_ACT_GELU_TANH)
    return PB2_ERR_INVALID_ARGUMENT;
  if (p.bias && p.bias_type != PB2_TYPE_F32 && p.bias_type != p.c_type) return PB2_ERR_INVALID_ARGUMENT;
  if (p.k % 16 != 0) return PB2_ERR_UNSUPPORTED_CONFIG;  // 16-byte rows of A and B
  if (p.m > 0 && (!p.A || !p.B || !p.A_scales || !p.B_scales || !p.C || !al16(p.A) || !al16(p.B)))
    return PB2_ERR_INVALID_ARGUMENT;
  int st = set_device(p.device);
  if (st) return st;
  if (p.m == 0) return PB2_OK;
  ProductArgs a;
  std::memset(&a, 0, sizeof(a));
  a.sA = p.A_scales;
  a.sB = p.B_scales;
  a.C = p.C;
  a.bias = p.bias;
  a.bias_kind = !p.bias ? kBiasNone : p.bias_type == PB2_TYPE_F32 ? kBiasF32 : kBiasHalf;
  a.residual = p.residual;
  a.c_f16 = p.c_type == PB2_TYPE_F16;
  a.act = p.activation;
  a.M = int(p.m);
  a.N = a.b_rows = int(p.n);
  a.K = int(p.k);
  a.vec = p.n % 8 == 0 && al16(p.C) && al16(p.residual) && al16(p.B_scales) && al16(p.bias);
  a.sync = static_cast<SignalSync*>(p.host_signal_sync);
  return run_linear(a, p.A, p.B, p.device, static_cast<cudaStream_t>(stream));
}

namespace pb2 {
// `b_rows`, `early`, `zero_rest`: see ProductArgs.
int gemm_grouped(const pb2_gemm_grouped_params& p, int64_t b_rows, bool early, bool zero_rest, cudaStream_t stream) {
  if (p.m < 0 || p.n <= 0 || p.k <= 0 || p.m > INT32_MAX || p.k > INT32_MAX) return PB2_ERR_INVALID_ARGUMENT;
  if (p.num_experts <= 0 || p.num_experts > kMaxGroups || b_rows > INT32_MAX / p.num_experts) return PB2_ERR_INVALID_ARGUMENT;
  if (!type16(p.c_type) && p.c_type != PB2_TYPE_F32) return PB2_ERR_INVALID_ARGUMENT;
  if (p.k % 16 != 0) return PB2_ERR_UNSUPPORTED_CONFIG;
  if (p.c_row_index && p.c_rows < 0) return PB2_ERR_INVALID_ARGUMENT;
  if (p.m > 0 && (!p.A || !p.B || !p.A_scales || !p.B_scales || !p.C || !p.routing_offsets || !al16(p.A) || !al16(p.B)))
    return PB2_ERR_INVALID_ARGUMENT;
  int st = set_device(p.device);
  if (st) return st;
  if (p.m == 0) return PB2_OK;
  ProductArgs a;
  std::memset(&a, 0, sizeof(a));
  a.sA = p.A_scales;
  a.sB = p.B_scales;
  a.C = p.C;
  a.c_f16 = p.c_type == PB2_TYPE_F16;
  a.c_f32 = p.c_type == PB2_TYPE_F32;
  a.M = int(p.m);
  a.N = int(p.n);
  a.b_rows = int(b_rows);
  a.K = int(p.k);
  a.groups = int(p.num_experts);
  a.ends = p.routing_offsets;
  a.c_rows = p.c_row_index;
  a.c_dst_rows = int(std::min<int64_t>(p.c_row_index ? p.c_rows : p.m, INT32_MAX));
  a.vec = p.n % 8 == 0 && b_rows % 8 == 0 && al16(p.C) && al16(p.B_scales);
  a.sync = static_cast<SignalSync*>(p.host_signal_sync);
  a.early = early;
  a.zero_rest = zero_rest;
  return run_grouped(a, p.A, p.B, p.device, stream);
}
}  // namespace pb2

extern "C" int pb2_gemm_grouped(const pb2_gemm_grouped_params* pp, void* stream) {
  pb2::NvtxRange nvtx_range("pb2_gemm_grouped");
  if (!pp) return PB2_ERR_INVALID_ARGUMENT;
  return pb2::gemm_grouped(*pp, pp->n, false, false, static_cast<cudaStream_t>(stream));
}

namespace pb2 {
// `out_n`, `round_f16`: see CombineArgs.
int combine(const pb2_combine_params& p, int64_t out_n, bool round_f16, cudaStream_t s) {
  if (p.num_tokens < 0 || p.top_k <= 0 || p.n <= 0 || p.num_tokens > INT32_MAX || p.top_k > INT32_MAX || p.n > INT32_MAX)
    return PB2_ERR_INVALID_ARGUMENT;
  if (!type16(p.type) || (p.slots_type != p.type && p.slots_type != PB2_TYPE_F32)) return PB2_ERR_INVALID_ARGUMENT;
  if (p.num_tokens > 0 && (!p.slots || !p.topk_weights || !p.out)) return PB2_ERR_INVALID_ARGUMENT;
  const int64_t vectors = (p.n + 7) / 8, threads = std::min<int64_t>(256, (vectors + 31) / 32 * 32);
  const int64_t across = (vectors + threads - 1) / threads;
  if (across > 65535) return PB2_ERR_INVALID_ARGUMENT;
  int st = set_device(p.device);
  if (st) return st;
  if (p.num_tokens == 0) return PB2_OK;
  CombineArgs a;
  a.slots = p.slots;
  a.weights = p.topk_weights;
  a.residual = p.residual;
  a.out = p.out;
  a.top_k = int(p.top_k);
  a.n = int(p.n);
  a.f16 = p.type == PB2_TYPE_F16;
  a.out_n = out_n;
  a.round_f16 = round_f16;
  a.vec = p.n % 8 == 0 && out_n % 8 == 0 && al16(p.slots) && al16(p.out) && al16(p.residual);
  const dim3 grid(unsigned(p.num_tokens), static_cast<unsigned>(across));
  if (p.slots_type == PB2_TYPE_F32) return launch_programmatic(combine_kernel<true>, grid, int(threads), 0, s, 1, a);
  return launch_programmatic(combine_kernel<false>, grid, int(threads), 0, s, 1, a);
}
}  // namespace pb2

extern "C" int pb2_combine_slots(const pb2_combine_params* pp, void* stream) {
  pb2::NvtxRange nvtx_range("pb2_combine_slots");
  if (!pp) return PB2_ERR_INVALID_ARGUMENT;
  return pb2::combine(*pp, pp->n, false, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t pb2_gated_experts_workspace_bytes(int64_t slots, int64_t inner, int64_t hidden) {
  if (slots <= 0 || inner <= 0 || hidden <= 0) return 0;
  return pb2::workspace_bytes(slots, inner, pb2::least_columns(slots, hidden));
}

extern "C" int pb2_gated_experts(const pb2_gated_experts_params* pp, void* stream) {
  pb2::NvtxRange nvtx_range("pb2_gated_experts");
  using namespace pb2;
  if (!pp) return PB2_ERR_INVALID_ARGUMENT;
  const pb2_gated_experts_params& p = *pp;
  if (p.num_tokens < 0 || p.top_k <= 0 || p.inner <= 0 || p.hidden <= 0 || p.top_k > INT32_MAX ||
      p.num_tokens > INT32_MAX / p.top_k)
    return PB2_ERR_INVALID_ARGUMENT;
  const int64_t slots = p.num_tokens * p.top_k;
  if (slots > 0 && (!p.workspace || !al16(p.workspace) ||
                    p.workspace_bytes < pb2_gated_experts_workspace_bytes(slots, p.inner, p.hidden) || !p.slot_indices))
    return PB2_ERR_INVALID_ARGUMENT;
  uint8_t* ws = static_cast<uint8_t*>(p.workspace);
  pb2_gated_quant_params q;
  std::memset(&q, 0, sizeof(q));
  q.device = p.device;
  q.x = p.x;
  q.x_type = p.type;
  q.m = q.x_rows = slots;
  q.n = p.inner;
  q.activation = p.activation;
  q.row_index = p.slot_indices;
  q.smooth = p.smooth;
  q.xq = reinterpret_cast<int8_t*>(ws);
  q.scales = reinterpret_cast<float*>(ws + round256(slots * p.inner));
  q.max_val = p.max_val;
  q.block_size = p.block_size;
  pb2_gemm_grouped_params g;
  std::memset(&g, 0, sizeof(g));
  g.device = p.device;
  g.m = slots;
  g.k = p.inner;
  g.A = q.xq;
  g.A_scales = q.scales;
  g.C = ws + round256(slots * p.inner) + round256(slots * 4);
  g.c_type = PB2_TYPE_F32;
  g.num_experts = p.num_experts;
  g.routing_offsets = p.routing_offsets;
  g.c_row_index = p.slot_indices;
  g.c_rows = slots;
  g.host_signal_sync = p.host_signal_sync;
  pb2_combine_params c;
  std::memset(&c, 0, sizeof(c));
  c.device = p.device;
  c.slots = g.C;
  c.slots_type = g.c_type;
  c.topk_weights = p.topk_weights;
  c.type = p.type;
  c.num_tokens = p.num_tokens;
  c.top_k = p.top_k;
  // The later steps' arguments before any step is queued.
  if (!type16(p.type) || p.num_experts <= 0 || p.num_experts > kMaxGroups || p.hidden > INT32_MAX / p.num_experts ||
      p.inner > INT32_MAX || (slots > 0 && (!p.w || !al16(p.w) || !p.w_scales || !p.routing_offsets || !p.topk_weights || !p.out)))
    return PB2_ERR_INVALID_ARGUMENT;
  if (p.inner % 16 != 0) return PB2_ERR_UNSUPPORTED_CONFIG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool whole = p.workspace_bytes >= workspace_bytes(slots, p.inner, p.hidden);
  const int64_t step = whole ? p.hidden : least_columns(slots, p.hidden);
  int st = pb2_quantize_gated(&q, stream);
  for (int64_t at = 0; at < p.hidden && !st; at += step) {
    g.n = c.n = std::min(step, p.hidden - at);
    g.B = p.w + at * p.inner;
    g.B_scales = p.w_scales + at;
    c.residual = p.residual ? static_cast<const uint16_t*>(p.residual) + at : nullptr;
    c.out = static_cast<uint16_t*>(p.out) + at;
    // The quantizer writes A and its scales; weights and routing are older.
    // The combination reads every slot, also those of no expert.
    st = gemm_grouped(g, p.hidden, true, true, s);
    if (!st) st = combine(c, p.hidden, p.type == PB2_TYPE_F16 && !slots_fit(slots, p.hidden), s);
  }
  return st;
}
