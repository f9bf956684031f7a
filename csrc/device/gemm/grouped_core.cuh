// Products of ragged groups of rows on the tcgen05 tensor cores: each group of rows with the weights of its expert.
//
//   FORWARD   y[t, n]     = sum over k of x[t, k] w[e, n, k]          e: the group of row t
//   DATA      dx[t, k]    = sum over n of dy[t, n] w[e, n, k]
//   WEIGHT    dw[e, n, k] = sum over the rows t of group e of dy[t, n] x[t, k]
//
// The groups are given by their ends on the device; the host knows only the number of rows.  Every CTA reads the ends, lays the
// tiles of all groups end to end and takes every gridDim-th of them.  A tile is 128 rows of ONE group (or of one expert's weights)
// by BN columns: the rows of a tile that belong to the next group are loaded and multiplied like any others and not stored, so a
// group's last tile costs a whole one (half a tile a group on average; nothing is padded or copied).
//
// The operands lie in memory as the model keeps them, so some have the contracted dimension inside (K-major, one box of 64
// elements x rows) and some outside (MN-major, boxes of 64 columns x 64 contracted rows); the matrix descriptors say which, and
// nothing is transposed.  In WEIGHT the contracted dimension is the ragged one: the rows of the last block behind the
// group's end are cleared in shared memory before the tensor core reads them (they may hold anything, and 0 x Inf is no zero).
//
//   warp 0      TMA producer
//   warp 1      issues the MMAs (one thread); clears the rows behind a group's end
//   warp 2      allocates and frees tensor memory
//   warps 4-11  epilogue: four lane quarters x two halves of the columns
// Every wait is bounded; a role that gives up records it, all roles leave, and what is in flight ends before the CTA does (drainLoads and
// drainProducts).  No counterpart in the reference.
#pragma once

#include <cuda_bf16.h>

#include "gemm_core.cuh"

namespace mccl {
namespace grouped {

using gemm::BM;
constexpr int kThreads = 384, kEpiWarps = 8, kMaxGroups = 1024;
constexpr int kStageBytes = 2048;      // shared memory of an epilogue warp
constexpr int kStageK = 128;           // bytes of the contracted dimension a stage holds, one swizzled row: 64 bf16
enum Mode { FORWARD = 0, DATA = 1, WEIGHT = 2 };

struct Args {
  CUtensorMap mapA;                    // FORWARD / DATA: x or dy [T, contracted], box 64 x 128; WEIGHT: dy [T, N], box 64 x 64
  CUtensorMap mapB;                    // FORWARD: w [E, N, K], box 64 x BN; DATA: the same, box 64 x 64; WEIGHT: x [T, K], box 64 x 64
  CUtensorMap mapC;                    // the output: [T, width], box 32 x 32; WEIGHT: [E, N, K], box 32 x 32 x 1, WHOLE 64 x 32 x 1
  const void* ends;                    // [groups] int32 or int64
  int ends64, groups;
  int rows;                            // T
  int contracted;                      // FORWARD: K, DATA: N
  int tileRows, width;                 // WEIGHT: N (rows of an expert's output); columns of the output
  __nv_bfloat16* out;                  // [T, width], or WEIGHT: [E, tileRows, width]
  int* errFlag;
  uint64_t budgetNs, blockNs;          // how long a wait may take, and a block of a contraction that one covers
};

template <int BN, bool WHOLE> struct Smem {
  static constexpr int A_BYTES = BM * kStageK, B_BYTES = BN * kStageK;
  // WHOLE: a stage less, for an epilogue that has a warp's whole part of a tile in shared memory (storeWhole).
  static constexpr int STAGES = BN == 256 ? (WHOLE ? 3 : 4) : (WHOLE ? 5 : 6);
  static constexpr int TILE_BYTES = STAGES * (A_BYTES + B_BYTES);
  static constexpr int EPI_BYTES = WHOLE ? 32 * BN : kStageBytes;                    // a warp: 32 rows x BN / 2 columns of bf16
  static constexpr int TABLE_BYTES = 2 * (kMaxGroups + 4) * 4;
  static constexpr int TOTAL = TILE_BYTES + kEpiWarps * EPI_BYTES + TABLE_BYTES + 256 + 1024;
};

// The two products of a backward pass read the same dy and need nothing of each other: the second is launched with programmatic stream
// serialization, so that its CTAs start on the SMs that the first one's last wave leaves free.  It waits for the first one's end before
// its own, which then stands for both.
__device__ __forceinline__ void letNextStart() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void waitForPrevious() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// MN-major bf16 tile written by TMA with the 128-byte swizzle: chunks of 64 columns, each 64 contracted rows of 128 bytes.
// Leading byte offset = distance of two chunks, stride byte offset = distance of two groups of eight contracted rows.
__device__ __forceinline__ uint64_t smemDescMn(const void* tile) {
  uint64_t d = 0;
  d |= (uint64_t)((umma::smemAddr(tile) & 0x3ffff) >> 4);
  d |= (uint64_t)(8192 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void tmaLoad3d(void* smemDst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      :: "r"(umma::smemAddr(smemDst)), "l"(map), "r"(umma::smemAddr(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

// Stores of a box from shared memory; elements outside the tensor are left out.
__device__ __forceinline__ void tmaStore3d(const CUtensorMap* map, const void* smemSrc, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
               :: "l"(map), "r"(umma::smemAddr(smemSrc)), "r"(x), "r"(y), "r"(z) : "memory");
}

// After a wait has run out the roles leave their loops with loads and products in flight, which end before the CTA's shared and tensor memory
// are another's: the loads by the barriers they complete on, the products (and copies of scales) by a commit of the thread that issued
// them.  With a limit of their own.
constexpr uint64_t kDrainNs = 1000000000ull;
// The last loads of `loads` stages in all, one after another.
__device__ __forceinline__ void drainLoads(uint64_t* full, uint32_t stages, uint32_t loads) {
  for (uint32_t i = loads > stages ? loads - stages : 0; i < loads; ++i)
    if (!umma::mbarWait(&full[i % stages], i / stages & 1, kDrainNs)) return;
}
// The warp that issued them; its elected thread is the same one every time.
__device__ __forceinline__ void drainProducts(uint64_t* drained) {
  if (umma::electOne()) {
    umma::mmaCommit(drained);
    umma::mbarWait(drained, 0, kDrainNs);
  }
}

// The groups as every role sees them: group e holds the rows [start[e], start[e + 1]); the tiles of all groups up to e number
// prefix[e + 1].  Ends that fall or lie outside the rows are read as the largest so far, within [0, T]: no access depends on them.
struct Groups {
  int* start;
  int* prefix;
};

// One warp.  `perRowTile`: column tiles of one row tile, or WEIGHT (rowTile 0): tiles of an expert.
__device__ __forceinline__ void readGroups(const Groups& g, const void* ends, int ends64, int groups, int T, int rowTile, int perRowTile, int lane) {
  int last = 0, tiles = 0;
  if (lane == 0) { g.start[0] = 0; g.prefix[0] = 0; }
  if (ends == nullptr) {                                   // one group of all rows
    if (lane == 0) { g.start[1] = T; g.prefix[1] = (T + rowTile - 1) / rowTile * perRowTile; }
    return;
  }
  // Eight rounds' ends are asked for at a time (1024 groups: one round after another 40 us a product, so 35 us, by halves below 15 us).
  constexpr int ROUNDS = 8;
  for (int base = 0; base < groups; base += 32 * ROUNDS) {
    int v[ROUNDS];
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
      const int e = base + 32 * u + lane;
      int64_t w = 0;
      if (e < groups) w = ends64 ? static_cast<const int64_t*>(ends)[e] : (int64_t) static_cast<const int32_t*>(ends)[e];
      v[u] = (int)(w < 0 ? 0 : w > T ? T : w);
    }
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
      if (base + 32 * u >= groups) break;
      const int e = base + 32 * u + lane;
      int end = v[u];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int w = __shfl_up_sync(0xffffffffu, end, o); if (lane >= o && w > end) end = w; }
      if (end < last) end = last;
      int begin = __shfl_up_sync(0xffffffffu, end, 1);
      if (lane == 0) begin = last;
      int n = e < groups ? (rowTile == 0 ? perRowTile : (end - begin + rowTile - 1) / rowTile * perRowTile) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int w = __shfl_up_sync(0xffffffffu, n, o); if (lane >= o) n += w; }
      if (e < groups) { g.start[e + 1] = end; g.prefix[e + 1] = tiles + n; }
      last = __shfl_sync(0xffffffffu, end, 31);
      tiles += __shfl_sync(0xffffffffu, n, 31);
    }
  }
}

// The group of tile t, from that of an earlier tile on; by halves, as many groups may have no rows (1024 of them one by one: 20 us).
__device__ __forceinline__ int groupOf(const Groups& g, int t, int e, int groups) {
  if (t < g.prefix[e + 1]) return e;
  int lo = e + 1, hi = groups - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (t < g.prefix[mid + 1]) hi = mid; else lo = mid + 1;
  }
  return lo;
}
// Tile t of all, which is one of group e: its first row and first column.  The tiles of a group go panel by panel of eight row tiles, the row
// fastest, so that what runs at a time shares a few weight tiles.
struct Tile { int e, row, col; };
__device__ __forceinline__ void tileAt(const Groups& g, int t, int e, int rowTiles, int colTiles, int rowStep, int colStep, Tile* out) {
  const int l = t - g.prefix[e];
  const int p = l / (8 * colTiles), within = l - p * 8 * colTiles, in = min(8, rowTiles - 8 * p);
  out->e = e;
  out->row = (p * 8 + within % in) * rowStep;
  out->col = (within / in) * colStep;
}

// A wait of a whole warp: all its lanes get the same answer, so that they leave a loop together.  False where it took too long, or
// where another role has given up.
template <bool PARKED>
__device__ __forceinline__ bool waitWarp(uint64_t* bar, uint32_t parity, uint64_t budget, volatile int* sFail) {
  bool ok = *sFail == 0;
  if (ok) ok = PARKED ? umma::mbarWaitParked(bar, parity, budget) : umma::mbarWait(bar, parity, budget);
  if (__all_sync(0xffffffffu, ok)) return true;
  *sFail = 1;
  return false;
}

// The same for a wait that covers `blocks` blocks of contractions, whose limit grows with them: a long one is no kernel that stands still.  It sees
// within a microsecond that another role has given up.
__device__ __forceinline__ bool waitWarpLong(uint64_t* bar, uint32_t parity, uint64_t budget, uint64_t blocks, uint64_t blockNs, volatile int* sFail) {
  const uint64_t limit = budget + blocks * blockNs;
  uint64_t t0 = 0;
  bool ok = false;
  for (uint32_t spins = 0; *sFail == 0; ++spins) {
    if (umma::mbarTryWaitParked(bar, parity)) { ok = true; break; }
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    if (spins == 0) t0 = t;
    else if (t - t0 > limit) break;
  }
  if (__all_sync(0xffffffffu, ok)) return true;
  *sFail = 1;
  return false;
}

// The epilogue of a warp: 32 rows (lane: row) x COLS sums as bf16, 32 columns at a time through 2 KB of shared memory, whose 16-byte pieces are
// swizzled over the rows (as a tensor map's 64-byte swizzle does: no bank is hit twice).  Whole sets of 32 rows leave by TMA; a group's last
// rows, up to `rows`, by stores of four lanes to 64 bytes of a row.  The epilogue runs beside the next tile's products and is what bounds short
// contractions: 64 experts of 128 rows, dw of 2048 x 1024, a store from where the sums are, a row per lane, 133 us; all through shared memory and
// lanes 72 us; by TMA 70 us.  16 experts of 512 rows, y of 512 x 2048: 36 and 35 us.
template <int COLS>
__device__ __forceinline__ void storeTile(const uint32_t* v, uint8_t* stage, const CUtensorMap* map, int x, int y, int z, __nv_bfloat16* out, int rows, int width,
                                          int lane) {
  if (rows <= 0) return;
  const bool byTma = z >= 0 || rows >= 32;
#pragma unroll
  for (int c = 0; c < COLS / 32; ++c) {
    if (x + 32 * c >= width) break;
    if (lane == 0) umma::tmaStoreWaitRead<0>();            // what left this memory before has been read
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 o;
      __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o2[i] = __floats2bfloat162_rn(__uint_as_float(v[32 * c + 8 * j + 2 * i]), __uint_as_float(v[32 * c + 8 * j + 2 * i + 1]));
      *reinterpret_cast<uint4*>(stage + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = o;
    }
    if (byTma) {
      umma::fenceProxyAsyncShared();
      __syncwarp();
      if (lane == 0) {
        if (z >= 0) tmaStore3d(map, stage, x + 32 * c, y, z); else umma::tmaStore2d(map, stage, x + 32 * c, y);
        umma::tmaStoreCommit();
      }
    } else {
      __syncwarp();
      const int col = x + 32 * c + (lane & 3) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 2);
        const uint4 o = *reinterpret_cast<const uint4*>(stage + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
        if (r < rows && col < width) *reinterpret_cast<uint4*>(out + (size_t)r * width + col) = o;
      }
    }
  }
}
// The same for the gradient of the weights of experts with few rows, whose contraction is one block: all COLS columns in shared memory at a time, one
// wait, one fence and a box of 64 columns or two in place of four of each, for one stage less.  32 experts of 2048 x 5504 with two rows each
// 143 -> 126 us, 64 of 520 x 776 with 47 rows 31 -> 28 us; but with 128 rows each (1024 x 2048) 69 -> 75 us, 16 with 512 rows 39 -> 45 us.
template <int COLS>
__device__ __forceinline__ void storeWhole(const uint32_t* v, uint8_t* stage, const CUtensorMap* map, int x, int y, int z, int rows, int width, int lane) {
  if (rows <= 0 || x >= width) return;
  if (lane == 0) umma::tmaStoreWaitRead<0>();
  __syncwarp();
#pragma unroll
  for (int j = 0; j < COLS / 8; ++j) {
    uint4 o;
    __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) o2[i] = __floats2bfloat162_rn(__uint_as_float(v[8 * j + 2 * i]), __uint_as_float(v[8 * j + 2 * i + 1]));
    *reinterpret_cast<uint4*>(stage + j / 8 * 4096 + lane * 128 + (((j & 7) ^ (lane & 7)) << 4)) = o;
  }
  umma::fenceProxyAsyncShared();
  __syncwarp();
  if (lane == 0) {
#pragma unroll
    for (int b = 0; b < COLS / 64; ++b)
      if (x + 64 * b < width) tmaStore3d(map, stage + b * 4096, x + 64 * b, y, z);
    umma::tmaStoreCommit();
  }
}

// Zeros in a warp's 32 rows x COLS columns.
template <int COLS>
__device__ __forceinline__ void clearTile(__nv_bfloat16* out, int rows, int col0, int width, int lane) {
  constexpr int PER = COLS / 8;                            // lanes a row
  const int col = col0 + lane % PER * 8;
#pragma unroll 4
  for (int r = lane / PER; r < 32; r += 32 / PER)
    if (r < rows && col < width) *reinterpret_cast<uint4*>(out + (size_t)r * width + col) = make_uint4(0, 0, 0, 0);
}
// The epilogue warps' share of the rows behind the last group, which belong to nobody.
__device__ __forceinline__ void clearRows(__nv_bfloat16* out, int from, int to, int width) {
  const int64_t lo = (int64_t)from * width / 8, hi = (int64_t)to * width / 8;
  for (int64_t i = lo + (int64_t)blockIdx.x * (kEpiWarps * 32) + (threadIdx.x - 128); i < hi; i += (int64_t)gridDim.x * (kEpiWarps * 32))
    reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
}

template <int BN, int MODE, bool WHOLE>
__global__ void __launch_bounds__(kThreads, 1) groupedKernel(const __grid_constant__ Args a) {
  static_assert(!WHOLE || MODE == WEIGHT, "storeWhole leaves the rows behind an expert's last out by the tensor map");
  using S = Smem<BN, WHOLE>;
  constexpr int ST = S::STAGES;
  constexpr int CK = 64;                                   // contracted elements a stage
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sB = smem + ST * S::A_BYTES;
  uint8_t* sStage = smem + S::TILE_BYTES;
  int* table = reinterpret_cast<int*>(sStage + kEpiWarps * S::EPI_BYTES);
  const Groups g{table, table + kMaxGroups + 4};
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(table) + S::TABLE_BYTES);
  uint64_t* full = bars;                                   // [ST] TMA -> MMA
  uint64_t* empty = bars + ST;                             // [ST] MMA -> TMA
  uint64_t* tmemFull = bars + 2 * ST;                      // [2] MMA -> epilogue
  uint64_t* tmemEmpty = bars + 2 * ST + 2;                 // [2] epilogue -> MMA
  uint64_t* drained = bars + 2 * ST + 4;                   // after a wait has run out
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(bars + 2 * ST + 5);
  volatile int* sFail = reinterpret_cast<volatile int*>(tmemSlot + 1);
  uint32_t* sLoads = tmemSlot + 2;                         // stages the producer has loaded

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int colTiles = (a.width + BN - 1) / BN;
  const int wRowTiles = MODE == WEIGHT ? (a.tileRows + BM - 1) / BM : 0;
  const uint64_t budget = a.budgetNs;
  letNextStart();

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) { umma::mbarInit(&full[s], 1); umma::mbarInit(&empty[s], 1); }
    for (int i = 0; i < 2; ++i) { umma::mbarInit(&tmemFull[i], 1); umma::mbarInit(&tmemEmpty[i], kEpiWarps); }
    umma::mbarInit(drained, 1);
    *sFail = 0;
    umma::fenceBarrierInit();
    umma::prefetchTensorMap(&a.mapA);
    umma::prefetchTensorMap(&a.mapB);
    umma::prefetchTensorMap(&a.mapC);
  }
  if (warp == 2) { umma::tmemAlloc(tmemSlot, gemm::kTmemCols); umma::tmemRelinquish(); }
  if (warp == 3) readGroups(g, a.ends, a.ends64, a.groups, a.rows, MODE == WEIGHT ? 0 : BM, MODE == WEIGHT ? wRowTiles * colTiles : colTiles, lane);
  umma::tcFenceBefore();
  __syncthreads();
  umma::tcFenceAfter();
  const uint32_t tmemBase = *tmemSlot;
  const int totalTiles = g.prefix[a.groups];
  const int kBlocks = (a.contracted + CK - 1) / CK;        // FORWARD / DATA; WEIGHT: of the group
  // Tile t, and how many blocks of the contracted dimension it has; `e` is carried from the tile before.
  auto at = [&](int t, int* e, Tile* tile) -> int {
    if constexpr (MODE == WEIGHT) {
      *e = t / (wRowTiles * colTiles);
      tileAt(g, t, *e, wRowTiles, colTiles, BM, BN, tile);
      return (g.start[*e + 1] - g.start[*e] + CK - 1) / CK;
    } else {
      *e = groupOf(g, t, *e, a.groups);
      tileAt(g, t, *e, (g.start[*e + 1] - g.start[*e] + BM - 1) / BM, colTiles, BM, BN, tile);
      return kBlocks;
    }
  };

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer
    int stage = 0, e = 0; uint32_t phase = 0, loads = 0;
    for (int t = blockIdx.x; t < totalTiles && *sFail == 0; t += gridDim.x) {
      Tile tile;
      const int blocks = at(t, &e, &tile);
      const int row0 = g.start[tile.e];
      for (int kb = 0; kb < blocks; ++kb) {
        if (!umma::mbarWaitParked(&empty[stage], phase ^ 1, budget)) { *sFail = 1; atomicExch(a.errFlag, 31); break; }
        umma::mbarExpectTx(&full[stage], S::A_BYTES + S::B_BYTES);
        uint8_t *pa = sA + stage * S::A_BYTES, *pb = sB + stage * S::B_BYTES;
        if (MODE == WEIGHT) {
#pragma unroll
          for (int c = 0; c < BM / 64; ++c) umma::tmaLoad2d(pa + c * 8192, &a.mapA, &full[stage], tile.row + c * 64, row0 + kb * CK);
#pragma unroll
          for (int c = 0; c < BN / 64; ++c) umma::tmaLoad2d(pb + c * 8192, &a.mapB, &full[stage], tile.col + c * 64, row0 + kb * CK);
        } else {
          umma::tmaLoad2d(pa, &a.mapA, &full[stage], kb * CK, row0 + tile.row);
          if (MODE == FORWARD) {
            tmaLoad3d(pb, &a.mapB, &full[stage], kb * CK, tile.col, tile.e);
          } else {
#pragma unroll
            for (int c = 0; c < BN / 64; ++c) tmaLoad3d(pb + c * 8192, &a.mapB, &full[stage], tile.col + c * 64, kb * CK, tile.e);
          }
        }
        ++loads;
        if (++stage == ST) { stage = 0; phase ^= 1; }
      }
    }
    *sLoads = loads;
  } else if (warp == 1) {
    // ---------------- MMA issuer: the warp walks the loop together and clears rows, one thread of it issues
    const bool issues = umma::electOne();
    constexpr bool aMn = MODE == WEIGHT, bMn = MODE != FORWARD;
    constexpr uint32_t idesc = umma::instrDescBf16(BM, BN) | (aMn ? 1u << 15 : 0) | (bMn ? 1u << 16 : 0);
    constexpr int aStep = aMn ? 128 : 2, bStep = bMn ? 128 : 2;    // 16 contracted elements on, in 16-byte units
    const uint64_t descA = aMn ? smemDescMn(sA) : umma::smemDescSw128(sA), descB = bMn ? smemDescMn(sB) : umma::smemDescSw128(sB);
    const uint32_t aLo0 = (uint32_t)descA, aHi = (uint32_t)(descA >> 32), bLo0 = (uint32_t)descB, bHi = (uint32_t)(descB >> 32);
    int stage = 0, e = 0, acc = 0; uint32_t phase = 0, accPhase = 0;
    for (int t = blockIdx.x; t < totalTiles; t += gridDim.x) {
      Tile tile;
      const int blocks = at(t, &e, &tile);
      if (blocks == 0) continue;                           // an expert without rows: the epilogue writes zeros by itself
      const int tail = MODE == WEIGHT ? (g.start[tile.e + 1] - g.start[tile.e]) % CK : 0, steps = (tail + 15) / 16;
      if (!waitWarp<false>(&tmemEmpty[acc], accPhase ^ 1, budget, sFail)) { if (lane == 0) atomicExch(a.errFlag, 32); break; }
      umma::tcFenceAfter();
      const uint32_t d = tmemBase + (uint32_t)acc * 256u;
      bool ok = true;
      for (int kb = 0; kb < blocks && ok; ++kb) {
        ok = umma::mbarWait(&full[stage], phase, budget);
        if (MODE == WEIGHT) {                              // the lanes meet below: they leave together
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        uint8_t *pa = sA + stage * S::A_BYTES, *pb = sB + stage * S::B_BYTES;
        const bool behind = MODE == WEIGHT && tail != 0 && kb == blocks - 1;
        if (behind) {
          // MMAs of 16 rows up to the end; of the last one's, the rows behind it in every chunk: whole 128-byte lines, which the swizzle
          // does not mix.
          for (int i = lane; i < (steps * 16 - tail) * 8; i += 32) {
            const int off = tail * 128 + i * 16;
#pragma unroll
            for (int c = 0; c < BM / 64; ++c) *reinterpret_cast<uint4*>(pa + c * 8192 + off) = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int c = 0; c < BN / 64; ++c) *reinterpret_cast<uint4*>(pb + c * 8192 + off) = make_uint4(0, 0, 0, 0);
          }
          umma::fenceProxyAsyncShared();
          __syncwarp();
        }
        umma::tcFenceAfter();
        if (issues && ok) {
          const uint32_t aLo = aLo0 + (uint32_t)(stage * (S::A_BYTES >> 4)), bLo = bLo0 + (uint32_t)(stage * (S::B_BYTES >> 4));
          umma::mmaBf16Split(d, aLo, aHi, bLo, bHi, idesc, kb != 0);
          if (!behind || steps > 1) umma::mmaBf16Split(d, aLo + aStep, aHi, bLo + bStep, bHi, idesc, 1);
          if (!behind || steps > 2) umma::mmaBf16Split(d, aLo + 2 * aStep, aHi, bLo + 2 * bStep, bHi, idesc, 1);
          if (!behind || steps > 3) umma::mmaBf16Split(d, aLo + 3 * aStep, aHi, bLo + 3 * bStep, bHi, idesc, 1);
          umma::mmaCommit(&empty[stage]);
        }
        if (++stage == ST) { stage = 0; phase ^= 1; }
      }
      if (!__all_sync(0xffffffffu, ok)) { *sFail = 1; if (lane == 0) atomicExch(a.errFlag, 33); break; }
      if (issues) umma::mmaCommit(&tmemFull[acc]);
      acc ^= 1; if (acc == 0) accPhase ^= 1;
    }
  } else if (warp >= 4) {
    // ---------------- epilogue
    const int q = warp & 3, half = (warp - 4) >> 2;        // warp % 4: the TMEM lane quarter this warp may read
    constexpr int COLS = BN / 2;
    int e = 0, acc = 0; uint32_t accPhase = 0;
    for (int t = blockIdx.x; t < totalTiles; t += gridDim.x) {
      Tile tile;
      const int blocks = at(t, &e, &tile);
      const int r = tile.row + q * 32;
      const int limit = MODE == WEIGHT ? a.tileRows : g.start[tile.e + 1] - g.start[tile.e];
      const size_t row = MODE == WEIGHT ? (size_t)tile.e * a.tileRows + r : (size_t)g.start[tile.e] + r;
      __nv_bfloat16* out = a.out + row * (size_t)a.width;
      if (MODE == WEIGHT && blocks == 0) {                 // an expert without rows
        clearTile<COLS>(out, limit - r, tile.col + half * COLS, a.width, lane);
        continue;
      }
      if (!waitWarpLong(&tmemFull[acc], accPhase, budget, blocks, a.blockNs, sFail)) { if (lane == 0) atomicExch(a.errFlag, 34); break; }
      umma::tcFenceAfter();
      uint32_t v[COLS];
      const uint32_t from = tmemBase + ((uint32_t)(q * 32) << 16) + (uint32_t)acc * 256u + (uint32_t)(half * COLS);
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c) umma::tmemLoad32x32(from + c * 32u, v + c * 32);
      umma::tmemLoadWait();
      umma::tcFenceBefore();
      __syncwarp();
      if (lane == 0) umma::mbarArrive(&tmemEmpty[acc]);
      acc ^= 1; if (acc == 0) accPhase ^= 1;
      uint8_t* stage = sStage + (warp - 4) * S::EPI_BYTES;
      if (WHOLE) storeWhole<COLS>(v, stage, &a.mapC, tile.col + half * COLS, r, tile.e, limit - r, a.width, lane);
      else storeTile<COLS>(v, stage, &a.mapC, tile.col + half * COLS, MODE == WEIGHT ? r : g.start[tile.e] + r, MODE == WEIGHT ? tile.e : -1, out, limit - r,
                           a.width, lane);
    }
    if (lane == 0) umma::tmaStoreWaitAll();
    if (MODE != WEIGHT) clearRows(a.out, g.start[a.groups], a.rows, a.width);
  }

  waitForPrevious();
  umma::tcFenceBefore();
  __syncthreads();
  if (*sFail != 0) {                                       // the same for all threads
    if (threadIdx.x == 0) drainLoads(full, ST, *sLoads);
    if (warp == 1) drainProducts(drained);
    __syncthreads();
  }
  if (warp == 2) umma::tmemDealloc(tmemBase, gemm::kTmemCols);
}

}  // namespace grouped
}  // namespace mccl
