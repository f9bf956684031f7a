// Product in 8-bit floating point (e4m3) with a power-of-two scale (e8m0) for each block of 128 of the contracted dimension, on the
// tcgen05 tensor cores; dense, or over ragged groups of rows as in grouped_core.cuh.
//
//   y[m, n] = sum over blocks b of sx[m, b] sw[n / 128, b] sum over k in b of x[m, k] w[n, k]
//
// The scales are applied by the tensor core itself: tcgen05.mma.block_scale multiplies every product of 32 by one scale of A's row and
// one of B's column, held in tensor memory, and adds up in fp32, so the sums never leave it between blocks.  (With the scales
// applied outside, every block's sums would be read from tensor memory and added up in registers: 128 x 256 fp32 for 512 cycles
// of products.)  The instruction's blocks are of 32, the operator's of 128: the four MMAs of a 128-byte stage name the same scale.
// Tensor memory takes scales in words of four bytes: a word is four blocks of one row, that is four stages; the MMA's descriptor
// picks the byte.  One warp fetches the words of 128 rows (and of the columns, where 128 share one) for the next four stages into
// shared memory in the order [row % 32][row / 32], from where tcgen05.cp replicates them to the four lane quarters.
// Tensor memory: 256 columns of sums (one accumulator of 256 columns, or two of 128) and three sets of scales.  A set is
// free once the MMAs that used it are done, which the commit that frees its shared memory says too.
#pragma once

#include "grouped_core.cuh"

namespace mccl {
namespace fp8 {

using gemm::BM;
using grouped::Groups;
using grouped::Tile;
constexpr int kThreads = grouped::kThreads, kEpiWarps = grouped::kEpiWarps;
constexpr int kBlock = 128;                     // contracted elements a scale, and a stage: 128 bytes
constexpr int kScaleSets = 3, kScaleCols = 12;  // tensor-memory columns a set: 4 for A's rows, 8 for B's
constexpr int kScaleBase = 256;

struct Args {
  CUtensorMap mapA;                    // x [M, K] bytes, box 128 x 128
  CUtensorMap mapB;                    // w [E, N, K] bytes, box 128 x BN
  CUtensorMap mapC;                    // y [M, N], box 32 x 32
  const uint8_t *sx, *sw;              // [M][ldsx], [E][N / 128][ldsw]: scales, a row a multiple of four bytes apart
  int64_t ldsx, ldsw;
  const void* ends;                    // nullable: one group
  int ends64, groups;
  int rows, N, K;
  __nv_bfloat16* out;                  // [M, N]
  int* errFlag;
  uint64_t budgetNs, blockNs;          // as in grouped::Args
};

template <int BN> struct Smem {
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128;
  static constexpr int STAGES = BN == 256 ? 4 : 6;
  static constexpr int ACCS = BN == 256 ? 1 : 2;
  static constexpr int TILE_BYTES = STAGES * (A_BYTES + B_BYTES);
  static constexpr int SCALE_BYTES = 512 + BN * 4;         // a set: 128 words of A, BN of B
  static constexpr int TABLE_BYTES = 2 * (grouped::kMaxGroups + 4) * 4;
  static constexpr int TOTAL = TILE_BYTES + kEpiWarps * grouped::kStageBytes + kScaleSets * SCALE_BYTES + TABLE_BYTES + 256 + 1024;
};

// Scales in shared memory, 32 rows of 16 bytes, as tcgen05.cp reads them: no swizzle, groups of eight rows 128 bytes apart.
__device__ __forceinline__ uint64_t smemDescScales(const void* p) {
  uint64_t d = 0;
  d |= (uint64_t)((umma::smemAddr(p) & 0x3ffff) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(128 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  return d;
}
// 32 rows x 128 bits from shared memory to four columns of tensor memory, in all four lane quarters.
__device__ __forceinline__ void copyScales(uint32_t tmem, uint32_t descLo, uint32_t descHi) {
  asm volatile("{\n .reg .b64 d;\n mov.b64 d, {%1, %2};\n tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n}" :: "r"(tmem), "r"(descLo), "r"(descHi) : "memory");
}
// Instruction descriptor of kind::mxf8f6f4 with e4m3 A and B, both K-major, e8m0 scales, M x N; plus kScaleByte for each byte of the
// scales' words after the first.
__host__ __device__ constexpr uint32_t instrDesc(int m, int n) { return ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24); }
constexpr uint32_t kScaleByte = (1u << 4) | (1u << 29);
__device__ __forceinline__ void mmaScaled(uint32_t d, uint32_t aLo, uint32_t bLo, uint32_t hi, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %3};\n setp.ne.b32 p, %7, 0;\n"
      " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %4, [%5], [%6], p;\n}"
      :: "r"(d), "r"(aLo), "r"(bLo), "r"(hi), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}

// With programmatic stream serialization this kernel starts before the one that quantises its rows has ended: nothing of that kernel's is
// read before this.  Without, it returns at once.
__device__ __forceinline__ void waitForPredecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Scales of blocks [4 i, 4 i + 4) of a row, of which there are `blocks`.
__device__ __forceinline__ uint32_t scaleWord(const uint8_t* row, int i, int blocks) {
  if (4 * i + 4 <= blocks) return *reinterpret_cast<const uint32_t*>(row + 4 * i);
  uint32_t w = 0;
  for (int b = 4 * i; b < blocks; ++b) w |= (uint32_t)row[b] << (8 * (b - 4 * i));
  return w;
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1) fp8Kernel(const __grid_constant__ Args a) {
  using S = Smem<BN>;
  constexpr int ST = S::STAGES, ACCS = S::ACCS;
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sB = smem + ST * S::A_BYTES;
  uint8_t* sStage = smem + S::TILE_BYTES;
  uint8_t* sScale = sStage + kEpiWarps * grouped::kStageBytes;
  int* table = reinterpret_cast<int*>(sScale + kScaleSets * S::SCALE_BYTES);
  const Groups g{table, table + grouped::kMaxGroups + 4};
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(table) + S::TABLE_BYTES);
  uint64_t* full = bars;                                   // [ST] TMA -> MMA
  uint64_t* empty = bars + ST;                             // [ST] MMA -> TMA
  uint64_t* tmemFull = bars + 2 * ST;                      // [ACCS] MMA -> epilogue
  uint64_t* tmemEmpty = bars + 2 * ST + 2;                 // [ACCS] epilogue -> MMA
  uint64_t* scaleFull = bars + 2 * ST + 4;                 // [kScaleSets] scale warp -> MMA
  uint64_t* scaleEmpty = scaleFull + kScaleSets;           // [kScaleSets] MMA -> scale warp
  uint64_t* drained = scaleEmpty + kScaleSets;             // after a wait has run out
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* sFail = reinterpret_cast<volatile int*>(tmemSlot + 1);
  uint32_t* sLoads = tmemSlot + 2;                         // stages the producer has loaded

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int colTiles = (a.N + BN - 1) / BN, kBlocks = (a.K + kBlock - 1) / kBlock;
  const uint64_t budget = a.budgetNs;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) { umma::mbarInit(&full[s], 1); umma::mbarInit(&empty[s], 1); }
    for (int i = 0; i < ACCS; ++i) { umma::mbarInit(&tmemFull[i], 1); umma::mbarInit(&tmemEmpty[i], kEpiWarps); }
    for (int i = 0; i < kScaleSets; ++i) { umma::mbarInit(&scaleFull[i], 1); umma::mbarInit(&scaleEmpty[i], 1); }
    umma::mbarInit(drained, 1);
    *sFail = 0;
    umma::fenceBarrierInit();
    umma::prefetchTensorMap(&a.mapA);
    umma::prefetchTensorMap(&a.mapB);
    umma::prefetchTensorMap(&a.mapC);
  }
  if (warp == 2) { umma::tmemAlloc(tmemSlot, gemm::kTmemCols); umma::tmemRelinquish(); }
  if (warp == 3) grouped::readGroups(g, a.ends, a.ends64, a.groups, a.rows, BM, colTiles, lane);
  umma::tcFenceBefore();
  __syncthreads();
  umma::tcFenceAfter();
  const uint32_t tmemBase = *tmemSlot;
  const int totalTiles = g.prefix[a.groups];
  auto at = [&](int t, int* e, Tile* tile) {               // tile t; `e` is carried from the tile before
    *e = grouped::groupOf(g, t, *e, a.groups);
    grouped::tileAt(g, t, *e, (g.start[*e + 1] - g.start[*e] + BM - 1) / BM, colTiles, BM, BN, tile);
  };

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer
    int stage = 0, e = 0; uint32_t phase = 0, loads = 0;
    waitForPredecessor();
    for (int t = blockIdx.x; t < totalTiles && *sFail == 0; t += gridDim.x) {
      Tile tile;
      at(t, &e, &tile);
      const int row = g.start[tile.e] + tile.row;
      for (int kb = 0; kb < kBlocks; ++kb) {
        if (!umma::mbarWaitParked(&empty[stage], phase ^ 1, budget)) { *sFail = 1; atomicExch(a.errFlag, 41); break; }
        umma::mbarExpectTx(&full[stage], S::A_BYTES + S::B_BYTES);
        umma::tmaLoad2d(sA + stage * S::A_BYTES, &a.mapA, &full[stage], kb * kBlock, row);
        grouped::tmaLoad3d(sB + stage * S::B_BYTES, &a.mapB, &full[stage], kb * kBlock, tile.col, tile.e);
        ++loads;
        if (++stage == ST) { stage = 0; phase ^= 1; }
      }
    }
    *sLoads = loads;
  } else if (warp == 1) {
    // ---------------- MMA issuer: the warp walks the loop together, one thread of it issues
    const bool issues = umma::electOne();
    const uint64_t descA = umma::smemDescSw128(sA), descScale = smemDescScales(sScale);
    const uint32_t aLo0 = (uint32_t)descA, bLo0 = (uint32_t)umma::smemDescSw128(sB), hi = (uint32_t)(descA >> 32);
    const uint32_t scaleLo0 = (uint32_t)descScale, scaleHi = (uint32_t)(descScale >> 32);
    int stage = 0, e = 0, acc = 0, set = 0; uint32_t phase = 0, accPhase = 0, setPhase = 0;
    for (int t = blockIdx.x; t < totalTiles; t += gridDim.x) {
      Tile tile;
      at(t, &e, &tile);
      if (!grouped::waitWarp<false>(&tmemEmpty[acc], accPhase ^ 1, budget, sFail)) { if (lane == 0) atomicExch(a.errFlag, 42); break; }
      umma::tcFenceAfter();
      const uint32_t d = tmemBase + (uint32_t)acc * 128u;
      bool ok = true;
      for (int kb = 0; kb < kBlocks && ok; ++kb) {
        const uint32_t sfa = tmemBase + kScaleBase + (uint32_t)(set * kScaleCols), sfb = sfa + 4;
        if ((kb & 3) == 0) {
          ok = umma::mbarWait(&scaleFull[set], setPhase, budget);
          umma::tcFenceAfter();
          if (issues && ok) {
            const uint32_t from = scaleLo0 + (uint32_t)(set * (S::SCALE_BYTES >> 4));
            copyScales(sfa, from, scaleHi);
#pragma unroll
            for (int b = 0; b < BN / 128; ++b) copyScales(sfb + 4 * b, from + 32 + 32 * b, scaleHi);
          }
        }
        ok = umma::mbarWait(&full[stage], phase, budget) && ok;
        umma::tcFenceAfter();
        const bool lastOfSet = (kb & 3) == 3 || kb == kBlocks - 1;
        if (issues && ok) {
          const uint32_t aLo = aLo0 + (uint32_t)(stage * (S::A_BYTES >> 4)), bLo = bLo0 + (uint32_t)(stage * (S::B_BYTES >> 4));
          const uint32_t idesc = instrDesc(BM, BN) + (uint32_t)(kb & 3) * kScaleByte;
          mmaScaled(d, aLo, bLo, hi, idesc, sfa, sfb, kb != 0);
          mmaScaled(d, aLo + 2, bLo + 2, hi, idesc, sfa, sfb, 1);
          mmaScaled(d, aLo + 4, bLo + 4, hi, idesc, sfa, sfb, 1);
          mmaScaled(d, aLo + 6, bLo + 6, hi, idesc, sfa, sfb, 1);
          umma::mmaCommit(&empty[stage]);
          if (lastOfSet) umma::mmaCommit(&scaleEmpty[set]);
        }
        if (lastOfSet && ++set == kScaleSets) { set = 0; setPhase ^= 1; }
        if (++stage == ST) { stage = 0; phase ^= 1; }
      }
      if (!__all_sync(0xffffffffu, ok)) { *sFail = 1; if (lane == 0) atomicExch(a.errFlag, 44); break; }
      if (issues) umma::mmaCommit(&tmemFull[acc]);
      if (++acc == ACCS) { acc = 0; accPhase ^= 1; }
    }
  } else if (warp == 3) {
    // ---------------- scales
    int set = 0, e = 0; uint32_t setPhase = 0;
    bool ok = true;
    waitForPredecessor();
    for (int t = blockIdx.x; t < totalTiles && ok; t += gridDim.x) {
      Tile tile;
      at(t, &e, &tile);
      const uint8_t* row[4];
      const uint8_t* col[BN / 128];
#pragma unroll
      for (int j = 0; j < 4; ++j) row[j] = a.sx + (int64_t)min(g.start[tile.e] + tile.row + j * 32 + lane, a.rows - 1) * a.ldsx;
      const int nBlocks = (a.N + kBlock - 1) / kBlock;
#pragma unroll
      for (int b = 0; b < BN / 128; ++b) col[b] = a.sw + ((int64_t)tile.e * nBlocks + min(tile.col / kBlock + b, nBlocks - 1)) * a.ldsw;
      for (int i = 0; i * 4 < kBlocks; ++i) {
        uint32_t r[4], c[BN / 128];
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = scaleWord(row[j], i, kBlocks);
#pragma unroll
        for (int b = 0; b < BN / 128; ++b) c[b] = scaleWord(col[b], i, kBlocks);
        if (!grouped::waitWarp<true>(&scaleEmpty[set], setPhase ^ 1, budget, sFail)) { if (lane == 0) atomicExch(a.errFlag, 45); ok = false; break; }
        uint4* to = reinterpret_cast<uint4*>(sScale + set * S::SCALE_BYTES) + lane;
        to[0] = make_uint4(r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int b = 0; b < BN / 128; ++b) to[32 + 32 * b] = make_uint4(c[b], c[b], c[b], c[b]);
        umma::fenceProxyAsyncShared();
        __syncwarp();
        if (lane == 0) umma::mbarArrive(&scaleFull[set]);
        if (++set == kScaleSets) { set = 0; setPhase ^= 1; }
      }
    }
  } else if (warp >= 4) {
    // ---------------- epilogue
    const int q = warp & 3, half = (warp - 4) >> 2;
    constexpr int COLS = BN / 2;
    int e = 0, acc = 0; uint32_t accPhase = 0;
    for (int t = blockIdx.x; t < totalTiles; t += gridDim.x) {
      Tile tile;
      at(t, &e, &tile);
      if (!grouped::waitWarpLong(&tmemFull[acc], accPhase, budget, kBlocks, a.blockNs, sFail)) { if (lane == 0) atomicExch(a.errFlag, 46); break; }
      umma::tcFenceAfter();
      uint32_t v[COLS];
      const uint32_t from = tmemBase + ((uint32_t)(q * 32) << 16) + (uint32_t)acc * 128u + (uint32_t)(half * COLS);
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c) umma::tmemLoad32x32(from + c * 32u, v + c * 32);
      umma::tmemLoadWait();
      umma::tcFenceBefore();
      __syncwarp();
      if (lane == 0) umma::mbarArrive(&tmemEmpty[acc]);    // the sums are in registers: the next tile may start
      if (++acc == ACCS) { acc = 0; accPhase ^= 1; }
      const int r = tile.row + q * 32;
      grouped::storeTile<COLS>(v, sStage + (warp - 4) * grouped::kStageBytes, &a.mapC, tile.col + half * COLS, g.start[tile.e] + r, -1,
                               a.out + ((size_t)g.start[tile.e] + r) * (size_t)a.N, g.start[tile.e + 1] - g.start[tile.e] - r, a.N, lane);
    }
    if (lane == 0) umma::tmaStoreWaitAll();
    grouped::clearRows(a.out, g.start[a.groups], a.rows, a.N);
  }

  waitForPredecessor();                                    // this grid's end stands for its predecessor's too
  umma::tcFenceBefore();
  __syncthreads();
  if (*sFail != 0) {                                       // the same for all threads
    if (threadIdx.x == 0) grouped::drainLoads(full, ST, *sLoads);
    if (warp == 1) grouped::drainProducts(drained);
    __syncthreads();
  }
  if (warp == 2) umma::tmemDealloc(tmemBase, gemm::kTmemCols);
}

}  // namespace fp8
}  // namespace mccl
