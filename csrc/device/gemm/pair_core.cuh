// The products of grouped_core.cuh by pairs of SMs: a cluster of two CTAs works on a tile of 256 x 256 with tcgen05.mma.cta_group::2, each CTA
// staging its own 128 rows of A and its own half of B.  A stage then takes 32 KB into an SM where a single SM's tile of 128 x 256 takes 48; under
// the power limit, which bounds the large products, that is time: 16384 tokens, 8 experts of 2048 x 5504, y 279 -> 267 us, dx 275 -> 263 us,
// dw 288 -> 260 us; 8192 tokens, 8 experts of 1024 x 2048, 33 -> 29.5, 32 -> 30.5 and 36.6 -> 35.5 us.  A group's last tile costs 256 rows: with 16
// such experts 36.4 -> 36.9, 33.7 -> 40.8 and 40.8 -> 41.3 us, so the pair form is for groups of many rows (pairWanted).
// (The 8-bit product gains nothing by it: 8192 x 3584 x 8192 181 us by single SMs, 194 us by pairs, which have one accumulator beside the scales.)
//
// The leader (rank 0) issues all MMAs; all loads of a stage complete on its barrier, and its commits free the stage in both CTAs.  In WEIGHT
// the rows of the last block behind the group's end are cleared by each CTA in its own shared memory: that block's loads complete on a
// barrier of their own CTA, whose warp 3 clears and reports to the leader.  No load is shared between the CTAs (no cluster multicast).
#pragma once

#include "fp8_core.cuh"
#include "gemm_core2.cuh"
#include "thin_core.cuh"

namespace mccl {
namespace pair {

using gemm::BM;
using grouped::Groups;
using grouped::Tile;
constexpr int kThreads = grouped::kThreads, kEpiWarps = grouped::kEpiWarps, kRows = 2 * BM;
constexpr int BN = 256, HALF = BN / 2, CK = 64, ST = 6;                             // columns of a tile, of a CTA's half of B; contracted elements a stage; stages
using grouped::DATA;
using grouped::FORWARD;
using grouped::WEIGHT;

using Args = grouped::Args;            // with boxes of half the tile's columns for B in FORWARD

constexpr int A_BYTES = BM * 128, B_BYTES = HALF * 128, TILE_BYTES = ST * (A_BYTES + B_BYTES), TABLE_BYTES = 2 * (grouped::kMaxGroups + 4) * 4;
constexpr int SMEM_BYTES = TILE_BYTES + kEpiWarps * grouped::kStageBytes + TABLE_BYTES + 512 + 1024;

__device__ __forceinline__ void tmaLoad2dPair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) { gemm::umma2::tmaLoad2dPair(dst, map, bar, x, y); }
__device__ __forceinline__ void tmaLoad3dPair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      :: "r"(umma::smemAddr(dst)), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void mmaBf16(uint32_t d, uint32_t aLo, uint32_t aHi, uint32_t bLo, uint32_t bHi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %2};\n mov.b64 db, {%3, %4};\n setp.ne.b32 p, %6, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n}"
      :: "r"(d), "r"(aLo), "r"(aHi), "r"(bLo), "r"(bHi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commitBoth(uint64_t* bar) { gemm::umma2::mmaCommitMask(bar, 3); }
// A wait of a whole warp for arrivals that may come from the other CTA.
__device__ __forceinline__ bool waitWarpCluster(uint64_t* bar, uint32_t parity, uint64_t budget, volatile int* sFail) {
  bool ok = *sFail == 0;
  if (ok) ok = thin::waitCluster(bar, parity, budget);
  if (__all_sync(0xffffffffu, ok)) return true;
  *sFail = 1;
  return false;
}
__device__ __forceinline__ void storeCluster(void* here, uint32_t cta, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" :: "r"(gemm::umma2::mapToCta(umma::smemAddr(here), cta)), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t loadCluster(const void* here, uint32_t cta) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(gemm::umma2::mapToCta(umma::smemAddr(here), cta)) : "memory");
  return v;
}
// The loads in flight after a wait has run out, as in grouped_core.cuh.  Those of both CTAs complete on the leader's barriers, but for a group's last
// blocks; what the other CTA alone has loaded completes on barriers that the leader has not armed yet.  (A stage that the leader alone has
// loaded does not complete: there the wait ends by its limit.)
__device__ __forceinline__ void drainLoads(uint64_t* full, uint64_t* tailFull, const uint32_t* sLoads, int rank) {
  for (int s = 0; s < ST; ++s)
    if (!umma::mbarWait(&tailFull[s], (sLoads[1] >> s & 1) ^ 1, grouped::kDrainNs)) return;
  if (rank != 0) return;
  uint32_t loads = sLoads[0];
  for (const uint32_t theirs = loadCluster(sLoads, 1); loads < theirs; ++loads) umma::mbarExpectTx(&full[loads % ST], A_BYTES + B_BYTES);
  grouped::drainLoads(full, ST, loads);
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1) pairKernel(const __grid_constant__ Args a) {
  constexpr bool aMn = MODE == WEIGHT, bMn = MODE != FORWARD;
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sB = smem + ST * A_BYTES;
  uint8_t* sStage = smem + TILE_BYTES;
  int* table = reinterpret_cast<int*>(sStage + kEpiWarps * grouped::kStageBytes);
  const Groups g{table, table + grouped::kMaxGroups + 4};
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(table) + TABLE_BYTES);
  uint64_t* full = bars;                                   // [ST] leader: all four loads of a stage
  uint64_t* empty = bars + ST;                             // [ST] each CTA: the MMAs have read the stage
  uint64_t* tmemFull = bars + 2 * ST;                      // [2] each CTA: accumulator complete
  uint64_t* tmemEmpty = tmemFull + 2;                      // [2] leader: both CTAs' epilogues have it in registers
  uint64_t* tailFull = tmemEmpty + 2;                      // WEIGHT [ST] each CTA: its loads of a block that reaches behind the group
  uint64_t* tailReady = tailFull + ST;                     // WEIGHT [ST] leader: both CTAs have cleared theirs
  uint64_t* drained = tailReady + ST;                      // each CTA, after a wait has run out
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* sFail = reinterpret_cast<volatile int*>(tmemSlot + 1);
  uint32_t* sLoads = tmemSlot + 2;                         // stages the producer has loaded, and those of tailFull's next phases (a bit per stage)

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)gemm::umma2::clusterCtaRank(), pairIdx = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int colTiles = (a.width + BN - 1) / BN;
  const int wRowTiles = MODE == WEIGHT ? (a.tileRows + kRows - 1) / kRows : 0;
  const uint64_t budget = a.budgetNs;
  grouped::letNextStart();

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) { umma::mbarInit(&full[s], 1); umma::mbarInit(&empty[s], 1); umma::mbarInit(&tailFull[s], 1); umma::mbarInit(&tailReady[s], 2); }
    for (int i = 0; i < 2; ++i) { umma::mbarInit(&tmemFull[i], 1); umma::mbarInit(&tmemEmpty[i], 2 * kEpiWarps); }
    umma::mbarInit(drained, 1);
    *sFail = 0;
    umma::fenceBarrierInit();
    umma::prefetchTensorMap(&a.mapA);
    umma::prefetchTensorMap(&a.mapB);
    umma::prefetchTensorMap(&a.mapC);
  }
  if (warp == 2) { gemm::umma2::tmemAlloc(tmemSlot, gemm::kTmemCols); gemm::umma2::tmemRelinquish(); }
  if (warp == 3) grouped::readGroups(g, a.ends, a.ends64, a.groups, a.rows, MODE == WEIGHT ? 0 : kRows, MODE == WEIGHT ? wRowTiles * colTiles : colTiles, lane);
  umma::tcFenceBefore();
  __syncthreads();
  gemm::umma2::clusterSync();                              // both CTAs' barriers exist before anything signals them
  umma::tcFenceAfter();
  const uint32_t tmemBase = *tmemSlot;
  const int totalTiles = g.prefix[a.groups];
  const int kBlocks = (a.contracted + CK - 1) / CK;
  // Tile t, and how many blocks of the contracted dimension it has; `e` is carried from the tile before.
  auto at = [&](int t, int* e, Tile* tile) -> int {
    if constexpr (MODE == WEIGHT) {
      *e = t / (wRowTiles * colTiles);
      grouped::tileAt(g, t, *e, wRowTiles, colTiles, kRows, BN, tile);
      return (g.start[*e + 1] - g.start[*e] + CK - 1) / CK;
    } else {
      *e = grouped::groupOf(g, t, *e, a.groups);
      grouped::tileAt(g, t, *e, (g.start[*e + 1] - g.start[*e] + kRows - 1) / kRows, colTiles, kRows, BN, tile);
      return kBlocks;
    }
  };

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer
    int stage = 0, e = 0; uint32_t phase = 0, loads = 0, tailNext = 0;
    for (int t = pairIdx; t < totalTiles && *sFail == 0; t += pairs) {
      Tile tile;
      const int blocks = at(t, &e, &tile);
      const int row0 = g.start[tile.e];
      const bool tail = MODE == WEIGHT && (g.start[tile.e + 1] - row0) % CK != 0;
      for (int kb = 0; kb < blocks; ++kb) {
        if (!umma::mbarWaitParked(&empty[stage], phase ^ 1, budget)) { *sFail = 1; atomicExch(a.errFlag, 61); break; }
        uint8_t *pa = sA + stage * A_BYTES, *pb = sB + stage * B_BYTES;
        const uint32_t leaderFull = gemm::umma2::mapToCta(umma::smemAddr(&full[stage]), 0);
        if (MODE == WEIGHT && tail && kb == blocks - 1) {  // cleared before the MMAs: complete in this CTA
          if (rank == 0) umma::mbarArrive(&full[stage]);
          tailNext ^= 1u << stage;
          umma::mbarExpectTx(&tailFull[stage], A_BYTES + B_BYTES);
#pragma unroll
          for (int c = 0; c < BM / 64; ++c) umma::tmaLoad2d(pa + c * 8192, &a.mapA, &tailFull[stage], tile.row + rank * BM + c * 64, row0 + kb * CK);
#pragma unroll
          for (int c = 0; c < HALF / 64; ++c) umma::tmaLoad2d(pb + c * 8192, &a.mapB, &tailFull[stage], tile.col + rank * HALF + c * 64, row0 + kb * CK);
        } else {
          if (rank == 0) umma::mbarExpectTx(&full[stage], 2 * (A_BYTES + B_BYTES));
          if (MODE == WEIGHT) {
#pragma unroll
            for (int c = 0; c < BM / 64; ++c) tmaLoad2dPair(pa + c * 8192, &a.mapA, leaderFull, tile.row + rank * BM + c * 64, row0 + kb * CK);
#pragma unroll
            for (int c = 0; c < HALF / 64; ++c) tmaLoad2dPair(pb + c * 8192, &a.mapB, leaderFull, tile.col + rank * HALF + c * 64, row0 + kb * CK);
          } else {
            tmaLoad2dPair(pa, &a.mapA, leaderFull, kb * CK, row0 + tile.row + rank * BM);
            if (MODE == DATA) {
#pragma unroll
              for (int c = 0; c < HALF / 64; ++c) tmaLoad3dPair(pb + c * 8192, &a.mapB, leaderFull, tile.col + rank * HALF + c * 64, kb * CK, tile.e);
            } else {
              tmaLoad3dPair(pb, &a.mapB, leaderFull, kb * CK, tile.col + rank * HALF, tile.e);
            }
          }
        }
        ++loads;
        if (++stage == ST) { stage = 0; phase ^= 1; }
      }
    }
    sLoads[0] = loads; sLoads[1] = tailNext;
  } else if (warp == 1 && rank == 0) {
    // ---------------- MMA issuer (leader): the warp walks the loop together, one thread of it issues
    const bool issues = umma::electOne();
    constexpr uint32_t idesc = umma::instrDescBf16(kRows, BN) | (aMn ? 1u << 15 : 0) | (bMn ? 1u << 16 : 0);
    constexpr int aStep = aMn ? 128 : 2, bStep = bMn ? 128 : 2;
    const uint64_t descA = aMn ? grouped::smemDescMn(sA) : umma::smemDescSw128(sA), descB = bMn ? grouped::smemDescMn(sB) : umma::smemDescSw128(sB);
    const uint32_t aLo0 = (uint32_t)descA, aHi = (uint32_t)(descA >> 32), bLo0 = (uint32_t)descB, bHi = (uint32_t)(descB >> 32);
    int stage = 0, e = 0, acc = 0; uint32_t phase = 0, accPhase = 0, tailPhase = 0;   // tailPhase: a bit per stage
    for (int t = pairIdx; t < totalTiles; t += pairs) {
      Tile tile;
      const int blocks = at(t, &e, &tile);
      if (blocks == 0) continue;                           // an expert without rows: the epilogues write zeros by themselves
      const int tail = MODE == WEIGHT ? (g.start[tile.e + 1] - g.start[tile.e]) % CK : 0, steps = (tail + 15) / 16;
      if (!waitWarpCluster(&tmemEmpty[acc], accPhase ^ 1, budget, sFail)) { if (lane == 0) atomicExch(a.errFlag, 62); break; }
      umma::tcFenceAfter();
      const uint32_t d = tmemBase + (uint32_t)(acc * BN);
      bool ok = true;
      for (int kb = 0; kb < blocks && ok; ++kb) {
        ok = umma::mbarWait(&full[stage], phase, budget);
        const bool behind = MODE == WEIGHT && tail != 0 && kb == blocks - 1;
        if (behind) {
          ok = thin::waitCluster(&tailReady[stage], tailPhase >> stage & 1, budget) && ok;
          tailPhase ^= 1u << stage;
        }
        umma::tcFenceAfter();
        if (issues && ok) {
          const uint32_t aLo = aLo0 + (uint32_t)(stage * (A_BYTES >> 4)), bLo = bLo0 + (uint32_t)(stage * (B_BYTES >> 4));
          mmaBf16(d, aLo, aHi, bLo, bHi, idesc, kb != 0);
          if (!behind || steps > 1) mmaBf16(d, aLo + aStep, aHi, bLo + bStep, bHi, idesc, 1);
          if (!behind || steps > 2) mmaBf16(d, aLo + 2 * aStep, aHi, bLo + 2 * bStep, bHi, idesc, 1);
          if (!behind || steps > 3) mmaBf16(d, aLo + 3 * aStep, aHi, bLo + 3 * bStep, bHi, idesc, 1);
          commitBoth(&empty[stage]);
        }
        if (++stage == ST) { stage = 0; phase ^= 1; }
      }
      if (!__all_sync(0xffffffffu, ok)) { *sFail = 1; if (lane == 0) atomicExch(a.errFlag, 63); break; }
      if (issues) commitBoth(&tmemFull[acc]);
      acc ^= 1; if (acc == 0) accPhase ^= 1;
    }
  } else if (warp == 3 && MODE == WEIGHT) {
    // ---------------- of a group's last block, the rows behind its end that the last MMA of 16 takes in (as in grouped_core.cuh)
    int stage = 0, e = 0; uint32_t tailPhase = 0;          // a bit per stage
    uint64_t walked = 0;                                   // blocks since the last such one
    for (int t = pairIdx; t < totalTiles; t += pairs) {
      Tile tile;
      const int blocks = at(t, &e, &tile), tail = (g.start[tile.e + 1] - g.start[tile.e]) % CK;
      stage = (stage + blocks) % ST;
      walked += blocks;
      if (tail == 0) continue;
      const int last = (stage + ST - 1) % ST;
      if (!grouped::waitWarpLong(&tailFull[last], tailPhase >> last & 1, budget, walked, a.blockNs, sFail)) { if (lane == 0) atomicExch(a.errFlag, 64); break; }
      tailPhase ^= 1u << last;
      walked = 0;
      uint8_t *pa = sA + last * A_BYTES, *pb = sB + last * B_BYTES;
      for (int i = lane; i < ((tail + 15) / 16 * 16 - tail) * 8; i += 32) {
        const int off = tail * 128 + i * 16;
#pragma unroll
        for (int c = 0; c < BM / 64; ++c) *reinterpret_cast<uint4*>(pa + c * 8192 + off) = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < HALF / 64; ++c) *reinterpret_cast<uint4*>(pb + c * 8192 + off) = make_uint4(0, 0, 0, 0);
      }
      umma::fenceProxyAsyncShared();
      __syncwarp();
      if (lane == 0) thin::arriveCluster(&tailReady[last], 0);
    }
  } else if (warp >= 4) {
    // ---------------- epilogue: this CTA's 128 rows
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint8_t* stage = sStage + (warp - 4) * grouped::kStageBytes;
    int e = 0, acc = 0; uint32_t accPhase = 0;
    for (int t = pairIdx; t < totalTiles; t += pairs) {
      Tile tile;
      const int blocks = at(t, &e, &tile);
      const int r = tile.row + rank * BM + q * 32;
      const int limit = MODE == WEIGHT ? a.tileRows : g.start[tile.e + 1] - g.start[tile.e];
      const size_t row = MODE == WEIGHT ? (size_t)tile.e * a.tileRows + r : (size_t)g.start[tile.e] + r;
      __nv_bfloat16* out = a.out + row * (size_t)a.width;
      if (MODE == WEIGHT && blocks == 0) {                 // an expert without rows
        grouped::clearTile<HALF>(out, limit - r, tile.col + half * HALF, a.width, lane);
        continue;
      }
      if (!grouped::waitWarpLong(&tmemFull[acc], accPhase, budget, blocks, a.blockNs, sFail)) { if (lane == 0) atomicExch(a.errFlag, 66); break; }
      umma::tcFenceAfter();
      uint32_t v[HALF];
      const uint32_t from = tmemBase + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + half * HALF);
#pragma unroll
      for (int c = 0; c < HALF / 32; ++c) umma::tmemLoad32x32(from + c * 32u, v + c * 32);
      umma::tmemLoadWait();
      umma::tcFenceBefore();
      __syncwarp();
      if (lane == 0) thin::arriveCluster(&tmemEmpty[acc], 0);
      acc ^= 1; if (acc == 0) accPhase ^= 1;
      grouped::storeTile<HALF>(v, stage, &a.mapC, tile.col + half * HALF, MODE == WEIGHT ? r : g.start[tile.e] + r, MODE == WEIGHT ? tile.e : -1, out, limit - r,
                               a.width, lane);
    }
    if (lane == 0) umma::tmaStoreWaitAll();
    if (MODE != WEIGHT) grouped::clearRows(a.out, g.start[a.groups], a.rows, a.width);
  }

  grouped::waitForPrevious();
  umma::tcFenceBefore();
  __syncthreads();
  if (threadIdx.x == 0 && *sFail != 0) storeCluster(const_cast<int*>(sFail), rank ^ 1, 1);
  gemm::umma2::clusterSync();                              // neither CTA frees tensor memory the other still uses
  if (*sFail != 0) {                                       // the same for all threads of both
    if (threadIdx.x == 0) drainLoads(full, tailFull, sLoads, rank);
    if (warp == 1 && umma::electOne()) {
      if (rank == 0) commitBoth(drained);
      umma::mbarWait(drained, 0, grouped::kDrainNs);
    }
    __syncthreads();
    gemm::umma2::clusterSync();
  }
  if (warp == 2) gemm::umma2::tmemDealloc(tmemBase, gemm::kTmemCols);
}

}  // namespace pair
}  // namespace mccl
