// The products of grouped_core.cuh and fp8_core.cuh (forward) for few rows, where the weights' bytes are what counts: a tile of 128 of
// the WEIGHTS' rows is the tensor core's A, and BT rows of x its B, so that a product of one row reads no more and computes no
// more than it has to, and its weights are spread over as many CTAs as there are 128-row tiles of them.  Where those are fewer than
// the SMs can hold, a cluster of up to eight CTAs shares a tile along the contracted dimension: each leaves its fp32 sums in its shared memory,
// and the CTAs add up, rank by rank in a fixed order, the results they store.  Nothing goes through global memory but operands and results.
//
// Launched behind the kernel that quantises the rows, with programmatic stream serialization: the weights' first stages are requested
// before that kernel has ended, the rows after it.
//
// Grid: x = tile x cluster rank, y = expert, z = share of the expert's rows.  Warps 0 TMA, 1 MMA, 2 tensor memory, 3 groups and scales, 4-7 sums.
#pragma once

#include "fp8_core.cuh"
#include "gemm_core2.cuh"

namespace mccl {
namespace thin {

using gemm::BM;
constexpr int kThreads = 256;

struct Args {
  CUtensorMap mapW;                    // w [E, N, K], box 128 rows x 128 bytes
  CUtensorMap mapX;                    // x [M, K], box BT rows x 128 bytes
  const uint8_t *sx, *sw;              // 8-bit: scales as in fp8::Args
  int64_t ldsx, ldsw;
  const void* ends;                    // nullable: one group
  int ends64, groups;
  int rows, N, K, slices;
  __nv_bfloat16* out;                  // [M, N]
  int* errFlag;
  uint64_t budgetNs, blockNs;          // as in grouped::Args
};

template <int BT> struct Smem {
  static constexpr int A_BYTES = BM * 128, B_BYTES = BT * 128;
  static constexpr int STAGES = BT == 16 ? 5 : BT == 32 ? 4 : 3;                     // two CTAs an SM
  static constexpr int TILE_BYTES = STAGES * (A_BYTES + B_BYTES);
  static constexpr int SUM_BYTES = BT * BM * 4;
  static constexpr int SCALE_BYTES = 1024;                 // a set: 512 of the weights, 512 of the rows
  static constexpr int TOTAL = TILE_BYTES + SUM_BYTES + fp8::kScaleSets * SCALE_BYTES + 256 + 1024;
  static constexpr int TMEM = BT <= 32 ? 64 : 128;         // BT columns of sums and 24 of scales
};

__device__ __forceinline__ void arriveCluster(uint64_t* bar, uint32_t cta) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(gemm::umma2::mapToCta(umma::smemAddr(bar), cta)) : "memory");
}
__device__ __forceinline__ bool waitCluster(uint64_t* bar, uint32_t parity, uint64_t budgetNs) {
  uint64_t t0 = 0;
  for (uint32_t spins = 0;; ++spins) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n selp.b32 %0, 1, 0, p;\n}"
        : "=r"(done) : "r"(umma::smemAddr(bar)), "r"(parity), "r"(1000u) : "memory");
    if (done) return true;
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    if (spins == 0) t0 = t;
    else if (t - t0 > budgetNs) return false;
  }
}
__device__ __forceinline__ float4 loadCluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void tmemLoad32x16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr) : "memory");
}
using fp8::waitForPredecessor;
// The two halves of a barrier over all threads of the cluster.
__device__ __forceinline__ void clusterArrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void clusterWait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

template <int BT, bool FP8>
__global__ void __launch_bounds__(kThreads, 2) thinKernel(const __grid_constant__ Args a) {
  using S = Smem<BT>;
  constexpr int ST = S::STAGES, CK = FP8 ? 128 : 64, UNIT = FP8 ? 4 : 1;             // a rank's share is whole words of scales
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sB = smem + ST * S::A_BYTES;
  float* sSum = reinterpret_cast<float*>(smem + S::TILE_BYTES);                      // [BT][128]
  uint8_t* sScale = smem + S::TILE_BYTES + S::SUM_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sScale + fp8::kScaleSets * S::SCALE_BYTES);
  uint64_t* full = bars;                                   // [ST] TMA -> MMA
  uint64_t* empty = bars + ST;                             // [ST] MMA -> TMA
  uint64_t* tmemFull = bars + 2 * ST;                      // MMA -> sums
  uint64_t* tmemEmpty = tmemFull + 1;                      // sums -> MMA
  uint64_t* sumFull = tmemFull + 2;                        // every rank's sums lie in its shared memory
  uint64_t* sumEmpty = tmemFull + 3;                       // every rank has read this rank's
  uint64_t* scaleFull = tmemFull + 4;                      // [kScaleSets]
  uint64_t* scaleEmpty = scaleFull + fp8::kScaleSets;      // [kScaleSets]
  uint64_t* drained = scaleEmpty + fp8::kScaleSets;        // after a wait has run out
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* sFail = reinterpret_cast<volatile int*>(tmemSlot + 1);
  int* sGroup = reinterpret_cast<int*>(tmemSlot + 2);      // this group's first row and end, the last group's end
  uint32_t* sLoads = tmemSlot + 5;                         // stages the producer has loaded

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slices = a.slices, rank = (int)(blockIdx.x % slices), n0 = (int)(blockIdx.x / slices) * BM, e = blockIdx.y;
  const uint64_t budget = a.budgetNs;

  if (warp == 3) {
    int before = 0, upTo = 0, last = 0;
    if (a.ends == nullptr) {
      upTo = last = a.rows;
    } else {
      for (int i = lane; i < a.groups; i += 32) {
        const int64_t v = a.ends64 ? static_cast<const int64_t*>(a.ends)[i] : (int64_t) static_cast<const int32_t*>(a.ends)[i];
        const int end = (int)(v < 0 ? 0 : v > a.rows ? a.rows : v);
        last = max(last, end);
        if (i <= e) upTo = max(upTo, end);
        if (i < e) before = max(before, end);
      }
      before = __reduce_max_sync(0xffffffffu, before);
      upTo = __reduce_max_sync(0xffffffffu, upTo);
      last = __reduce_max_sync(0xffffffffu, last);
    }
    if (lane == 0) { sGroup[0] = before; sGroup[1] = upTo; sGroup[2] = last; }
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) { umma::mbarInit(&full[s], 1); umma::mbarInit(&empty[s], 1); }
    umma::mbarInit(tmemFull, 1); umma::mbarInit(tmemEmpty, 4);
    umma::mbarInit(sumFull, slices); umma::mbarInit(sumEmpty, slices);
    for (int i = 0; i < fp8::kScaleSets; ++i) { umma::mbarInit(&scaleFull[i], 1); umma::mbarInit(&scaleEmpty[i], 1); }
    umma::mbarInit(drained, 1);
    *sFail = 0;
    umma::fenceBarrierInit();
    umma::prefetchTensorMap(&a.mapW);
    umma::prefetchTensorMap(&a.mapX);
  }
  __syncthreads();
  const int first = sGroup[0], count = sGroup[1] - first;
  // Rows behind the last group belong to nobody.
  if (rank == 0 && e == a.groups - 1 && blockIdx.z == 0)
    for (int64_t i = threadIdx.x; i < (int64_t)(a.rows - sGroup[2]) * 16; i += kThreads) {
      const int col = n0 + (int)(i & 15) * 8;
      if (col < a.N) *reinterpret_cast<uint4*>(a.out + ((size_t)sGroup[2] + (i >> 4)) * a.N + col) = make_uint4(0, 0, 0, 0);
    }
  if ((int64_t)blockIdx.z * BT >= count) {                 // no rows here: the same in all CTAs of the cluster
    waitForPredecessor();
    return;
  }
  const int kBlocks = (a.K + CK - 1) / CK, units = (kBlocks + UNIT - 1) / UNIT;
  const int kb0 = rank * units / slices * UNIT, kb1 = min((rank + 1) * units / slices * UNIT, kBlocks);
  const int64_t step = (int64_t)gridDim.z * BT, r0 = (int64_t)blockIdx.z * BT;
  const int early = min(ST, kb1 - kb0);                    // weights that wait for nothing
  if (threadIdx.x == 0)
    for (int i = 0; i < early; ++i) {
      umma::mbarExpectTx(&full[i], S::A_BYTES + S::B_BYTES);
      grouped::tmaLoad3d(sA + i * S::A_BYTES, &a.mapW, &full[i], (kb0 + i) * CK, n0, e);
    }
  if (warp == 2) { umma::tmemAlloc(tmemSlot, S::TMEM); umma::tmemRelinquish(); }
  umma::tcFenceBefore();
  __syncthreads();
  umma::tcFenceAfter();
  clusterArrive();                                         // this rank's barriers exist; the warps that reach for another's wait for its word
  const uint32_t tmemBase = *tmemSlot;

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer
    int stage = 0; uint32_t phase = 0, loads = 0;
    waitForPredecessor();
    // The first turn whatever another role says: the stages whose weights are requested get their rows.
    for (int64_t r = r0; r < count && (r == r0 || *sFail == 0); r += step) {
      for (int kb = kb0; kb < kb1; ++kb) {
        if (r != r0 || kb - kb0 >= early) {
          if (!umma::mbarWaitParked(&empty[stage], phase ^ 1, budget)) { *sFail = 1; atomicExch(a.errFlag, 51); break; }
          umma::mbarExpectTx(&full[stage], S::A_BYTES + S::B_BYTES);
          grouped::tmaLoad3d(sA + stage * S::A_BYTES, &a.mapW, &full[stage], kb * CK, n0, e);
        }
        umma::tmaLoad2d(sB + stage * S::B_BYTES, &a.mapX, &full[stage], kb * CK, first + (int)r);
        ++loads;
        if (++stage == ST) { stage = 0; phase ^= 1; }
      }
    }
    *sLoads = loads;
  } else if (warp == 1) {
    // ---------------- MMA issuer: the warp walks the loop together, one thread of it issues
    const bool issues = umma::electOne();
    const uint64_t descA0 = umma::smemDescSw128(sA), descB0 = umma::smemDescSw128(sB);
    const uint32_t aLo0 = (uint32_t)descA0, bLo0 = (uint32_t)descB0, hi = (uint32_t)(descA0 >> 32);
    const uint64_t descS0 = fp8::smemDescScales(sScale);
    const uint32_t sLo0 = (uint32_t)descS0, sHi = (uint32_t)(descS0 >> 32);
    int stage = 0, set = 0; uint32_t phase = 0, accPhase = 0, setPhase = 0;
    const uint32_t scaleBase = tmemBase + BT;
    for (int64_t r = r0; r < count; r += step) {
      if (!grouped::waitWarp<false>(tmemEmpty, accPhase ^ 1, budget, sFail)) { if (lane == 0) atomicExch(a.errFlag, 52); break; }
      umma::tcFenceAfter();
      bool ok = true;
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        const uint32_t sfa = scaleBase + (uint32_t)(set * 8), sfb = sfa + 4;
        if (FP8 && (kb & 3) == 0) {
          ok = umma::mbarWait(&scaleFull[set], setPhase, budget);
          umma::tcFenceAfter();
          if (issues && ok) {
            const uint32_t lo = sLo0 + (uint32_t)(set * (S::SCALE_BYTES >> 4));
            fp8::copyScales(sfa, lo, sHi);
            fp8::copyScales(sfb, lo + 32, sHi);
          }
        }
        ok = umma::mbarWait(&full[stage], phase, budget) && ok;
        umma::tcFenceAfter();
        const bool lastOfSet = FP8 && ((kb & 3) == 3 || kb == kb1 - 1);
        if (issues && ok) {
          const uint32_t aLo = aLo0 + (uint32_t)(stage * (S::A_BYTES >> 4)), bLo = bLo0 + (uint32_t)(stage * (S::B_BYTES >> 4));
          if (FP8) {
            const uint32_t idesc = fp8::instrDesc(BM, BT) + (uint32_t)(kb & 3) * fp8::kScaleByte;
            fp8::mmaScaled(tmemBase, aLo, bLo, hi, idesc, sfa, sfb, kb != kb0);
            fp8::mmaScaled(tmemBase, aLo + 2, bLo + 2, hi, idesc, sfa, sfb, 1);
            fp8::mmaScaled(tmemBase, aLo + 4, bLo + 4, hi, idesc, sfa, sfb, 1);
            fp8::mmaScaled(tmemBase, aLo + 6, bLo + 6, hi, idesc, sfa, sfb, 1);
          } else {
            constexpr uint32_t idesc = umma::instrDescBf16(BM, BT);
            umma::mmaBf16Split(tmemBase, aLo, hi, bLo, hi, idesc, kb != kb0);
            umma::mmaBf16Split(tmemBase, aLo + 2, hi, bLo + 2, hi, idesc, 1);
            umma::mmaBf16Split(tmemBase, aLo + 4, hi, bLo + 4, hi, idesc, 1);
            umma::mmaBf16Split(tmemBase, aLo + 6, hi, bLo + 6, hi, idesc, 1);
          }
          umma::mmaCommit(&empty[stage]);
          if (lastOfSet) umma::mmaCommit(&scaleEmpty[set]);
        }
        if (lastOfSet && ++set == fp8::kScaleSets) { set = 0; setPhase ^= 1; }
        if (++stage == ST) { stage = 0; phase ^= 1; }
      }
      if (!__all_sync(0xffffffffu, ok)) { *sFail = 1; if (lane == 0) atomicExch(a.errFlag, 54); break; }
      if (issues) umma::mmaCommit(tmemFull);
      accPhase ^= 1;
    }
  } else if (FP8 && warp == 3) {
    // ---------------- scales
    int set = 0; uint32_t setPhase = 0;
    bool ok = true;
    const uint8_t* col = a.sw + ((int64_t)e * ((a.N + BM - 1) / BM) + n0 / BM) * a.ldsw;
    waitForPredecessor();
    for (int64_t r = r0; r < count && ok; r += step) {
      const uint8_t* row[(BT + 31) / 32];
#pragma unroll
      for (int j = 0; j < (BT + 31) / 32; ++j) row[j] = a.sx + (int64_t)min(first + (int)r + j * 32 + lane, a.rows - 1) * a.ldsx;
      for (int i = kb0 / 4; i * 4 < kb1; ++i) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < (BT + 31) / 32; ++j) w[j] = fp8::scaleWord(row[j], i, kBlocks);
        const uint32_t c = fp8::scaleWord(col, i, kBlocks);
        if (!grouped::waitWarp<true>(&scaleEmpty[set], setPhase ^ 1, budget, sFail)) { if (lane == 0) atomicExch(a.errFlag, 55); ok = false; break; }
        uint4* to = reinterpret_cast<uint4*>(sScale + set * S::SCALE_BYTES) + lane;
        to[0] = make_uint4(c, c, c, c);
        to[32] = make_uint4(w[0], w[1], w[2], w[3]);
        umma::fenceProxyAsyncShared();
        __syncwarp();
        if (lane == 0) umma::mbarArrive(&scaleFull[set]);
        if (++set == fp8::kScaleSets) { set = 0; setPhase ^= 1; }
      }
    }
  } else if (warp >= 4) {
    // ---------------- sums: lane quarter q holds 32 of the weights' rows, a column a row of x
    const int q = warp & 3, et = threadIdx.x - 128;
    uint32_t parity = 0;
    const uint64_t others = budget + (uint64_t)kBlocks * a.blockNs;                  // until another rank's sums are there: its share, and what it waits for
    clusterWait();
    for (int64_t r = r0; r < count; r += step, parity ^= 1) {
      bool ok = grouped::waitWarpLong(tmemFull, parity, budget, kb1 - kb0, a.blockNs, sFail);
      if (!ok && lane == 0) atomicExch(a.errFlag, 56);
      if (ok && r != r0) ok = __all_sync(0xffffffffu, waitCluster(sumEmpty, parity ^ 1, others));
      if (gemm::namedBarrierOr(1, 128, !ok)) { *sFail = 1; break; }      // the four warps meet below: they leave together
      umma::tcFenceAfter();
#pragma unroll
      for (int c = 0; c < BT / 16; ++c) {
        uint32_t v[16];
        tmemLoad32x16(tmemBase + ((uint32_t)(q * 32) << 16) + c * 16u, v);
        umma::tmemLoadWait();
#pragma unroll
        for (int i = 0; i < 16; ++i) sSum[(c * 16 + i) * BM + q * 32 + lane] = __uint_as_float(v[i]);
      }
      umma::tcFenceBefore();
      __syncwarp();
      if (lane == 0) umma::mbarArrive(tmemEmpty);
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (et < slices) arriveCluster(sumFull, et);
      ok = __all_sync(0xffffffffu, waitCluster(sumFull, parity, others));
      if (!ok && lane == 0) atomicExch(a.errFlag, 57);
      if (gemm::namedBarrierOr(1, 128, !ok)) { *sFail = 1; break; }
      // Rank p of the cluster stores the rows p, p + slices, ...: a warp a row, four columns a lane.
      const int valid = (int)min((int64_t)BT, count - r), col = n0 + lane * 4;
      for (int t = rank + q * slices; t < valid; t += 4 * slices) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        const uint32_t from = umma::smemAddr(sSum + t * BM + lane * 4);
        float4 x[8];
#pragma unroll
        for (int p = 0; p < 8; ++p) if (p < slices) x[p] = loadCluster(gemm::umma2::mapToCta(from, p));
#pragma unroll
        for (int p = 0; p < 8; ++p) if (p < slices) { s.x += x[p].x; s.y += x[p].y; s.z += x[p].z; s.w += x[p].w; }
        if (col < a.N) {
          __nv_bfloat162 lo = __floats2bfloat162_rn(s.x, s.y), hi = __floats2bfloat162_rn(s.z, s.w);
          *reinterpret_cast<uint2*>(a.out + ((size_t)first + r + t) * a.N + col) =
              make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (et < slices) arriveCluster(sumEmpty, et);
    }
  }

  if (warp < 4) clusterWait();
  waitForPredecessor();                                    // this grid's end stands for its predecessor's too
  umma::tcFenceBefore();
  __syncthreads();
  if (*sFail != 0) {                                       // the same for all threads
    if (threadIdx.x == 0) grouped::drainLoads(full, ST, *sLoads);
    if (warp == 1) grouped::drainProducts(drained);
    __syncthreads();
  }
  gemm::umma2::clusterSync();                              // no rank leaves while another reads its sums
  if (warp == 2) umma::tmemDealloc(tmemBase, S::TMEM);
}

}  // namespace thin
}  // namespace mccl
