// Product of e4m3 matrices with one fp32 scale per block of 128: A in blocks of 1 x 128 along the inner dimension, B in
// tiles of 128 x 128.
//
//   C[m, n] = sum over kb of  sa(m, kb) * sb(n / 128, kb) * sum over k in block kb of A[m, k] * B[n, k]
//
// The tensor core multiplies one block of 128 at a time into a fresh accumulator in TMEM; eight warps take each one out
// and add it, scaled, to sums in registers (fp32, one rounding an addition; the product of the two scales is rounded too).
// Operands may be stored transposed, as in gemm_tc2.cu: the two gradients of a linear layer contract over a dimension
// that is not the contiguous one.
//
// PAIR: two CTAs of a cluster share one tile of 256 rows (cta_group::2), each with its 128 rows of A, half of the tile's
// rows of B and its half of the accumulator; the leader (cluster rank 0) issues for both.
//
// Without PAIR a tile of 128 rows is one CTA's, or that of a cluster of up to eight which share out the blocks along K
// (few tiles, so that the others of the chip's SMs load and multiply too).  Each then leaves its sums in its shared memory
// and adds up its share of the tile's rows from all of them, in the order of the blocks: the same bits every time.  (Sending
// them instead, with stores or bulk copies to the other CTAs' shared memory, took 1 - 2 us longer for 128 rows.)
//
// POW2 (with PAIR): the caller says that all scales are powers of two, as this library's own encoding makes them.  Then the
// tensor core applies them itself (kind::mxf8f6f4, a scale byte for each 32 elements: four alike) and adds up a whole tile;
// a scale that is not one counts as NaN.
//
//   warps 0..7   sums: a thread has one row and half of the tile's columns; then they store C
//   warp 8       TMA producer: own halves of A and B; the bytes of both CTAs count on the leader's "stage full" barrier
//   warp 9       (leader) issues tcgen05.mma: four a stage; commits to "stage empty" and "accumulator full" of both CTAs
//   warps 10, 11 scales: the products sa * sb of a block for the CTA's rows and both halves, blocks ahead of their use
//
// Measured (bf16 out, scales of any value / powers of two): 8192 x 1792 x 4096 63 / 50 us, 8192 x 4096 x 4096 131 / 100 (2.1 / 2.75
// PFLOP/s).  With scales of any value the sum warps' chain is the bound: about 380 cycles a block and 128 columns, where the
// tensor core and its operands' way through shared memory need 340.  A product's loads are 7.2 % of the HBM's time then.
// Tiles of 128 columns with four accumulators: with 256 columns and two, the tensor core waits for the sums after every
// block (890 cycles for the 256); POW2 has tiles of 256, whose only accumulator is drained once a tile.
//
// Every wait is bounded; on expiry the CTA raises its abort flag, all roles leave their loops, TMEM is freed and the
// device's error word is set, until fp8_gemm_error reads it.
//
// The reference has no compute kernels (README.md:5 only asks that collectives fuse with others).
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../device/prims.cuh"
#include "../device/reduce_ops.cuh"
#include "../device/tc_prims.cuh"
#include "../device/tc_wait.cuh"
#include "fp8.h"
#include "launch.h"

namespace mt {
using namespace tc;
namespace fp8g {

constexpr int BM = 128, BK = 128;   // rows of a CTA
constexpr int kSumWarps = 8, kSumThreads = 32 * kSumWarps, kThreads = kSumThreads + 128;
// Registers a thread after the split of the launch's own; the launch has to bring at least kRegsLaunch (checked on the host).
constexpr int kRegsSum = 224, kRegsRest = 56, kRegsLaunch = 168;
static_assert(kRegsSum * kSumThreads + kRegsRest * 128 <= kRegsLaunch * kThreads, "registers of the CTA");
constexpr int kScaleSlots = 16;     // blocks whose scales wait in shared memory
constexpr int kPitch = 144;         // bytes of a staged row of C: 128 and padding
constexpr int kSumPitch = 132;      // floats of a row of sums in shared memory
constexpr uint32_t A_BYTES = BM * BK, TMEM_COLS = 512;

template <int BN, bool PAIR, bool POW2 = false>
struct Shape {
  static constexpr int BNC = PAIR ? BN / 2 : BN;          // rows of B staged by a CTA
  static constexpr uint32_t B_BYTES = BNC * BK;
  static constexpr int STAGES = PAIR && BN == 128 ? 7 : 5;
  static constexpr uint32_t SF_BYTES = 512 * (1 + BN / 128);   // POW2: scale bytes of a stage, A's rows and B's
  static constexpr int ACC = POW2 ? 256 / BN : TMEM_COLS / BN;   // accumulators (POW2: the columns behind them hold scales)
  static constexpr uint32_t OPERANDS = STAGES * (A_BYTES + B_BYTES);
  static constexpr uint32_t RING = POW2 ? STAGES * SF_BYTES : kScaleSlots * 2 * BM * 4, STAGING = kSumWarps * 32 * kPitch;
  static constexpr uint32_t SMEM = 1024 + OPERANDS + RING + STAGING + 256;
  static_assert(SMEM <= 232448, "shared memory of one CTA");
  static_assert(PAIR || OPERANDS >= BM * kSumPitch * 4, "the sums of a split tile are left where the stages were");
};
struct Ctl {
  uint64_t full[7], empty[7], acc_full[4], acc_empty[4], drain;
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(Ctl) <= 256, "control block");

__device__ int g_error;

// Two sums in a register pair: one instruction adds to both, which leaves issue slots to the warps that feed the tensor core.
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t p, uint64_t f) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(p), "l"(f));
}

// Tile t: groups of 16 row blocks, in a group row block fastest, so that a wave's operands stay in the L2.
__device__ __forceinline__ void tile_of(int t, int mt_, int nt, int* mb, int* nb) {
  const int per = 16 * nt, gr = t / per, in = t - gr * per, rows = min(16, mt_ - gr * 16);
  *nb = in / rows;
  *mb = gr * 16 + in - *nb * rows;
}

// The sums of a warp's 32 rows and CW columns to C, 128 bytes of every row at a time through shared memory, so that stores
// are whole lines: 16 bytes a lane where C's rows are aligned to that, else neighbouring elements on neighbouring lanes.
template <class T, int CW>
__device__ __forceinline__ void store_sums(const Fp8GemmArgs& a, const uint64_t* acc, uint8_t* stg, int row0, int col, int lane) {
  using E = typename T::elem;
  constexpr int kE = (int)sizeof(E), kPer = 128 / kE;   // columns of a round
  static_assert(CW % kPer == 0, "whole rounds");
  const int n = min(CW, a.N - col), rows = min(32, a.M - row0);
  uint8_t* base = (uint8_t*)a.c + ((int64_t)row0 * a.ldc + col) * kE;
#pragma unroll
  for (int r = 0; r < CW / kPer; ++r) {
    uint4* mine = (uint4*)(stg + lane * kPitch);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f[16 / kE];
#pragma unroll
      for (int i = 0; i < 8 / kE; ++i) {
        const float2 x = unpack2(acc[(r * kPer + j * 16 / kE) / 2 + i]);
        f[2 * i] = x.x;
        f[2 * i + 1] = x.y;
      }
      const uint64_t lo = T::pack(f), hi = T::pack(f + T::kPer64);
      mine[j] = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
    }
    __syncwarp();
    if (a.vec_out && n == CW) {
      const int c16 = lane & 7;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const int rr = p * 4 + (lane >> 3);
        if (rr < rows) *(uint4*)(base + ((int64_t)rr * a.ldc + r * kPer) * kE + c16 * 16) = *(const uint4*)(stg + rr * kPitch + c16 * 16);
      }
    } else {
      E* to = (E*)base + r * kPer + lane;
#pragma unroll 4
      for (int rr = 0; rr < rows; ++rr, to += a.ldc) {
        const E* from = (const E*)(stg + rr * kPitch) + lane;
#pragma unroll
        for (int i = 0; i < kPer; i += 32)
          if (r * kPer + i + lane < n) to[i] = from[i];
      }
    }
    __syncwarp();
  }
}

// This CTA's share of a split tile's rows to C: the sums of all CTAs of the cluster, four columns a thread, two rows' loads
// in flight.
template <class T, int SPLIT>
__device__ __forceinline__ void store_split(const Fp8GemmArgs& a, uint32_t sums, int rank, int row0, int col0) {
  using E = typename T::elem;
  constexpr int kRowsEach = BM / SPLIT;
  const int c = (threadIdx.x & 31) * 4, n = a.N - (col0 + c);
  if (n <= 0) return;
#pragma unroll 2
  for (int i = threadIdx.x >> 5; i < kRowsEach; i += kSumWarps) {
    const int r = rank * kRowsEach + i, row = row0 + r;
    if (row >= a.M) break;
    float4 x[SPLIT];
#pragma unroll
    for (int s = 0; s < SPLIT; ++s) x[s] = ld_cluster_f4(map_to_cta(sums + (r * kSumPitch + c) * 4, s));
    float f[4] = {x[0].x, x[0].y, x[0].z, x[0].w};
#pragma unroll
    for (int s = 1; s < SPLIT; ++s) {
      f[0] += x[s].x;
      f[1] += x[s].y;
      f[2] += x[s].z;
      f[3] += x[s].w;
    }
    E* to = (E*)a.c + (int64_t)row * a.ldc + col0 + c;
    if (a.vec_out && n >= 4) {
      if constexpr (sizeof(E) == 4) *(float4*)to = make_float4(f[0], f[1], f[2], f[3]);
      else *(uint64_t*)to = T::pack(f);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < n) to[j] = float_to_elem<T>(f[j]);
    }
  }
}
template <class T>
__device__ __forceinline__ void store_split(const Fp8GemmArgs& a, uint32_t sums, int split, int rank, int row0, int col0) {
  if (split == 2) store_split<T, 2>(a, sums, rank, row0, col0);
  else if (split == 4) store_split<T, 4>(a, sums, rank, row0, col0);
  else store_split<T, 8>(a, sums, rank, row0, col0);
}

// The ue8m0 byte of a power of two, four times; NaN for anything else.
__device__ __forceinline__ uint32_t scale_byte4(float s) {
  const uint32_t b = __float_as_uint(s), e = b >> 23;
  return ((b & 0x7fffffu) == 0 && e - 1u < 254u ? e : 255u) * 0x01010101u;
}

template <int BN, bool PAIR, bool POW2, bool TA, bool TB>
__global__ void __launch_bounds__(kThreads, 1) gemm_fp8_kernel(const __grid_constant__ Fp8GemmArgs a) {
  static_assert(PAIR || !POW2, "the tensor core applies scales on pairs");
  static_assert(!POW2 || Shape<BN, PAIR, POW2>::ACC * BN + Shape<BN, PAIR, POW2>::STAGES * 16 <= TMEM_COLS, "columns of TMEM");
  using S = Shape<BN, PAIR, POW2>;
  constexpr int STAGES = S::STAGES, ACC = S::ACC, BNC = S::BNC, CW = BN / 2;   // CW: columns of a sum thread
  constexpr uint32_t B_BYTES = S::B_BYTES;
  constexpr int kRows = PAIR ? 2 * BM : BM;   // of a tile
  static_assert(BNC == 128 || BNC == 64, "columns of B that a CTA stages: one chunk");
  extern __shared__ uint8_t smem_raw[];
  // the same offsets in both CTAs: the MMA descriptors name shared memory of the pair by offset
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  float* sScale = (float*)(smem + S::OPERANDS);
  uint8_t* sOut = (uint8_t*)sScale + S::RING;
  Ctl* ctl = (Ctl*)(sOut + S::STAGING);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int cr = PAIR ? (int)cluster_ctarank() : 0;

  const int mt_ = (a.M + kRows - 1) / kRows, nt = (a.N + BN - 1) / BN, tiles = mt_ * nt, allblocks = (a.K + BK - 1) / BK;
  // a split tile is the only one of its cluster
  const int split = PAIR ? 1 : (int)cluster_nctas(), share = PAIR ? 0 : (int)cluster_ctarank();
  const int group = PAIR ? 2 : split, first = (int)blockIdx.x / group, step = (int)gridDim.x / group;
  const int kfirst = allblocks * share / split, kblocks = allblocks * (share + 1) / split - kfirst;

  // one stage of tile (mb, nb), by one thread
  auto load_stage = [&](uint32_t s, int mb, int nb, int kb) {
    const int arow = mb * kRows + cr * BM, brow = nb * BN + cr * BNC, k = (kfirst + kb) * BK;
    const uint32_t full = PAIR ? map_to_cta(smem_u32(&ctl->full[s]), 0) : 0;
    auto load = [&](uint8_t* dst, const CUtensorMap* map, int x, int y) {
      if (PAIR) tma_load_2d_pair(dst, map, x, y, full);
      else tma_load_2d(dst, map, x, y, &ctl->full[s]);
    };
    if (cr == 0) mbar_expect_tx(&ctl->full[s], (PAIR ? 2 : 1) * (A_BYTES + B_BYTES));
    if (TA) load(sA + s * A_BYTES, &a.a, arow, k);
    else load(sA + s * A_BYTES, &a.a, k, arow);
    if (TB) load(sB + s * B_BYTES, &a.b, brow, k);
    else load(sB + s * B_BYTES, &a.b, k, brow);
  };
  // the first tile's stages that need not wait for anything (a pair has to meet first)
  const int early = PAIR || first >= tiles ? 0 : min(STAGES, kblocks);
  if (warp == kSumWarps) {
    if (elect_one()) {
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(&ctl->full[s], PAIR ? 3 : 2);   // the producer's byte count and the scales of each CTA
        mbar_init(&ctl->empty[s], 1);
      }
      for (int s = 0; s < ACC; ++s) {
        mbar_init(&ctl->acc_full[s], POW2 ? 1 : 2);   // the products; of a block also the CTA's own scale warp
        mbar_init(&ctl->acc_empty[s], PAIR ? 2 * kSumWarps : kSumWarps);   // the leader's counts both CTAs
      }
      mbar_init(&ctl->drain, 1);
      ctl->abort = 0;
      fence_barrier_init();
      if (early) {
        int mb, nb;
        tile_of(first, mt_, nt, &mb, &nb);
        for (int s = 0; s < early; ++s) load_stage(s, mb, nb, s);
      }
    }
    __syncwarp();
  }
  if (warp == kSumWarps + 1) {
    if (PAIR) {
      tmem_alloc_pair(&ctl->tmem_base, TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&ctl->tmem_base, TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();   // both CTAs' barriers exist before anybody signals across
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
  volatile int* abort_flag = &ctl->abort;

  if (warp >= kSumWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
    if (warp == kSumWarps) {
      // ---------------------------------------------------------- TMA producer: a uniform warp, one lane issues
      uint32_t s = early == STAGES ? 0 : early, ph = early == STAGES;
      bool ok = true, free = early < STAGES;   // free: a probe found the next stage empty
      for (int t = first; ok && t < tiles; t += step) {
        int mb, nb;
        tile_of(t, mt_, nt, &mb, &nb);
        for (int kb = t == first ? early : 0; kb < kblocks; ++kb) {
          if (!free && !wait_bar_warp(&ctl->empty[s], ph ^ 1, abort_flag, a.timeout_ns)) {
            ok = false;
            break;
          }
          const uint32_t sn = s + 1 == STAGES ? 0 : s + 1, phn = s + 1 == STAGES ? ph ^ 1 : ph;
          free = __all_sync(0xffffffffu, mbar_test(&ctl->empty[sn], phn ^ 1));
          if (elect_one()) load_stage(s, mb, nb, kb);
          __syncwarp();
          s = sn;
          ph = phn;
        }
      }
      if (aborted_warp(abort_flag)) {
        // copies in flight may still be landing in shared memory: give them a bounded time
        const uint64_t t0 = globaltimer();
        while (globaltimer() - t0 < 100000ull) __nanosleep(1000);
      }
    } else if (warp == kSumWarps + 1 && cr == 0) {
      // ---------------------------------------------------------- MMA issuer: uniform, one lane issues
      constexpr uint32_t trans = (TA ? kIdescTransA : 0u) | (TB ? kIdescTransB : 0u), idesc = make_idesc_e4m3(kRows, BN) | trans;
      // a step of 32 along K: 32 bytes of a row, or 32 rows of 128 bytes
      constexpr uint64_t step_a = TA ? 256 : 2, step_b = !TB ? 2 : BNC == 128 ? 256 : 128;
      uint32_t s = 0, ph = 0, b = 0, bph = 0;
      bool ok = true;
      auto commit = [&](uint64_t* bar) {
        if (PAIR) umma_commit_both(bar);
        else umma_commit(bar);
      };
      for (int t = first; ok && t < tiles; t += step) {
        for (int kb = 0; kb < kblocks; ++kb) {
          // an accumulator is one block's, with POW2 a whole tile's
          const bool fresh = !POW2 || kb == 0, done = !POW2 || kb + 1 == kblocks;
          // both probes in flight at once: each takes some 230 cycles beside the tensor core's own shared-memory traffic
          const bool drained = !fresh || mbar_test(&ctl->acc_empty[b], bph ^ 1),
                     loaded = POW2 ? mbar_test_cluster(&ctl->full[s], ph) : mbar_test(&ctl->full[s], ph);
          if (!__all_sync(0xffffffffu, drained && loaded) &&
              ((fresh && !wait_bar_warp(&ctl->acc_empty[b], bph ^ 1, abort_flag, a.timeout_ns)) ||
               !wait_bar_warp<POW2>(&ctl->full[s], ph, abort_flag, a.timeout_ns))) {
            ok = false;
            break;
          }
          if (POW2) fence_acquire_cluster_smem();   // scales that threads of both CTAs have written
          tc_fence_after();
          const uint64_t da = TA ? make_smem_desc_mn_sw128(sA + s * A_BYTES, 128 * BK) : make_smem_desc_sw128(sA + s * A_BYTES);
          const uint64_t db = !TB          ? make_smem_desc_sw128(sB + s * B_BYTES)
                              : BNC == 128 ? make_smem_desc_mn_sw128(sB + s * B_BYTES, 128 * BK)
                                           : make_smem_desc_mn_sw64(sB + s * B_BYTES);
          if (elect_one()) {
            if constexpr (POW2) {
              const uint32_t sfa = tmem_base + ACC * BN + s * 16, sfb = sfa + 4;
              const uint8_t* sf = (const uint8_t*)sScale + s * S::SF_BYTES;
              tmem_cp_sf_pair(sfa, make_smem_desc_sf(sf));
              tmem_cp_sf_pair(sfb, make_smem_desc_sf(sf + 512));
              if (BN > 128) tmem_cp_sf_pair(sfb + 4, make_smem_desc_sf(sf + 1024));
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_mxfp8_pair(tmem_base + b * BN, da + k * step_a, db + k * step_b, make_idesc_mxfp8(kRows, BN, k, k) | trans, sfa, sfb,
                                kb > 0 || k > 0 ? 1u : 0u);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (PAIR) umma_f8_pair(tmem_base + b * BN, da + k * step_a, db + k * step_b, idesc, k > 0 ? 1u : 0u);
                else umma_f8(tmem_base + b * BN, da + k * step_a, db + k * step_b, idesc, k > 0 ? 1u : 0u);
              }
            }
            commit(&ctl->empty[s]);
            if (done) commit(&ctl->acc_full[b]);
          }
          __syncwarp();
          if (++s == STAGES) {
            s = 0;
            ph ^= 1;
          }
          if (done && ++b == ACC) {
            b = 0;
            bph ^= 1;
          }
        }
      }
      // no MMA may still be writing TMEM when it is freed
      if (elect_one()) {
        if (PAIR) umma_commit_pair(smem_u32(&ctl->drain));
        else umma_commit(&ctl->drain);
      }
      __syncwarp();
      wait_bar_warp(&ctl->drain, 0, abort_flag, a.timeout_ns);
    } else if (warp >= kSumWarps + 2) {
      // ---------------------------------------------------------- scales: one warp for even blocks, one for odd; a lane has
      // four rows, 32 apart.  They count on the stage's "full" barrier, so that no block overtakes its scales: a slot is free
      // when its stage is, the sums are at most ACC + STAGES blocks behind and have used what was there.  With POW2 the tensor
      // core reads the bytes of both CTAs: the leader, which waits for "full" and issues for both, sees them by the fences of
      // the two.  Factors are for the sum warps of the same CTA: they count on its "accumulator full" barrier as well, once the
      // block before on that accumulator has come out.  (A barrier of their own for the sums to wait on, on whose time
      // everything hangs: 8192 x 4096 x 4096 136 us, with one for four blocks 142, this way 131.)
      static_assert(POW2 || (ACC + STAGES < kScaleSlots && ACC == 4), "slots of the scales, their accumulators");
      const int w = warp - kSumWarps - 2;
      const uint32_t full_leader = map_to_cta(smem_u32(&ctl->full[0]), 0);
      uint32_t s = w, ph = 0, pos = 0;   // stage of this warp's next block, and the tile's first block among all
      bool ok = true;
      for (int t = first; ok && t < tiles; t += step, pos += kblocks) {
        int mb, nb;
        tile_of(t, mt_, nt, &mb, &nb);
        const int row = mb * kRows + cr * BM + lane, c0 = nb * BN, c1 = c0 + CW;
        const float* pa[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pa[i] = a.sa + (int64_t)(row + 32 * i < a.M ? row + 32 * i : 0) * a.sa_m + kfirst * a.sa_k;
        const float* pb0 = a.sb + (int64_t)(c0 >> 7) * a.sb_n + kfirst * a.sb_k;
        const float* pb1 = a.sb + (int64_t)(c1 < a.N ? c1 >> 7 : 0) * a.sb_n + kfirst * a.sb_k;
        for (int kb = (pos + w) & 1; ok && kb < kblocks; kb += 4) {
          float va[2][4], vb[2][2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int64_t k = min(kb + 2 * j, kblocks - 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) va[j][i] = __ldg(pa[i] + k * a.sa_k);
            vb[j][0] = __ldg(pb0 + k * a.sb_k);
            vb[j][1] = __ldg(pb1 + k * a.sb_k);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (!ok || kb + 2 * j >= kblocks) continue;
            ok = wait_bar_warp(&ctl->empty[s], ph ^ 1, abort_flag, a.timeout_ns);
            if constexpr (POW2) {
              // byte (r % 32) * 16 + (r / 32) * 4 + k of an atom is row r's scale of the k-th 32 elements
              uint4* sf = (uint4*)((uint8_t*)sScale + s * S::SF_BYTES) + lane;
              const uint32_t eb = scale_byte4(vb[j][0]), eb1 = scale_byte4(vb[j][1]);
              sf[0] = make_uint4(scale_byte4(va[j][0]), scale_byte4(va[j][1]), scale_byte4(va[j][2]), scale_byte4(va[j][3]));
              sf[32] = make_uint4(eb, eb, eb, eb);
              if (BN > 128) sf[64] = make_uint4(eb1, eb1, eb1, eb1);
              fence_proxy_async_smem();
            } else {
              float* f = sScale + ((pos + kb + 2 * j) & (kScaleSlots - 1)) * (2 * BM) + lane;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                f[32 * i] = va[j][i] * vb[j][0];
                f[BM + 32 * i] = va[j][i] * vb[j][1];
              }
            }
            __syncwarp();
            if (lane == 0) {
              if (POW2) mbar_arrive_cluster_release(full_leader + s * 8);
              else if (PAIR) mbar_arrive_cluster(full_leader + s * 8);
              else mbar_arrive(&ctl->full[s]);
            }
            if constexpr (!POW2) {
              const uint32_t n = pos + kb + 2 * j, b = n & (ACC - 1);
              ok = ok && wait_bar_warp(&ctl->acc_full[b], (n / ACC & 1) ^ 1, abort_flag, a.timeout_ns);
              if (ok && lane == 0) mbar_arrive(&ctl->acc_full[b]);
              __syncwarp();
            }
            s += 2;
            if (s >= STAGES) {
              s -= STAGES;
              ph ^= 1;
            }
          }
        }
      }
    }
    if (!PAIR && split > 1) {   // as the sum warps do
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    // ------------------------------------------------------------ sums and C
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSum));
    const int q = warp & 3, half = warp >> 2;   // TMEM lane quarter, half of the columns
    const uint32_t empty_leader = map_to_cta(smem_u32(&ctl->acc_empty[0]), 0);
    uint8_t* stg = sOut + warp * 32 * kPitch;
    const float* factor = sScale + half * BM + q * 32 + lane;
    uint32_t pos = 0, b = 0, bph = 0;
    bool ok = true, ready = false;   // ready: a probe found the next accumulator full
    for (int t = first; ok && t < tiles; t += step) {
      int mb, nb;
      tile_of(t, mt_, nt, &mb, &nb);
      const int row0 = mb * kRows + cr * BM + q * 32, col = nb * BN + half * CW;
      const bool work = row0 < a.M && col < a.N;   // the same for the whole warp
      uint64_t acc[CW / 2];
#pragma unroll
      for (int i = 0; i < CW / 2; ++i) acc[i] = 0;
      for (int kb = 0; kb < (POW2 ? 1 : kblocks); ++kb) {
        // one answer for all lanes
        if (!__all_sync(0xffffffffu, ready || wait_bar(&ctl->acc_full[b], bph, abort_flag, a.timeout_ns))) {
          ok = false;
          break;
        }
        tc_fence_after();
        // all columns to registers, and the accumulator back to the tensor core before they are added
        const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + b * BN + half * CW;
        const uint32_t bn = b + 1 == ACC ? 0 : b + 1, bphn = b + 1 == ACC ? bph ^ 1 : bph;
        uint32_t r[CW / 32][32];
#pragma unroll
        for (int c = 0; c < CW / 32; ++c) tmem_ld_32x32(taddr + c * 32, r[c]);
        const uint32_t f = POW2 ? 0u : __float_as_uint(factor[(pos++ & (kScaleSlots - 1)) * (2 * BM)]);
        const uint64_t f2 = pack2(f, f);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster(empty_leader + b * 8);
          else mbar_arrive(&ctl->acc_empty[b]);
        }
        ready = mbar_test(&ctl->acc_full[bn], bphn);   // known by the time it is needed
#pragma unroll
        for (int c = 0; c < CW / 32; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (POW2) acc[c * 16 + i] = pack2(r[c][2 * i], r[c][2 * i + 1]);
            else fma2(acc[c * 16 + i], pack2(r[c][2 * i], r[c][2 * i + 1]), f2);
          }
        b = bn;
        bph = bphn;
      }
      if (!PAIR && split > 1) {
        // all products have arrived: the stages are free
        float* mine = (float*)smem + (q * 32 + lane) * kSumPitch + half * CW;
#pragma unroll
        for (int i = 0; i < CW / 4; ++i) {
          const float2 x = unpack2(acc[2 * i]), y = unpack2(acc[2 * i + 1]);
          *(float4*)(mine + 4 * i) = make_float4(x.x, x.y, y.x, y.y);
        }
      } else if (ok && work) {
        if (a.out_dtype == DT_F32) store_sums<F32, CW>(a, acc, stg, row0, col, lane);
        else if (a.out_dtype == DT_BF16) store_sums<BF16, CW>(a, acc, stg, row0, col, lane);
        else store_sums<F16, CW>(a, acc, stg, row0, col, lane);
      }
    }
    if (!PAIR && split > 1) {
      int mb, nb;
      tile_of(first, mt_, nt, &mb, &nb);
      const uint32_t sums = smem_u32(smem);
      cluster_sync_all();   // the sums of all are in place
      if (a.out_dtype == DT_F32) store_split<F32>(a, sums, split, share, mb * BM, nb * BN);
      else if (a.out_dtype == DT_BF16) store_split<BF16>(a, sums, split, share, mb * BM, nb * BN);
      else store_split<F16>(a, sums, split, share, mb * BM, nb * BN);
      __syncwarp();
      cluster_sync_all();   // nobody leaves while its sums may still be read
    }
  }

  // ---------------------------------------------------------------- tear-down
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) {
    if (PAIR) st_cluster_u32(map_to_cta(smem_u32(&ctl->abort), cr ^ 1), 1u);   // the peer would notice after its own time limit
    atomicExch(&g_error, 1);
  }
  if (PAIR) cluster_sync_all();   // neither CTA leaves, or frees TMEM, while the other may still signal into it
  if (warp == kSumWarps + 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int BN, bool PAIR, bool POW2, bool TA, bool TB>
cudaError_t go(const Fp8GemmArgs& a, int cluster, int nctas, cudaStream_t s) {
  const void* fn = (const void*)gemm_fp8_kernel<BN, PAIR, POW2, TA, TB>;
  static std::atomic<uint64_t> ready{0};   // devices on which the kernel has been looked over and given its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev > 63 || !(ready.load(std::memory_order_acquire) & bit)) {
    cudaFuncAttributes at;
    if ((e = cudaFuncGetAttributes(&at, fn)) != cudaSuccess) return e;
    if (at.numRegs < kRegsLaunch) return cudaErrorLaunchOutOfResources;   // the register split would wait forever for what is missing
    if ((e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<BN, PAIR, POW2>::SMEM)) != cudaSuccess) return e;
    if (dev <= 63) ready.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(nctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Shape<BN, PAIR, POW2>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, gemm_fp8_kernel<BN, PAIR, POW2, TA, TB>, a);
}
template <int BN, bool PAIR, bool POW2>
cudaError_t go_form(bool ta, bool tb, const Fp8GemmArgs& a, int cluster, int nctas, cudaStream_t s) {
  if (ta) return go<BN, PAIR, POW2, true, true>(a, cluster, nctas, s);
  return tb ? go<BN, PAIR, POW2, false, true>(a, cluster, nctas, s) : go<BN, PAIR, POW2, false, false>(a, cluster, nctas, s);
}

// Self test: a wait that nothing ends, for 1 ms.
__global__ void expire_kernel() {
  __shared__ uint64_t bar;
  __shared__ int abort;
  mbar_init(&bar, 1);
  abort = 0;
  if (!wait_bar(&bar, 0, &abort, 1000000ull)) atomicExch(&g_error, 1);
}

}  // namespace fp8g

cudaError_t launch_fp8_gemm(int bn, bool pair, bool pow2, int split, bool ta, bool tb, const Fp8GemmArgs& a, int nctas, cudaStream_t s) {
  if ((ta && !tb) || split < 1 || (pair && split > 1) || (bn != 128 && !(bn == 256 && pair && pow2))) return cudaErrorInvalidValue;
  count_launch();
  if (bn == 256) return fp8g::go_form<256, true, true>(ta, tb, a, 2, nctas, s);
  if (pair) return pow2 ? fp8g::go_form<128, true, true>(ta, tb, a, 2, nctas, s) : fp8g::go_form<128, true, false>(ta, tb, a, 2, nctas, s);
  return fp8g::go_form<128, false, false>(ta, tb, a, split, nctas, s);
}

cudaError_t fp8_gemm_error(int* expired) {
  cudaError_t e = cudaDeviceSynchronize();   // products on every stream, those too that the copy would not wait for
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(expired, fp8g::g_error, sizeof(int));
  const int none = 0;
  if (e == cudaSuccess && *expired) e = cudaMemcpyToSymbol(fp8g::g_error, &none, sizeof(int));
  return e;
}

cudaError_t launch_fp8_gemm_expire(cudaStream_t s) {
  fp8g::expire_kernel<<<1, 1, 0, s>>>();
  return cudaGetLastError();
}

}  // namespace mt
