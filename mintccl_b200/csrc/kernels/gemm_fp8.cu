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
//   warps 0..7  sums: a thread has one row and half of the tile's columns; then they store C
//   warp 8      TMA producer: 128 rows of A and BN of B a stage, 128 bytes each
//   warp 9      issues tcgen05.mma: four a stage; commits to "stage empty" and "accumulator full"
//
// Every wait is bounded; on expiry the CTA raises its abort flag, all roles leave their loops, TMEM is freed and a
// device-side error word is set for the host.
//
// The reference has no compute kernels (README.md:5 only asks that collectives fuse with others).
#include <cuda.h>
#include <cuda_runtime.h>

#include "../device/prims.cuh"
#include "../device/reduce_ops.cuh"
#include "../device/tc_prims.cuh"
#include "../device/tc_wait.cuh"
#include "fp8.h"
#include "launch.h"

namespace mt {
using namespace tc;
namespace fp8g {

constexpr int BM = 128, BK = 128;
constexpr int kSumWarps = 8, kThreads = 32 * (kSumWarps + 2);
constexpr uint32_t A_BYTES = BM * BK, CHUNK = 128 * 128, TMEM_COLS = 512;

template <int BN>
struct Shape {
  static constexpr int STAGES = BN == 256 ? 4 : 6;
  static constexpr int ACC = BN == 256 ? 2 : 4;   // accumulators in TMEM
  static constexpr uint32_t B_BYTES = BN * BK;
  static constexpr uint32_t SMEM = 1024 + STAGES * (A_BYTES + B_BYTES) + 256;
};
struct Ctl {
  uint64_t full[6], empty[6], acc_full[4], acc_empty[4], drain;
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(Ctl) <= 256, "control block");

__device__ int g_error;

__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
// acc += p * f on two floats at once
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t p, uint64_t f) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(p), "l"(f));
}

// Tile t: groups of 16 row blocks, in a group row block fastest, so that a wave's operands stay in the L2.
__device__ __forceinline__ void tile_of(int t, int mt_, int nt, int* mb, int* nb) {
  const int per = 16 * nt, gr = t / per, in = t - gr * per, rows = min(16, mt_ - gr * 16);
  *nb = in / rows;
  *mb = gr * 16 + in - *nb * rows;
}

// 32 sums of one row to C: whole vectors, or elements where the row is not aligned or ends.
template <class T>
__device__ __forceinline__ void store32(uint8_t* p, const uint64_t* acc, int n, bool vec) {
  using E = typename T::elem;
  float f[32];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 t = unpack2(acc[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
  if (vec && n >= 32) {
    constexpr int kPer = 2 * T::kPer64;   // elements of a 16-byte vector
#pragma unroll
    for (int i = 0; i < 32 / kPer; ++i) {
      const uint64_t lo = T::pack(f + i * kPer), hi = T::pack(f + i * kPer + T::kPer64);
      *(uint4*)(p + 16 * i) = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
    }
  } else {
    E* e = (E*)p;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n) e[i] = float_to_elem<T>(f[i]);
  }
}

template <int BN, bool TA, bool TB>
__global__ void __launch_bounds__(kThreads, 1) gemm_fp8_kernel(const __grid_constant__ Fp8GemmArgs a) {
  using S = Shape<BN>;
  constexpr int STAGES = S::STAGES, ACC = S::ACC, CW = BN / 2;   // CW: columns of a sum thread
  constexpr uint32_t B_BYTES = S::B_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  Ctl* ctl = (Ctl*)(smem + STAGES * (A_BYTES + B_BYTES));
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 1);
    }
    for (int s = 0; s < ACC; ++s) {
      mbar_init(&ctl->acc_full[s], 1);
      mbar_init(&ctl->acc_empty[s], kSumWarps);
    }
    mbar_init(&ctl->drain, 1);
    ctl->abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&a.a);
    tma_prefetch_desc(&a.b);
  }
  if (warp == 9) {
    tmem_alloc(&ctl->tmem_base, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
  volatile int* abort_flag = &ctl->abort;
  const int mt_ = (a.M + BM - 1) / BM, nt = (a.N + BN - 1) / BN, tiles = mt_ * nt, kblocks = (a.K + BK - 1) / BK;

  if (warp == 8) {
    // ------------------------------------------------------------ TMA producer: a uniform warp, one lane issues
    uint32_t s = 0, ph = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      int mb, nb;
      tile_of(t, mt_, nt, &mb, &nb);
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!wait_bar_warp(&ctl->empty[s], ph ^ 1, abort_flag, a.timeout_ns)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          mbar_expect_tx(&ctl->full[s], A_BYTES + B_BYTES);
          if (TA) tma_load_2d(sA + s * A_BYTES, &a.a, mb * BM, kb * BK, &ctl->full[s]);
          else tma_load_2d(sA + s * A_BYTES, &a.a, kb * BK, mb * BM, &ctl->full[s]);
          if (TB) {
#pragma unroll
            for (int c = 0; c < BN / 128; ++c)
              tma_load_2d(sB + s * B_BYTES + c * CHUNK, &a.b, nb * BN + c * 128, kb * BK, &ctl->full[s]);
          } else {
            tma_load_2d(sB + s * B_BYTES, &a.b, kb * BK, nb * BN, &ctl->full[s]);
          }
        }
        __syncwarp();
        if (++s == STAGES) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    if (aborted_warp(abort_flag)) {
      // copies in flight may still be landing in shared memory: give them a bounded time
      const uint64_t t0 = globaltimer();
      while (globaltimer() - t0 < 100000ull) __nanosleep(1000);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer: uniform, one lane issues
    constexpr uint32_t idesc = make_idesc_e4m3(BM, BN) | (TA ? kIdescTransA : 0u) | (TB ? kIdescTransB : 0u);
    // a step of 32 along K: 32 bytes of a row, or 32 rows of 128 bytes
    constexpr uint64_t step_a = TA ? 256 : 2, step_b = TB ? 256 : 2;
    uint32_t s = 0, ph = 0, b = 0, bph = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!wait_bar_warp(&ctl->acc_empty[b], bph ^ 1, abort_flag, a.timeout_ns) ||
            !wait_bar_warp(&ctl->full[s], ph, abort_flag, a.timeout_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t da = TA ? make_smem_desc_mn_sw128(sA + s * A_BYTES, CHUNK) : make_smem_desc_sw128(sA + s * A_BYTES);
        const uint64_t db = TB ? make_smem_desc_mn_sw128(sB + s * B_BYTES, CHUNK) : make_smem_desc_sw128(sB + s * B_BYTES);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f8(tmem_base + b * BN, da + k * step_a, db + k * step_b, idesc, k > 0 ? 1u : 0u);
          umma_commit(&ctl->empty[s]);
          umma_commit(&ctl->acc_full[b]);
        }
        __syncwarp();
        if (++s == STAGES) {
          s = 0;
          ph ^= 1;
        }
        if (++b == ACC) {
          b = 0;
          bph ^= 1;
        }
      }
    }
    // no MMA may still be writing TMEM when it is freed
    if (elect_one()) umma_commit(&ctl->drain);
    __syncwarp();
    wait_bar_warp(&ctl->drain, 0, abort_flag, a.timeout_ns);
  } else {
    // ------------------------------------------------------------ sums and C
    const int q = warp & 3, half = warp >> 2;   // TMEM lane quarter, half of the columns
    uint32_t b = 0, bph = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      int mb, nb;
      tile_of(t, mt_, nt, &mb, &nb);
      const int row = mb * BM + q * 32 + lane, col = nb * BN + half * CW;
      const bool live = row < a.M, work = mb * BM + q * 32 < a.M && col < a.N;   // work: the same for the whole warp
      const float* pa = a.sa + (int64_t)row * a.sa_m;
      const float* pb = a.sb + (int64_t)(col >> 7) * a.sb_n;
      uint64_t acc[CW / 2];
#pragma unroll
      for (int i = 0; i < CW / 2; ++i) acc[i] = 0;
      float fa = live ? __ldg(pa) : 0.f, fb = work ? __ldg(pb) : 0.f;
      for (int kb = 0; kb < kblocks; ++kb) {
        const float f = fa * fb;
        if (kb + 1 < kblocks) {   // the next block's scales arrive while this one is waited for
          fa = live ? __ldg(pa + (int64_t)(kb + 1) * a.sa_k) : 0.f;
          fb = work ? __ldg(pb + (int64_t)(kb + 1) * a.sb_k) : 0.f;
        }
        if (!wait_bar_warp(&ctl->acc_full[b], bph, abort_flag, a.timeout_ns)) {
          ok = false;
          break;
        }
        if (work) {
          tc_fence_after();
          const uint64_t f2 = pack2(f, f);
          const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + b * BN + half * CW;
#pragma unroll
          for (int c = 0; c < CW / 32; ++c) {
            uint32_t r[32];
            tmem_ld_32x32(taddr + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i)
              fma2(acc[c * 16 + i], (uint64_t)r[2 * i] | ((uint64_t)r[2 * i + 1] << 32), f2);
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->acc_empty[b]);
        if (++b == ACC) {
          b = 0;
          bph ^= 1;
        }
      }
      if (ok && live && work) {
        const int esz = a.out_dtype == DT_F32 ? 4 : 2;
        uint8_t* p = (uint8_t*)a.c + ((int64_t)row * a.ldc + col) * esz;
#pragma unroll
        for (int c = 0; c < CW / 32; ++c) {
          const int n = a.N - col - c * 32;
          if (n > 0) {
            if (a.out_dtype == DT_F32) store32<F32>(p + c * 128, acc + c * 16, n, a.vec_out);
            else if (a.out_dtype == DT_BF16) store32<BF16>(p + c * 64, acc + c * 16, n, a.vec_out);
            else store32<F16>(p + c * 64, acc + c * 16, n, a.vec_out);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_error, 1);
}

template <int BN, bool TA, bool TB>
cudaError_t go(const Fp8GemmArgs& a, int nctas, cudaStream_t s) {
  const void* fn = (const void*)gemm_fp8_kernel<BN, TA, TB>;
  // per device, and cheap enough to say at every launch
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<BN>::SMEM);
  if (e != cudaSuccess) return e;
  gemm_fp8_kernel<BN, TA, TB><<<nctas, kThreads, Shape<BN>::SMEM, s>>>(a);
  return cudaGetLastError();
}
template <int BN>
cudaError_t go_form(bool ta, bool tb, const Fp8GemmArgs& a, int nctas, cudaStream_t s) {
  if (ta) return go<BN, true, true>(a, nctas, s);
  return tb ? go<BN, false, true>(a, nctas, s) : go<BN, false, false>(a, nctas, s);
}

}  // namespace fp8g

cudaError_t launch_fp8_gemm(int bn, bool ta, bool tb, const Fp8GemmArgs& a, int nctas, cudaStream_t s) {
  if (ta && !tb) return cudaErrorInvalidValue;
  count_launch();
  switch (bn) {
    case 256: return fp8g::go_form<256>(ta, tb, a, nctas, s);
    case 128: return fp8g::go_form<128>(ta, tb, a, nctas, s);
    default: return cudaErrorInvalidValue;
  }
}

int fp8_gemm_error() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, fp8g::g_error, sizeof(int)) != cudaSuccess) return -1;
  return v;
}

}  // namespace mt
