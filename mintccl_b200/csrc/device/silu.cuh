// silu and its derivative, for the epilogue of the CTA-pair GEMM and the element-wise kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mt {

// silu and its derivative in fp32: the bits that x / (1 + exp(-x)) and sig * (1 + x * (1 - sig)) have as separate fp32
// operations.  The quotients are Newton's iteration with Markstein's last correction (Computation of elementary functions on
// the IBM RISC System/6000 processor, 1990) on y / 4, which keeps 4 / y a normal number up to the largest y: no branches, so
// that the 32 elements of a step overlap.  CUDA's own quotient has a slow path for large y, which a lane in six takes where
// h is spread over +- 64: silu in the epilogue of 8192 x 1792 x 4096 then took 205 us, 88.8 this way
// (plain 83.0).  The fast exponential and quotient (87.3) are off by up to 1e-5 far from zero and flush silu to zero below
// -87.3, where bf16 still has values.
__device__ __forceinline__ float four_over(float y4) {   // 1 / y4 = 4 / y, y4 in [1 / 4, 2^126)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y4));
  return __fmaf_rn(r, __fmaf_rn(-y4, r, 1.f), r);
}
__device__ __forceinline__ float silu1(float x) {
  const float y = 1.f + expf(-x), y4 = 0.25f * y, x4 = 0.25f * x, r = four_over(y4), q0 = __fmul_rn(x4, r);
  const float q = fabsf(q0) <= 3.4028234e38f ? __fmaf_rn(__fmaf_rn(-y4, q0, x4), r, q0) : q0;   // x infinite or NaN: as it is
  return y <= 3.4028234e38f ? q : (y != y ? y : x * 0.f);                                       // y infinite: a zero
}
__device__ __forceinline__ float dsilu1(float d, float x) {
  const float y = 1.f + expf(-x);
  const float s = y <= 3.4028234e38f ? 0.25f * four_over(0.25f * y) : (y != y ? y : 0.f);
  return __fmul_rn(d, __fmul_rn(s, __fadd_rn(1.f, __fmul_rn(x, 1.f - s))));
}

}  // namespace mt
