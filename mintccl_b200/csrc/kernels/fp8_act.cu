// silu(h) and silu(h) * u whose inputs are kept in 8 bits (row blocks, device/fp8_block.cuh) for the backward pass, and the
// gradients from what was kept.  One pass each way; bound by HBM.
//
//   forward   y = silu(h) [* u] from the inputs as they are; h [and u] encoded beside it
//   backward  with h, u restored from 8 bits and p = 1 / (1 + exp(-h)):
//             dh = dy [* u] * p * (1 + h * (1 - p)),  du = dy * h * p,  and on request the activation itself again
//
// Arithmetic is fp32 with one rounding at the end.  For 16-bit tensors the exponential is ex2 and the quotient one Newton
// step short (relative error below 1e-5, a rounding to fp16 is 2.4e-4); for fp32 ones they are those of device/silu.cuh.
//
// The reference has no element-wise operators (README.md:5).
#include <cuda_runtime.h>

#include "../device/fp8_block.cuh"
#include "../device/silu.cuh"
#include "fp8.h"
#include "launch.h"

namespace mt {
namespace {

constexpr int kThreads = 256;

// (1 + exp(-x)) / 4, whose reciprocal does not underflow before the sum overflows
__device__ __forceinline__ float quarter_y(float x) {
  float e;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  return __fmaf_rn(e, 0.25f, 0.25f);
}
__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 1 / (1 + exp(-x))
template <bool EXACT>
__device__ __forceinline__ float sigmoid_of(float x) {
  if constexpr (EXACT) {
    const float y = 1.f + expf(-x);
    return y <= 3.4028234e38f ? 0.25f * four_over(0.25f * y) : (y != y ? y : 0.f);
  } else {
    return 0.25f * rcp_fast(quarter_y(x));
  }
}
template <bool EXACT>
__device__ __forceinline__ float silu_of(float x) {
  if constexpr (EXACT) return silu1(x);
  else return (0.25f * x) * rcp_fast(quarter_y(x));
}

template <class T, int VEC, bool GATED>
__global__ void __launch_bounds__(kThreads) fp8_act_fwd_kernel(Fp8ActArgs a, uint32_t nkb) {
  using E = typename T::elem;
  using W = WarpSpans<T, VEC>;
  constexpr int kE = (int)sizeof(E);
  constexpr bool kExact = kE == 4;
  __shared__ __align__(16) uint8_t stages[8][W::kStage];
  uint8_t* stage = stages[threadIdx.x >> 5];
  const int g = threadIdx.x >> 3, l = threadIdx.x & 7;
  const RowSpan at = row_span(blockIdx.x, g, a.rows, nkb);
  const int64_t c0 = (int64_t)at.kb * 128 + l * 16;
  const int n = at.live ? (int)min((int64_t)16, max((int64_t)0, a.cols - c0)) : 0;
  Span16<T, VEC> h, u;
  W::load(h, (const uint8_t*)a.h + (at.row * a.ldh + c0) * kE, n, stage);
  if (GATED) W::load(u, (const uint8_t*)a.u + (at.row * a.ldu + c0) * kE, n, stage);
  const bool put = at.live && c0 < a.ldq;
  float f[16], y[16];
  uint32_t e;
  h.get(f);
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = silu_of<kExact>(f[i]);
  uint4 q = encode_row16(h, f, &e);
  if (put) *(uint4*)(a.kh.data + at.row * a.ldq + c0) = q;
  if (at.live && l == 0) a.kh.scale[at.row * a.kh.s_row + at.kb * a.kh.s_col] = fp8_scale(e);
  if (GATED) {
    u.get(f);
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] *= f[i];
    q = encode_row16(u, f, &e);
    if (put) *(uint4*)(a.ku.data + at.row * a.ldq + c0) = q;
    if (at.live && l == 0) a.ku.scale[at.row * a.ku.s_row + at.kb * a.ku.s_col] = fp8_scale(e);
  }
  h.set(y);
  W::store(h, (uint8_t*)a.y + (at.row * a.ldy + c0) * kE, n, stage);
}

template <class T, int VEC, bool GATED>
__global__ void __launch_bounds__(kThreads) fp8_act_bwd_kernel(Fp8ActArgs a, uint32_t nkb) {
  using E = typename T::elem;
  using W = WarpSpans<T, VEC>;
  constexpr int kE = (int)sizeof(E);
  constexpr bool kExact = kE == 4;
  __shared__ __align__(16) uint8_t stages[8][W::kStage];
  uint8_t* stage = stages[threadIdx.x >> 5];
  const int g = threadIdx.x >> 3, l = threadIdx.x & 7;
  const RowSpan at = row_span(blockIdx.x, g, a.rows, nkb);
  const int64_t c0 = (int64_t)at.kb * 128 + l * 16;
  const int n = at.live ? (int)min((int64_t)16, max((int64_t)0, a.cols - c0)) : 0;
  if (VEC > 0 && n <= 0) return;   // by elements the warp works as one
  u128 hq = {0, 0}, uq = {0, 0};
  float hs = 0.f, us = 0.f;
  if (VEC > 0 || n > 0) {
    hq = load128_stream(a.kh.data + at.row * a.ldq + c0);
    hs = __ldg(a.kh.scale + at.row * a.kh.s_row + at.kb * a.kh.s_col);
    if (GATED) {
      uq = load128_stream(a.ku.data + at.row * a.ldq + c0);
      us = __ldg(a.ku.scale + at.row * a.ku.s_row + at.kb * a.ku.s_col);
    }
  }
  Span16<T, VEC> d;
  W::load(d, (const uint8_t*)a.dy + (at.row * a.lddy + c0) * kE, n, stage);
  float h[16], u[16], f[16], act[16];
  e4m3_16_to_float(make_uint4((uint32_t)hq.x, (uint32_t)(hq.x >> 32), (uint32_t)hq.y, (uint32_t)(hq.y >> 32)), h);
  if (GATED) e4m3_16_to_float(make_uint4((uint32_t)uq.x, (uint32_t)(uq.x >> 32), (uint32_t)uq.y, (uint32_t)(uq.y >> 32)), u);
  d.get(f);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float x = clamp_nan(h[i] * hs, 3.4028234663852886e38f);
    const float p = sigmoid_of<kExact>(x);
    const float slope = p * (1.f + x * (1.f - p)), s = x * p;
    if (GATED) {
      const float v = clamp_nan(u[i] * us, 3.4028234663852886e38f);
      act[i] = s * v;
      h[i] = f[i] * v * slope;
      u[i] = f[i] * s;
    } else {
      act[i] = s;
      h[i] = f[i] * slope;
    }
  }
  d.set(h);
  W::store(d, (uint8_t*)a.dh + (at.row * a.lddh + c0) * kE, n, stage);
  if (GATED) {
    d.set(u);
    W::store(d, (uint8_t*)a.du + (at.row * a.lddu + c0) * kE, n, stage);
  }
  if (a.y) {
    d.set(act);
    W::store(d, (uint8_t*)a.y + (at.row * a.ldy + c0) * kE, n, stage);
  }
}

template <class T, int VEC>
cudaError_t act_go(const Fp8ActArgs& a, bool forward, cudaStream_t s) {
  const int64_t nkb = (a.cols + 127) / 128, items = row_items(a.rows, nkb);
  const bool gated = forward ? a.u != nullptr : a.ku.data != nullptr;
  if (items >= 0x7fffffffll) return cudaErrorInvalidValue;
  auto go = [&](auto kernel) { kernel<<<(unsigned)items, kThreads, 0, s>>>(a, (uint32_t)nkb); };
  if (forward) {
    if (gated) go(fp8_act_fwd_kernel<T, VEC, true>);
    else go(fp8_act_fwd_kernel<T, VEC, false>);
  } else {
    if (gated) go(fp8_act_bwd_kernel<T, VEC, true>);
    else go(fp8_act_bwd_kernel<T, VEC, false>);
  }
  return cudaGetLastError();
}
template <class T>
cudaError_t act_vec(const Fp8ActArgs& a, bool forward, cudaStream_t s) {
  return a.vec == 2 ? act_go<T, 2>(a, forward, s) : a.vec == 1 ? act_go<T, 1>(a, forward, s) : act_go<T, 0>(a, forward, s);
}
cudaError_t act_any(int dtype, const Fp8ActArgs& a, bool forward, cudaStream_t s) {
  count_launch();
  switch (dtype) {
    case DT_F32: return act_vec<F32>(a, forward, s);
    case DT_F16: return act_vec<F16>(a, forward, s);
    case DT_BF16: return act_vec<BF16>(a, forward, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t launch_fp8_act_forward(int dtype, const Fp8ActArgs& a, cudaStream_t s) { return act_any(dtype, a, true, s); }
cudaError_t launch_fp8_act_backward(int dtype, const Fp8ActArgs& a, cudaStream_t s) { return act_any(dtype, a, false, s); }

}  // namespace mt
