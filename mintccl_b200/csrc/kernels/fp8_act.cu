// silu(h) and silu(h) * u whose inputs are kept in 8 bits (row blocks, device/fp8_block.cuh) for the backward pass, and the
// gradients from what was kept.  One pass each way; bound by HBM.
//
//   forward   y = silu(h) [* u] from the inputs as they are; h [and u] encoded beside it
//   backward  with h, u restored from 8 bits and p = 1 / (1 + exp(-h)):
//             dh = dy [* u] * p * (1 + h * (1 - p)),  du = dy * h * p,  and on request the activation itself again
//
// Arithmetic is fp32 with one rounding at the end.  For 16-bit tensors the exponential is ex2 and the quotient the
// approximate reciprocal (relative error below 1e-5, a rounding to fp16 is 2.4e-4); for fp32 ones they are those of device/silu.cuh.
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

// (1 + exp(-x)) / 4, whose reciprocal does not underflow before the sum overflows (an exponential below 2^-126 may be zero
// beside the 1)
__device__ __forceinline__ float quarter_y(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
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

// 8192 x 4096 bf16, us: forward 29.7 (5.7 TB/s), gated 48 (5.6), backward 29.6 (5.7), gated 53 (5.1); a copy runs at 6.0.  What is
// in the way is some 18 instructions an element.  U: blocks a thread has in flight; with one the ungated forms took 36 and 34,
// with two the gated ones 53 and 62.
template <class T, int VEC, bool GATED, int U>
__global__ void __launch_bounds__(kThreads, 4) fp8_act_fwd_kernel(Fp8ActArgs a, RowGrid grid) {
  using E = typename T::elem;
  using W = WarpSpans<T, VEC>;
  constexpr int kE = (int)sizeof(E);
  constexpr bool kExact = kE == 4;
  __shared__ __align__(16) uint8_t stages[8][W::kStage];
  uint8_t* stage = stages[threadIdx.x >> 5];
  const Place<U> p(grid);
  const bool first = (threadIdx.x & 7) == 0;
  const uint8_t* hp = (const uint8_t*)a.h + (p.row * a.ldh + p.c0) * kE;
  const uint8_t* gp = GATED ? (const uint8_t*)a.u + (p.row * a.ldu + p.c0) * kE : nullptr;
  Span16<T, VEC> h[U], g[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    W::load(h[u], hp + 128 * u * kE, p.n(u), stage);
    if (GATED) W::load(g[u], gp + 128 * u * kE, p.n(u), stage);
  }
  const int64_t at = p.row * a.ldq + p.c0;
  uint8_t* yp = (uint8_t*)a.y + (p.row * a.ldy + p.c0) * kE;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int n = p.n(u);
    float f[16], y[16];
    uint32_t e;
    h[u].get(f);
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = silu_of<kExact>(f[i]);
    uint4 q = encode_row16(h[u], f, &e);
    if (n > 0) *(uint4*)(a.kh.data + at + 128 * u) = q;
    if (first && p.live(u)) a.kh.scale[p.row * a.kh.s_row + (p.kb + u) * a.kh.s_col] = fp8_scale(e);
    if (GATED) {
      g[u].get(f);
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] *= f[i];
      q = encode_row16(g[u], f, &e);
      if (n > 0) *(uint4*)(a.ku.data + at + 128 * u) = q;
      if (first && p.live(u)) a.ku.scale[p.row * a.ku.s_row + (p.kb + u) * a.ku.s_col] = fp8_scale(e);
    }
    h[u].set(y);
    W::store(h[u], yp + 128 * u * kE, n, stage);
  }
}

template <class T, int VEC, bool GATED, int U>
__global__ void __launch_bounds__(kThreads) fp8_act_bwd_kernel(Fp8ActArgs a, RowGrid grid) {
  using E = typename T::elem;
  using W = WarpSpans<T, VEC>;
  constexpr int kE = (int)sizeof(E);
  constexpr bool kExact = kE == 4;
  __shared__ __align__(16) uint8_t stages[8][W::kStage];
  uint8_t* stage = stages[threadIdx.x >> 5];
  const Place<U> p(grid);
  if (VEC > 0 && p.n(0) <= 0) return;   // by elements the warp works as one
  const int64_t at = p.row * a.ldq + p.c0;
  const uint8_t* dp = (const uint8_t*)a.dy + (p.row * a.lddy + p.c0) * kE;
  u128 hq[U], gq[U];
  float hs[U], gs[U];
  Span16<T, VEC> d[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    hq[u] = gq[u] = {0, 0};
    hs[u] = gs[u] = 0.f;
    if (p.n(u) > 0) {
      hq[u] = load128_stream(a.kh.data + at + 128 * u);
      hs[u] = __ldg(a.kh.scale + p.row * a.kh.s_row + (p.kb + u) * a.kh.s_col);
      if (GATED) {
        gq[u] = load128_stream(a.ku.data + at + 128 * u);
        gs[u] = __ldg(a.ku.scale + p.row * a.ku.s_row + (p.kb + u) * a.ku.s_col);
      }
    }
    W::load(d[u], dp + 128 * u * kE, p.n(u), stage);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int n = p.n(u);
    if (VEC > 0 && n <= 0) break;
    float h[16], g[16], f[16], act[16];
    restore16<F32>(hq[u], hs[u], h);
    if (GATED) restore16<F32>(gq[u], gs[u], g);
    d[u].get(f);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      // slope = s (1 + x (1 - s))
      const float x = h[i], s = sigmoid_of<kExact>(x), slope = __fmaf_rn(s, __fmaf_rn(-s, x, x), s), y = x * s;
      if (GATED) {
        act[i] = y * g[i];
        h[i] = f[i] * g[i] * slope;
        g[i] = f[i] * y;
      } else {
        act[i] = y;
        h[i] = f[i] * slope;
      }
    }
    d[u].set(h);
    W::store(d[u], (uint8_t*)a.dh + (p.row * a.lddh + p.c0 + 128 * u) * kE, n, stage);
    if (GATED) {
      d[u].set(g);
      W::store(d[u], (uint8_t*)a.du + (p.row * a.lddu + p.c0 + 128 * u) * kE, n, stage);
    }
    if (a.y) {
      d[u].set(act);
      W::store(d[u], (uint8_t*)a.y + (p.row * a.ldy + p.c0 + 128 * u) * kE, n, stage);
    }
  }
}

template <class T, int VEC, bool GATED>
cudaError_t act_go(const Fp8ActArgs& a, bool forward, cudaStream_t s) {
  // spans a thread: two pay where they fit the registers of enough threads
  constexpr int U = GATED || VEC == 0 ? 1 : 2;
  RowGrid g;
  dim3 grid;
  if (cudaError_t e = row_grid<U>(a.rows, a.cols, &g, &grid); e != cudaSuccess) return e;
  if (forward) fp8_act_fwd_kernel<T, VEC, GATED, U><<<grid, kThreads, 0, s>>>(a, g);
  else fp8_act_bwd_kernel<T, VEC, GATED, U><<<grid, kThreads, 0, s>>>(a, g);
  return cudaGetLastError();
}
template <class T, int VEC>
cudaError_t act_gated(const Fp8ActArgs& a, bool forward, cudaStream_t s) {
  const bool gated = forward ? a.u != nullptr : a.ku.data != nullptr;
  return gated ? act_go<T, VEC, true>(a, forward, s) : act_go<T, VEC, false>(a, forward, s);
}
template <class T>
cudaError_t act_vec(const Fp8ActArgs& a, bool forward, cudaStream_t s) {
  return a.vec == 2 ? act_gated<T, 2>(a, forward, s) : a.vec == 1 ? act_gated<T, 1>(a, forward, s) : act_gated<T, 0>(a, forward, s);
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
