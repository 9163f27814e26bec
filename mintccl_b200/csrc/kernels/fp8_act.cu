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

__device__ __forceinline__ float ex2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 4 / (1 + exp(-x)) of two values: the reciprocal of (1 + exp(-x)) / 4 does not underflow before the sum overflows (an
// exponential below 2^-126 may be zero beside the 1)
__device__ __forceinline__ F2 sigmoid4_fast(F2 x) {
  float a, b;
  (x * F2(-1.4426950408889634f)).get(a, b);
  fma2(F2(ex2_fast(a), ex2_fast(b)), F2(0.25f), F2(0.25f)).get(a, b);
  return F2(rcp_fast(a), rcp_fast(b));
}
// y = silu(x), 16 values
template <bool EXACT>
__device__ __forceinline__ void silu16(const float* x, float* y) {
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    if constexpr (EXACT) {
      y[i] = silu1(x[i]);
      y[i + 1] = silu1(x[i + 1]);
    } else {
      const F2 v(x[i], x[i + 1]);
      (F2(0.25f) * v * sigmoid4_fast(v)).get(y[i], y[i + 1]);
    }
  }
}
// s = 1 / (1 + exp(-x)) of two values
template <bool EXACT>
__device__ __forceinline__ F2 sigmoid2(float x0, float x1) {
  if constexpr (EXACT) {
    auto one = [](float x) {
      const float y = 1.f + expf(-x);
      return y <= 3.4028234e38f ? 0.25f * four_over(0.25f * y) : (y != y ? y : 0.f);
    };
    return F2(one(x0), one(x1));
  } else {
    return F2(0.25f) * sigmoid4_fast(F2(x0, x1));
  }
}

// 8192 x 4096 bf16, us: forward 28.8 (5.8 TB/s), gated 45.6 (5.9), backward 28.7 (5.8), gated 49.5 (5.4); a copy runs at 6.0.
// Multiplications go two to an instruction (29.7, 48, 29.6 and 53 one by one): the rest is some 12 an element.  U: blocks a
// thread has in flight; with one the ungated forms took 36 and 34, with two the gated ones 53 and 62.
// Four CTAs an SM for 16-bit types; fp32 ones have twice the words in flight and spill under that limit (8192 x 1792, gated
// forward 38, without it 33.5).  Gated and off the vector grid 16-bit ones spill 20 - 44 bytes a thread too (3000 x 4095 39.7).
template <class T, int VEC, bool GATED, int U>
__global__ void __launch_bounds__(kThreads, sizeof(typename T::elem) == 2 ? 4 : 0) fp8_act_fwd_kernel(Fp8ActArgs a, RowGrid grid) {
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
    silu16<kExact>(f, y);
    uint4 q = encode_row16(h[u], f, &e);
    if (n > 0) *(uint4*)(a.kh.data + at + 128 * u) = q;
    if (first && p.live(u)) a.kh.scale[p.row * a.kh.s_row + (p.kb + u) * a.kh.s_col] = fp8_scale(e);
    if (GATED) {
      g[u].get(f);
#pragma unroll
      for (int i = 0; i < 16; i += 2) (F2(y[i], y[i + 1]) * F2(f[i], f[i + 1])).get(y[i], y[i + 1]);
      q = encode_row16(g[u], f, &e);
      if (n > 0) *(uint4*)(a.ku.data + at + 128 * u) = q;
      if (first && p.live(u)) a.ku.scale[p.row * a.ku.s_row + (p.kb + u) * a.ku.s_col] = fp8_scale(e);
    }
    h[u].set(y);
    W::store(h[u], yp + 128 * u * kE, n, stage);
  }
}

// ACT: the activation is wanted too (its values cost 16 registers, a quarter of a thread's)
template <class T, int VEC, bool GATED, int U, bool ACT>
__global__ void __launch_bounds__(kThreads, sizeof(typename T::elem) == 2 && VEC ? 4 : 0) fp8_act_bwd_kernel(Fp8ActArgs a, RowGrid grid) {
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
    float h[16], g[16], f[16], act[ACT ? 16 : 1];
    restore16<F32>(hq[u], hs[u], h);
    if (GATED) restore16<F32>(gq[u], gs[u], g);
    d[u].get(f);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      // slope = s (1 + x (1 - s))
      const F2 x(h[i], h[i + 1]), s = sigmoid2<kExact>(h[i], h[i + 1]), d2(f[i], f[i + 1]), y = x * s;
      // x (1 - s): as x - y it is off by half a place of x, beside the 1 added to it no more than the sigmoid itself
      const F2 rest = kExact ? fma2(s * F2(-1.f), x, x) : fma2(y, F2(-1.f), x), slope = fma2(s, rest, s);
      if constexpr (GATED) {
        const F2 g2(g[i], g[i + 1]);
        if constexpr (ACT) (y * g2).get(act[i], act[i + 1]);
        (d2 * g2 * slope).get(h[i], h[i + 1]);
        (d2 * y).get(g[i], g[i + 1]);
      } else {
        if constexpr (ACT) y.get(act[i], act[i + 1]);
        (d2 * slope).get(h[i], h[i + 1]);
      }
    }
    d[u].set(h);
    W::store(d[u], (uint8_t*)a.dh + (p.row * a.lddh + p.c0 + 128 * u) * kE, n, stage);
    if (GATED) {
      d[u].set(g);
      W::store(d[u], (uint8_t*)a.du + (p.row * a.lddu + p.c0 + 128 * u) * kE, n, stage);
    }
    if constexpr (ACT) {
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
  else if (a.y) fp8_act_bwd_kernel<T, VEC, GATED, U, true><<<grid, kThreads, 0, s>>>(a, g);
  else fp8_act_bwd_kernel<T, VEC, GATED, U, false><<<grid, kThreads, 0, s>>>(a, g);
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
