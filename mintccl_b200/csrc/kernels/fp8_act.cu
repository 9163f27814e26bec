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

// Where this thread works, and how many of its 16 elements exist.
struct Place {
  RowSpan at;
  int64_t c0;
  int n;
  __device__ __forceinline__ Place(const Fp8ActArgs& a, uint32_t nkb) {
    at = row_span(blockIdx.x, threadIdx.x >> 3, a.rows, nkb);
    c0 = (int64_t)at.kb * 128 + (threadIdx.x & 7) * 16;
    n = at.live ? (int)min((int64_t)16, max((int64_t)0, a.cols - c0)) : 0;
  }
};

// 8192 x 4096 bf16: forward 35.5 us (4.7 TB/s), gated 49 (5.4), backward 34 (5.0), gated 54 (4.9); a copy runs at 6.0.  About 22
// instructions an element are what is in the way: two spans a thread (34.6 forward, 58 - 69 the others) and more or fewer
// CTAs than these an SM were slower.
template <class T, int VEC, bool GATED>
__global__ void __launch_bounds__(kThreads, 4) fp8_act_fwd_kernel(Fp8ActArgs a, uint32_t nkb) {
  using E = typename T::elem;
  using W = WarpSpans<T, VEC>;
  constexpr int kE = (int)sizeof(E);
  constexpr bool kExact = kE == 4;
  __shared__ __align__(16) uint8_t stages[8][W::kStage];
  uint8_t* stage = stages[threadIdx.x >> 5];
  const bool first = (threadIdx.x & 7) == 0;
  const Place p(a, nkb);
  const RowSpan& at = p.at;
  Span16<T, VEC> h, g;
  W::load(h, (const uint8_t*)a.h + (at.row * a.ldh + p.c0) * kE, p.n, stage);
  if (GATED) W::load(g, (const uint8_t*)a.u + (at.row * a.ldu + p.c0) * kE, p.n, stage);
  const bool put = at.live && p.c0 < a.ldq;
  float f[16], y[16];
  uint32_t e;
  h.get(f);
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = silu_of<kExact>(f[i]);
  uint4 q = encode_row16(h, f, &e);
  if (put) *(uint4*)(a.kh.data + at.row * a.ldq + p.c0) = q;
  if (at.live && first) a.kh.scale[at.row * a.kh.s_row + at.kb * a.kh.s_col] = fp8_scale(e);
  if (GATED) {
    g.get(f);
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] *= f[i];
    q = encode_row16(g, f, &e);
    if (put) *(uint4*)(a.ku.data + at.row * a.ldq + p.c0) = q;
    if (at.live && first) a.ku.scale[at.row * a.ku.s_row + at.kb * a.ku.s_col] = fp8_scale(e);
  }
  h.set(y);
  W::store(h, (uint8_t*)a.y + (at.row * a.ldy + p.c0) * kE, p.n, stage);
}

template <class T, int VEC, bool GATED>
__global__ void __launch_bounds__(kThreads) fp8_act_bwd_kernel(Fp8ActArgs a, uint32_t nkb) {
  using E = typename T::elem;
  using W = WarpSpans<T, VEC>;
  constexpr int kE = (int)sizeof(E);
  constexpr bool kExact = kE == 4;
  __shared__ __align__(16) uint8_t stages[8][W::kStage];
  uint8_t* stage = stages[threadIdx.x >> 5];
  const Place p(a, nkb);
  const RowSpan& at = p.at;
  if (VEC > 0 && p.n <= 0) return;   // by elements the warp works as one
  u128 hq = {0, 0}, gq = {0, 0};
  float hs = 0.f, gs = 0.f;
  if (VEC > 0 || p.n > 0) {
    hq = load128_stream(a.kh.data + at.row * a.ldq + p.c0);
    hs = __ldg(a.kh.scale + at.row * a.kh.s_row + at.kb * a.kh.s_col);
    if (GATED) {
      gq = load128_stream(a.ku.data + at.row * a.ldq + p.c0);
      gs = __ldg(a.ku.scale + at.row * a.ku.s_row + at.kb * a.ku.s_col);
    }
  }
  Span16<T, VEC> d;
  W::load(d, (const uint8_t*)a.dy + (at.row * a.lddy + p.c0) * kE, p.n, stage);
  float h[16], g[16], f[16], act[16];
  restore16<F32>(hq, hs, h);
  if (GATED) restore16<F32>(gq, gs, g);
  d.get(f);
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
  d.set(h);
  W::store(d, (uint8_t*)a.dh + (at.row * a.lddh + p.c0) * kE, p.n, stage);
  if (GATED) {
    d.set(g);
    W::store(d, (uint8_t*)a.du + (at.row * a.lddu + p.c0) * kE, p.n, stage);
  }
  if (a.y) {
    d.set(act);
    W::store(d, (uint8_t*)a.y + (at.row * a.ldy + p.c0) * kE, p.n, stage);
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
