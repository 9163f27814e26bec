// Encoding to and decoding from e4m3 with one fp32 scale per block of 128 (device/fp8_block.cuh): 1 x 128 along rows,
// 128 x 1 along columns, 128 x 128.  Bound by HBM.
//
// The reference has no fp8 path; it is on its roadmap (README.md:58-60).
#include <cuda_runtime.h>

#include "../device/fp8_block.cuh"
#include "fp8.h"
#include "launch.h"

namespace mt {
namespace {

constexpr int kThreads = 256;

// ---- row blocks: eight lanes a block, U blocks of every lane group in flight.  8192 x 4096 bf16 takes 16.1 us (6.3 TB/s).
template <class T, int VEC, int U>
__global__ void __launch_bounds__(kThreads) fp8_row_kernel(Fp8QuantArgs a, RowGrid grid) {
  constexpr int kE = (int)sizeof(typename T::elem);
  using W = WarpSpans<T, VEC>;
  __shared__ __align__(16) uint8_t stage[8][W::kStage];
  const Place<U> p(grid);
  const uint8_t* x = (const uint8_t*)a.x + (p.row * a.ldx + p.c0) * kE;
  Span16<T, VEC> in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) W::load(in[u], x + 128 * u * kE, p.n(u), stage[threadIdx.x >> 5]);
  uint32_t top[U];
  const bool special = row_tops<T, VEC, U>(in, top);
  uint8_t* data = a.row.data + p.row * a.ldq + p.c0;
  float* scale = a.row.scale + p.row * a.row.s_row + p.kb * a.row.s_col;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[16];
    in[u].get(f);
    only_finite16(f, special);
    const uint32_t e = fp8_scale_exp(top[u]);
    const uint4 q = e4m3_16(f, fp8_inverse(e));
    if (p.n(u) > 0) *(uint4*)(data + 128 * u) = q;   // a row's padding to 16 bytes is zeros
    if ((threadIdx.x & 7) == 0 && p.live(u)) scale[u * a.row.s_col] = fp8_scale(e);
  }
}

// ---- any of the three from one read: a CTA holds a tile of 128 x 128 in registers, a thread 4 rows (32 apart) of 16
// adjacent columns.  Largest magnitudes are taken on the bit patterns, two to a word; tiles with values that are not finite
// look at them again.  8192 x 4096 bf16, us: tiles 17.2 (5.9 TB/s), column blocks 18.7, row blocks and tiles from one read 29.6 (4.5),
// row and column blocks 31.6 (4.2), tiles and column blocks 28.1, all three 36.7; row blocks and then tiles take 34.5, or column
// blocks 36.1, with the input from the L2 the second time.  The 120 - 128 registers of forms with row blocks leave two CTAs
// an SM; with three they spill (50 - 60 us).  Tiles and column blocks are under the limit of three for 16-bit types and spill
// 84 - 96 bytes a thread there; off the vector grid, where shared memory takes part, every form with two encodings does.
template <class T, int VEC, bool ROW, bool COL, bool TILE>
__global__ void __launch_bounds__(kThreads, sizeof(typename T::elem) == 2 && !ROW ? 3 : 2) fp8_tile_kernel(Fp8QuantArgs a, uint32_t nct) {
  constexpr int kE = (int)sizeof(typename T::elem);
  using M = Mags<T>;
  using W = WarpSpans<T, VEC>;
  __shared__ __align__(16) uint8_t stage[8][W::kStage];
  __shared__ uint32_t s_max[8][8 * M::kWords];   // column magnitudes as words, per warp
  __shared__ __align__(16) float s_inv[128];
  __shared__ uint32_t s_tile[8];
  const int g = threadIdx.x >> 3, l = threadIdx.x & 7, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rt = blockIdx.x / nct, ct = blockIdx.x - rt * nct;
  const int64_t c0 = (int64_t)ct * 128 + l * 16;
  const int n = (int)min((int64_t)16, max((int64_t)0, a.cols - c0));
  // rows of this thread that exist, of four; where the first is in a payload, and the distance to the next
  const int64_t r0 = (int64_t)rt * 128 + g, q0 = r0 * a.ldq + c0, qstep = 32 * a.ldq;
  const int live = (int)min((int64_t)4, max((int64_t)0, (a.rows - r0 + 31) >> 5));
  const bool put = n > 0;   // a row's padding to 16 bytes is zeros; what lies between that and the next row is not ours
  Span16<T, VEC> in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    W::load(in[i], (const uint8_t*)a.x + ((r0 + i * 32) * a.ldx + c0) * kE, i < live ? n : 0, stage[warp]);
  if (ROW) {
    uint32_t top[4];
    const bool special = row_tops<T, VEC, 4>(in, top);
    uint8_t* to = a.row.data + q0;
    float* scale = a.row.scale + r0 * a.row.s_row + ct * a.row.s_col;
#pragma unroll
    for (int i = 0; i < 4; ++i, to += qstep, scale += 32 * a.row.s_row) {
      float f[16];
      in[i].again();
      in[i].get(f);
      only_finite16(f, special);
      const uint32_t e = fp8_scale_exp(top[i]);
      const uint4 q = e4m3_16(f, fp8_inverse(e));
      if (i < live) {
        if (put) *(uint4*)to = q;
        if (l == 0) *scale = fp8_scale(e);
      }
    }
  }
  if (!COL && !TILE) return;
  M m;
  auto reduce = [&] {   // this warp's columns and tile to shared memory
    if (TILE) {
      const uint32_t t = __reduce_max_sync(0xffffffffu, m.top());
      if (lane == 0) s_tile[warp] = t;
    }
    if (COL) {
#pragma unroll
      for (int d = 8; d < 32; d <<= 1)
#pragma unroll
        for (int j = 0; j < M::kWords; ++j) m.m[j] = M::larger(m.m[j], __shfl_xor_sync(0xffffffffu, m.m[j], d));
      if (lane < 8)
#pragma unroll
        for (int j = 0; j < M::kWords; ++j) s_max[warp][l * M::kWords + j] = m.m[j];
    }
  };
  m.clear();
#pragma unroll
  for (int i = 0; i < 4; ++i) m.template fold<false>(in[i].v);
  const bool special = __syncthreads_or(m.top() >= kInfBits);
  if (special) {
    asm volatile("");
    m.clear();
#pragma unroll
    for (int i = 0; i < 4; ++i) m.template fold<true>(in[i].v);
  }
  reduce();
  __syncthreads();
  if (TILE) {
    uint32_t t = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) t = max(t, s_tile[w]);
    const uint32_t e = fp8_scale_exp(t);
    const float inv = fp8_inverse(e);
    uint8_t* to = a.tile.data + q0;
#pragma unroll
    for (int i = 0; i < 4; ++i, to += qstep) {
      float f[16];
      in[i].again();
      in[i].get(f);
      only_finite16(f, special);
      const uint4 q = e4m3_16(f, inv);
      if (i < live && put) *(uint4*)to = q;
    }
    if (threadIdx.x == 0) a.tile.scale[rt * a.tile.s_row + ct * a.tile.s_col] = fp8_scale(e);
  }
  if (COL) {
    if (threadIdx.x < 128) {
      // column c is half of a word for 16-bit types
      const int c = threadIdx.x, w0 = (c >> 4) * M::kWords + (M::kHalf ? (c & 15) >> 1 : c & 15);
      uint32_t t = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) t = M::larger(t, s_max[w][w0]);
      if (M::kHalf) t = (c & 1) ? t >> 16 : t & 0xffffu;
      const uint32_t e = fp8_scale_exp(M::bits(t));
      s_inv[c] = fp8_inverse(e);
      const int64_t cc = (int64_t)ct * 128 + c;
      if (cc < a.cols) a.col.scale[rt * a.col.s_row + cc * a.col.s_col] = fp8_scale(e);
    }
    __syncthreads();
    float inv[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) *(float4*)(inv + 4 * j) = *(const float4*)(s_inv + l * 16 + 4 * j);
    uint8_t* to = a.col.data + q0;
#pragma unroll
    for (int i = 0; i < 4; ++i, to += qstep) {
      float f[16];
      in[i].again();
      in[i].get(f);
      only_finite16(f, special);
#pragma unroll
      for (int j = 0; j < 16; j += 2) (F2(f[j], f[j + 1]) * F2(inv[j], inv[j + 1])).get(f[j], f[j + 1]);
      const uint4 q = e4m3_16(f);
      if (i < live && put) *(uint4*)to = q;
    }
  }
}

template <class T, int VEC>
cudaError_t quant_go(const Fp8QuantArgs& a, cudaStream_t s) {
  const int64_t nkb = (a.cols + 127) / 128;
  const bool row = a.row.data, col = a.col.data, tile = a.tile.data;
  if (col || tile) {
    const int64_t grid = (a.rows + 127) / 128 * nkb;
    if (grid >= 0x7fffffffll) return cudaErrorInvalidValue;
    auto go = [&](auto kernel) { kernel<<<(unsigned)grid, kThreads, 0, s>>>(a, (uint32_t)nkb); };
    if (row) {
      if (col && tile) go(fp8_tile_kernel<T, VEC, true, true, true>);
      else if (col) go(fp8_tile_kernel<T, VEC, true, true, false>);
      else go(fp8_tile_kernel<T, VEC, true, false, true>);
    } else {
      if (col && tile) go(fp8_tile_kernel<T, VEC, false, true, true>);
      else if (col) go(fp8_tile_kernel<T, VEC, false, true, false>);
      else go(fp8_tile_kernel<T, VEC, false, false, true>);
    }
    return cudaGetLastError();
  }
  RowGrid g;
  dim3 grid;
  if (cudaError_t e = row_grid<2>(a.rows, a.cols, &g, &grid); e != cudaSuccess) return e;
  fp8_row_kernel<T, VEC, 2><<<grid, kThreads, 0, s>>>(a, g);
  return cudaGetLastError();
}
template <class T>
cudaError_t quant_vec(const Fp8QuantArgs& a, cudaStream_t s) {
  return a.vec == 2 ? quant_go<T, 2>(a, s) : a.vec == 1 ? quant_go<T, 1>(a, s) : quant_go<T, 0>(a, s);
}

// ---- decoding: 8192 x 4096 bf16 takes 16.5 us (6.1 TB/s)
template <class T, int VEC, int U>
__global__ void __launch_bounds__(kThreads) fp8_dequant_kernel(Fp8DequantArgs a, RowGrid grid) {
  constexpr int kE = (int)sizeof(typename T::elem);
  using W = WarpSpans<T, VEC>;
  __shared__ __align__(16) uint8_t stage[8][W::kStage];
  const Place<U> p(grid);
  if (VEC > 0 && p.n(0) <= 0) return;   // by elements the warp works as one
  const uint8_t* data = a.data + p.row * a.ldq + p.c0;
  const float* sp = a.scale + (p.row >> a.rshift) * a.s_row;
  uint8_t* out = (uint8_t*)a.out + (p.row * a.ldo + p.c0) * kE;
  u128 w[U];
  float sc[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    w[u] = {0, 0};
    sc[u] = 1.f;
    if (p.n(u) > 0) {
      w[u] = load128_stream(data + 128 * u);
      if (a.cshift) sc[u] = __ldg(sp + (p.kb + u) * a.s_col);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int n = p.n(u);
    if (VEC > 0 && n <= 0) break;
    float f[16];
    if (a.cshift) {
      restore16<T>(w[u], sc[u], f);
    } else {
      float c[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) c[i] = i < n ? __ldg(sp + (p.c0 + 128 * u + i) * a.s_col) : 0.f;
      restore16<F32>(w[u], 1.f, f);
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = clamp_nan(f[i] * c[i], MaxOf<T>::value);
    }
    Span16<T, VEC> o;
    o.set(f);
    W::store(o, out + 128 * u * kE, n, stage[threadIdx.x >> 5]);
  }
}

template <class T, int VEC>
cudaError_t dequant_go(const Fp8DequantArgs& a, cudaStream_t s) {
  RowGrid g;
  dim3 grid;
  if (cudaError_t e = row_grid<2>(a.rows, a.cols, &g, &grid); e != cudaSuccess) return e;
  fp8_dequant_kernel<T, VEC, 2><<<grid, kThreads, 0, s>>>(a, g);
  return cudaGetLastError();
}
template <class T>
cudaError_t dequant_vec(const Fp8DequantArgs& a, cudaStream_t s) {
  return a.vec == 2 ? dequant_go<T, 2>(a, s) : a.vec == 1 ? dequant_go<T, 1>(a, s) : dequant_go<T, 0>(a, s);
}

}  // namespace

cudaError_t launch_fp8_quant(int dtype, const Fp8QuantArgs& a, cudaStream_t s) {
  count_launch();
  switch (dtype) {
    case DT_F32: return quant_vec<F32>(a, s);
    case DT_F16: return quant_vec<F16>(a, s);
    case DT_BF16: return quant_vec<BF16>(a, s);
    default: return cudaErrorInvalidValue;
  }
}
cudaError_t launch_fp8_dequant(int dtype, const Fp8DequantArgs& a, cudaStream_t s) {
  count_launch();
  switch (dtype) {
    case DT_F32: return dequant_vec<F32>(a, s);
    case DT_F16: return dequant_vec<F16>(a, s);
    case DT_BF16: return dequant_vec<BF16>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace mt
