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

// ---- row blocks: eight lanes a block, U blocks of every lane group in flight
template <class T, int VEC, int U>
__global__ void __launch_bounds__(kThreads) fp8_row_kernel(Fp8QuantArgs a, int64_t nkb, int64_t items, bool by_rows) {
  constexpr int kE = (int)sizeof(typename T::elem);
  const int g = threadIdx.x >> 3, l = threadIdx.x & 7;
  Span16<T, VEC> in[U];
  RowSpan at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t item = (int64_t)blockIdx.x * U + u;
    at[u] = row_span(item, g, a.rows, nkb, by_rows);
    at[u].live = at[u].live && item < items;
    const int64_t c0 = at[u].kb * 128 + l * 16;
    const int n = at[u].live ? (int)min((int64_t)16, max((int64_t)0, a.cols - c0)) : 0;
    in[u].load((const uint8_t*)a.x + (at[u].row * a.ldx + c0) * kE, n);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[16];
    in[u].get(f);
    uint32_t e;
    const uint4 q = encode_row16(f, &e);
    if (!at[u].live) continue;
    const int64_t c0 = at[u].kb * 128 + l * 16;
    if (c0 < a.ldq) *(uint4*)(a.row.data + at[u].row * a.ldq + c0) = q;   // the padding of a row is zeros
    if (l == 0) a.row.scale[at[u].row * a.row.s_row + at[u].kb * a.row.s_col] = fp8_scale(e);
  }
}

// ---- any of the three from one read: a CTA holds a tile of 128 x 128 in registers, a thread 4 rows (32 apart) of 16
// adjacent columns
template <class T, int VEC>
__global__ void __launch_bounds__(kThreads) fp8_tile_kernel(Fp8QuantArgs a, int64_t nct) {
  constexpr int kE = (int)sizeof(typename T::elem);
  __shared__ uint32_t s_max[8][128];
  __shared__ uint32_t s_tile[8];
  const int g = threadIdx.x >> 3, l = threadIdx.x & 7, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t rt = blockIdx.x / nct, ct = blockIdx.x - rt * nct;
  const int64_t c0 = ct * 128 + l * 16;
  const int n = (int)min((int64_t)16, max((int64_t)0, a.cols - c0));
  Span16<T, VEC> in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = rt * 128 + i * 32 + g;
    in[i].load((const uint8_t*)a.x + (r * a.ldx + c0) * kE, r < a.rows ? n : 0);
  }
  if (a.row.data) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = rt * 128 + i * 32 + g;
      float f[16];
      in[i].get(f);
      uint32_t e;
      const uint4 q = encode_row16(f, &e);
      if (r < a.rows) {
        if (c0 < a.ldq) *(uint4*)(a.row.data + r * a.ldq + c0) = q;
        if (l == 0) a.row.scale[r * a.row.s_row + ct * a.row.s_col] = fp8_scale(e);
      }
    }
  }
  if (!a.col.data && !a.tile.data) return;
  // largest finite magnitudes of the columns, then of the tile
  uint32_t m[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) m[j] = 0;
  bool special = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[16];
    in[i].get(f);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      special |= abs_bits(f[j]) >= kInfBits;
      m[j] = max(m[j], finite_bits(f[j]));
    }
  }
  if (a.tile.data) {
    uint32_t t = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) t = max(t, m[j]);
    t = __reduce_max_sync(0xffffffffu, t);
    if (lane == 0) s_tile[warp] = t;
  }
  if (a.col.data) {
#pragma unroll
    for (int d = 8; d < 32; d <<= 1)
#pragma unroll
      for (int j = 0; j < 16; ++j) m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], d));
    if (lane < 8)
#pragma unroll
      for (int j = 0; j < 16; ++j) s_max[warp][l * 16 + j] = m[j];
  }
  __syncthreads();
  if (a.tile.data) {
    uint32_t t = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) t = max(t, s_tile[w]);
    const uint32_t e = fp8_scale_exp(t);
    const float inv = fp8_inverse(e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = rt * 128 + i * 32 + g;
      float f[16];
      in[i].get(f);
      if (r < a.rows && c0 < a.ldq) *(uint4*)(a.tile.data + r * a.ldq + c0) = e4m3_16(f, inv, special);
    }
    if (threadIdx.x == 0) a.tile.scale[rt * a.tile.s_row + ct * a.tile.s_col] = fp8_scale(e);
  }
  if (a.col.data) {
    if (threadIdx.x < 128) {
      uint32_t t = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) t = max(t, s_max[w][threadIdx.x]);
      const uint32_t e = fp8_scale_exp(t);
      s_max[0][threadIdx.x] = __float_as_uint(fp8_inverse(e));   // read by this thread alone before
      const int64_t c = ct * 128 + threadIdx.x;
      if (c < a.cols) a.col.scale[rt * a.col.s_row + c * a.col.s_col] = fp8_scale(e);
    }
    __syncthreads();
    float inv[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) inv[j] = __uint_as_float(s_max[0][l * 16 + j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = rt * 128 + i * 32 + g;
      float f[16];
      in[i].get(f);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const bool bad = abs_bits(f[j]) >= kInfBits;
        f[j] = bad ? __uint_as_float(0x7fc00000u) : f[j] * inv[j];
      }
      if (r < a.rows && c0 < a.ldq) *(uint4*)(a.col.data + r * a.ldq + c0) = e4m3_16(f, 1.f, false);
    }
  }
}

template <class T, int VEC>
cudaError_t quant_go(const Fp8QuantArgs& a, cudaStream_t s) {
  const int64_t nkb = (a.cols + 127) / 128;
  if (a.col.data || a.tile.data) {
    const int64_t grid = (a.rows + 127) / 128 * nkb;
    if (grid >= 0x7fffffffll) return cudaErrorInvalidValue;
    fp8_tile_kernel<T, VEC><<<(unsigned)grid, kThreads, 0, s>>>(a, nkb);
    return cudaGetLastError();
  }
  const bool by_rows = a.rows >= 32;
  const int64_t items = row_items(a.rows, nkb, by_rows), grid = (items + 1) / 2;
  if (grid >= 0x7fffffffll) return cudaErrorInvalidValue;
  fp8_row_kernel<T, VEC, 2><<<(unsigned)grid, kThreads, 0, s>>>(a, nkb, items, by_rows);
  return cudaGetLastError();
}
template <class T>
cudaError_t quant_vec(const Fp8QuantArgs& a, cudaStream_t s) {
  return a.vec == 2 ? quant_go<T, 2>(a, s) : a.vec == 1 ? quant_go<T, 1>(a, s) : quant_go<T, 0>(a, s);
}

// ---- decoding: 16 elements a thread
template <class T, int VEC>
__global__ void __launch_bounds__(kThreads) fp8_dequant_kernel(Fp8DequantArgs a, int64_t nkb, int64_t items, bool by_rows) {
  constexpr int kE = (int)sizeof(typename T::elem);
  const int g = threadIdx.x >> 3, l = threadIdx.x & 7;
  const RowSpan at = row_span(blockIdx.x, g, a.rows, nkb, by_rows);
  const int64_t c0 = at.kb * 128 + l * 16;
  if (!at.live || c0 >= a.cols) return;
  const u128 w = load128_stream(a.data + at.row * a.ldq + c0);
  const float* sp = a.scale + (at.row >> a.rshift) * a.s_row;
  const int n = (int)min((int64_t)16, a.cols - c0);
  float f[16];
  const uint4 q = make_uint4((uint32_t)w.x, (uint32_t)(w.x >> 32), (uint32_t)w.y, (uint32_t)(w.y >> 32));
  if (a.cshift) {
    const float sc = __ldg(sp + at.kb * a.s_col);
    e4m3_16_to_float(q, f);
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = clamp_nan(f[i] * sc, MaxOf<T>::value);
  } else {
    float sc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = i < n ? __ldg(sp + (c0 + i) * a.s_col) : 0.f;
    e4m3_16_to_float(q, f);
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = clamp_nan(f[i] * sc[i], MaxOf<T>::value);
  }
  Span16<T, VEC> o;
  o.set(f);
  o.store((uint8_t*)a.out + (at.row * a.ldo + c0) * kE, n);
}

template <class T, int VEC>
cudaError_t dequant_go(const Fp8DequantArgs& a, cudaStream_t s) {
  const int64_t nkb = (a.cols + 127) / 128;
  const bool by_rows = a.rows >= 32;
  const int64_t items = row_items(a.rows, nkb, by_rows);
  if (items >= 0x7fffffffll) return cudaErrorInvalidValue;
  fp8_dequant_kernel<T, VEC><<<(unsigned)items, kThreads, 0, s>>>(a, nkb, items, by_rows);
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
