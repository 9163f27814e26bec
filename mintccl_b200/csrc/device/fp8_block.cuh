// e4m3 with one fp32 power-of-two scale per block: the scale of a block, and spans of 16 elements between memory, fp32
// and e4m3.  A scale is the smallest 2^e >= 2^-126 with which the block's largest finite magnitude is at most 448; 1 for
// a block without one.  Dividing by it is exact, so the only rounding is the one to e4m3; what is not finite becomes NaN.
#pragma once
#include <cuda_fp8.h>
#include <stdint.h>

#include "prims.cuh"
#include "reduce_ops.cuh"

namespace mt {

constexpr uint32_t kInfBits = 0x7f800000u;

// Exponent (biased by 127) of the scale for a block whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t fp8_scale_exp(uint32_t amax) {
  if (amax == 0) return 127;
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);   // 448 = 1.75 * 2^8
  return (uint32_t)max(e, 1);
}
__device__ __forceinline__ float fp8_scale(uint32_t e) { return __uint_as_float(e << 23); }
__device__ __forceinline__ float fp8_inverse(uint32_t e) { return __uint_as_float((254u - e) << 23); }   // e <= 247

__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t finite_bits(float f) {
  const uint32_t b = abs_bits(f);
  return b < kInfBits ? b : 0u;
}
// 16 values (quotients by the scale) as e4m3.  `special`: some may not be finite.
__device__ __forceinline__ uint4 e4m3_16(const float* f, float inv, bool special) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = f[4 * i + j] * inv;
      if (special && abs_bits(f[4 * i + j]) >= kInfBits) v[j] = __uint_as_float(0x7fc00000u);
    }
    w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3) |
           ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3) << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void e4m3_16_to_float(const uint4& q, float* f) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&h));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

__device__ __forceinline__ void ld_vec32(const uint8_t* p, uint32_t* v) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p));
}
__device__ __forceinline__ void st_vec32(uint8_t* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// 16 consecutive elements in flight.  VEC 2: 32-byte vectors, 1: 16-byte ones, 0: by elements.  `n` of them exist (a
// vector is only read where all do); the others are zeros.
template <class T, int VEC>
struct Span16 {
  using E = typename T::elem;
  static constexpr int kWords = 4 * (int)sizeof(E);
  uint32_t v[kWords];
  __device__ __forceinline__ void load(const uint8_t* p, int n) {
    if (VEC > 0 && n >= 16) {
      if constexpr (VEC == 2) {
#pragma unroll
        for (int i = 0; i < kWords / 8; ++i) ld_vec32(p + 32 * i, v + 8 * i);
      } else {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
          const u128 t = load128_stream(p + 16 * i);
          v[4 * i] = (uint32_t)t.x;
          v[4 * i + 1] = (uint32_t)(t.x >> 32);
          v[4 * i + 2] = (uint32_t)t.y;
          v[4 * i + 3] = (uint32_t)(t.y >> 32);
        }
      }
    } else if constexpr (sizeof(E) == 2) {
      const uint16_t* e = (const uint16_t*)p;
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        v[i] = (2 * i < n ? (uint32_t)__ldg(e + 2 * i) : 0u) | (2 * i + 1 < n ? (uint32_t)__ldg(e + 2 * i + 1) << 16 : 0u);
    } else {
      const uint32_t* e = (const uint32_t*)p;
#pragma unroll
      for (int i = 0; i < kWords; ++i) v[i] = i < n ? __ldg(e + i) : 0u;
    }
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < kWords / 2; ++i) T::unpack((uint64_t)v[2 * i] | ((uint64_t)v[2 * i + 1] << 32), f + i * T::kPer64);
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int i = 0; i < kWords / 2; ++i) {
      const uint64_t w = T::pack(f + i * T::kPer64);
      v[2 * i] = (uint32_t)w;
      v[2 * i + 1] = (uint32_t)(w >> 32);
    }
  }
  __device__ __forceinline__ void store(uint8_t* p, int n) const {
    if (VEC > 0 && n >= 16) {
      if constexpr (VEC == 2) {
#pragma unroll
        for (int i = 0; i < kWords / 8; ++i) st_vec32(p + 32 * i, v + 8 * i);
      } else {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i)
          *(uint4*)(p + 16 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
    } else if constexpr (sizeof(E) == 2) {
      uint16_t* e = (uint16_t*)p;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if (2 * i < n) e[2 * i] = (uint16_t)v[i];
        if (2 * i + 1 < n) e[2 * i + 1] = (uint16_t)(v[i] >> 16);
      }
    } else {
      uint32_t* e = (uint32_t*)p;
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        if (i < n) e[i] = v[i];
    }
  }
};
// Largest finite value of a type, for restored values that rounding took past it.
template <class T>
struct MaxOf;
template <>
struct MaxOf<F32> { static constexpr float value = 3.4028234663852886e38f; };
template <>
struct MaxOf<F16> { static constexpr float value = 65504.f; };
template <>
struct MaxOf<BF16> { static constexpr float value = 3.3895313892515355e38f; };
// v within +- m, NaN kept
__device__ __forceinline__ float clamp_nan(float v, float m) {
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(m));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(-m));
  return v;
}

// Where a thread of the row-block kernels works: eight lanes share a block of 128, 16 elements each, and a CTA of 256
// threads has 32 blocks per step: 32 rows where there are that many (their scales are neighbours in memory), else 32
// blocks that follow one another along the rows.
struct RowSpan {
  int64_t row, kb;
  bool live;
};
__device__ __forceinline__ RowSpan row_span(int64_t item, int g, int64_t rows, int64_t nkb, bool by_rows) {
  RowSpan r;
  if (by_rows) {
    const int64_t rt = item / nkb;
    r.kb = item - rt * nkb;
    r.row = rt * 32 + g;
    r.live = r.row < rows;
  } else {
    const int64_t id = item * 32 + g;
    r.row = id / nkb;
    r.kb = id - r.row * nkb;
    r.live = r.row < rows;
  }
  return r;
}
// One step of a CTA is an item; this many there are.
__host__ __device__ __forceinline__ int64_t row_items(int64_t rows, int64_t nkb, bool by_rows) {
  return by_rows ? (rows + 31) / 32 * nkb : (rows * nkb + 31) / 32;
}

// Encodes the 16 values of this lane as part of its row block.  All lanes of the warp take part.
__device__ __forceinline__ uint4 encode_row16(const float* f, uint32_t* exp_out) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, abs_bits(f[i]));
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  const bool special = __any_sync(0xffffffffu, m >= kInfBits);
  if (special) {
    m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, finite_bits(f[i]));
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  }
  const uint32_t e = fp8_scale_exp(m);
  *exp_out = e;
  return e4m3_16(f, fp8_inverse(e), special);
}

}  // namespace mt
