// e4m3 with one fp32 power-of-two scale per block: the scale of a block, and spans of 16 elements between memory, fp32
// and e4m3.  A scale is the smallest 2^e >= 2^-126 with which the block's largest finite magnitude is at most 448; 1 for
// a block without one.  Dividing by it is exact, so the only rounding is the one to e4m3; what is not finite becomes NaN.
#pragma once
#include <cuda_fp8.h>
#include <stdint.h>

#include <type_traits>

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

// Two fp32 operations in one instruction, each rounded as by itself.
struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ explicit F2(float both) : F2(both, both) {}
  __device__ __forceinline__ void get(float& lo, float& hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
};
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(a.v) : "l"(b.v), "l"(c.v));
  return a;
}
__device__ __forceinline__ void scale16(float* f, float s) {
#pragma unroll
  for (int i = 0; i < 16; i += 2) (F2(f[i], f[i + 1]) * F2(s)).get(f[i], f[i + 1]);
}

__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }
// 16 values as e4m3: finite ones or NaN.
__device__ __forceinline__ uint4 e4m3_16(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[4 * i], f[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
           ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2], f[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The same of their products with inv.
__device__ __forceinline__ uint4 e4m3_16(float* f, float inv) {
  scale16(f, inv);
  return e4m3_16(f);
}
// What is not finite as NaN.  Rare: the empty statement keeps the compiler from doing it for every block and selecting after.
__device__ __forceinline__ void only_finite16(float* f, bool special) {
  if (special) {
    asm volatile("");
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (abs_bits(f[i]) >= kInfBits) f[i] = __uint_as_float(0x7fc00000u);
  }
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
  // What follows unpacks the words anew: without this the compiler keeps the fp32 values of an earlier use alive, at twice the
  // registers of the words.
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) asm volatile("" : "+r"(v[i]));
  }
  __device__ __forceinline__ void clear(int n) {   // elements from the n-th on
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(E) == 2) v[i] = 2 * i + 1 < n ? v[i] : 2 * i < n ? v[i] & 0xffffu : 0u;
      else v[i] = i < n ? v[i] : 0u;
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
// The same for a whole warp, whose lanes have the spans of four blocks of 128, eight lanes each.  By elements the blocks go
// through shared memory (kStage bytes a warp), neighbouring elements on neighbouring lanes: a lane that reads or writes its
// own 16 elements one by one touches as many sectors with every instruction as the warp has lanes (3000 x 4095 in bf16,
// decoding: 67 us that way, 17 encoding).
template <class T, int VEC>
struct WarpSpans {
  using E = typename T::elem;
  static constexpr int kPitch = 128 * (int)sizeof(E) + 16, kStage = VEC ? 16 : 4 * kPitch;
  // p: the lane's span, n: elements of the lane's that exist
  static __device__ __forceinline__ void load(Span16<T, VEC>& v, const uint8_t* p, int n, uint8_t* stage) {
    if constexpr (VEC > 0) {
      v.load(p, n);
    } else {
      const int lane = threadIdx.x & 31;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const E* from = (const E*)(uintptr_t)__shfl_sync(0xffffffffu, (unsigned long long)(uintptr_t)p, 8 * b);
        const int have = __reduce_add_sync(0xffffffffu, (lane >> 3) == b ? n : 0);
        E e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i * 32 + lane < have) e[i] = from[i * 32 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i * 32 + lane < have) ((E*)(stage + b * kPitch))[i * 32 + lane] = e[i];
      }
      __syncwarp();
      const uint4* mine = (const uint4*)(stage + (lane >> 3) * kPitch + (lane & 7) * 16 * sizeof(E));
#pragma unroll
      for (int i = 0; i < Span16<T, VEC>::kWords / 4; ++i) {
        const uint4 t = mine[i];
        v.v[4 * i] = t.x;
        v.v[4 * i + 1] = t.y;
        v.v[4 * i + 2] = t.z;
        v.v[4 * i + 3] = t.w;
      }
      v.clear(n);
      __syncwarp();
    }
  }
  static __device__ __forceinline__ void store(const Span16<T, VEC>& v, uint8_t* p, int n, uint8_t* stage) {
    if constexpr (VEC > 0) {
      v.store(p, n);
    } else {
      const int lane = threadIdx.x & 31;
      uint4* mine = (uint4*)(stage + (lane >> 3) * kPitch + (lane & 7) * 16 * sizeof(E));
#pragma unroll
      for (int i = 0; i < Span16<T, VEC>::kWords / 4; ++i) mine[i] = make_uint4(v.v[4 * i], v.v[4 * i + 1], v.v[4 * i + 2], v.v[4 * i + 3]);
      __syncwarp();
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        E* to = (E*)(uintptr_t)__shfl_sync(0xffffffffu, (unsigned long long)(uintptr_t)p, 8 * b);
        const int have = __reduce_add_sync(0xffffffffu, (lane >> 3) == b ? n : 0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i * 32 + lane < have) to[i * 32 + lane] = ((const E*)(stage + b * kPitch))[i * 32 + lane];
      }
      __syncwarp();
    }
  }
};

// Magnitudes as integers, which order as the values do, NaN above everything: 16-bit types two to a word.
template <class T>
struct Mags {
  static constexpr bool kHalf = sizeof(typename T::elem) == 2;
  static constexpr int kWords = kHalf ? 8 : 16;
  uint32_t m[kWords];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) m[i] = 0;
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return kHalf ? __vmaxu2(a, b) : max(a, b); }
  static __device__ __forceinline__ uint32_t mag(uint32_t v) { return v & (kHalf ? 0x7fff7fffu : 0x7fffffffu); }
  // with what is not finite counted as nothing
  static __device__ __forceinline__ uint32_t finite(uint32_t v) {
    const uint32_t a = mag(v);
    if constexpr (!kHalf) {
      return a < kInfBits ? a : 0u;
    } else {
      const uint32_t inf = std::is_same<T, F16>::value ? 0x7c00u : 0x7f80u;
      return ((a & 0xffffu) < inf ? a & 0xffffu : 0u) | ((a >> 16) < inf ? a & 0xffff0000u : 0u);
    }
  }
  template <bool FINITE>
  __device__ __forceinline__ void fold(const uint32_t* v) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) m[i] = larger(m[i], FINITE ? finite(v[i]) : mag(v[i]));
  }
  // fp32 bits of one magnitude
  static __device__ __forceinline__ uint32_t bits(uint32_t h) {
    if constexpr (!kHalf) return h;
    else if constexpr (std::is_same<T, BF16>::value) return h << 16;
    else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
  }
  __device__ __forceinline__ uint32_t of(int column) const {   // raw, before bits()
    if constexpr (!kHalf) return m[column];
    else return (column & 1) ? m[column >> 1] >> 16 : m[column >> 1] & 0xffffu;
  }
  __device__ __forceinline__ uint32_t top() const {            // fp32 bits of the largest
    uint32_t t = m[0];
#pragma unroll
    for (int i = 1; i < kWords; ++i) t = larger(t, m[i]);
    if constexpr (kHalf) t = max(t & 0xffffu, t >> 16);
    return bits(t);
  }
};

// Largest finite value of a type, for restored values that rounding took past it: 448 times a scale above `scale` (2^119,
// 2^7 for fp16) may be.
template <class T>
struct MaxOf;
template <>
struct MaxOf<F32> { static constexpr float value = 3.4028234663852886e38f, scale = 6.646139978924579e35f; };
template <>
struct MaxOf<F16> { static constexpr float value = 65504.f, scale = 128.f; };
template <>
struct MaxOf<BF16> { static constexpr float value = 3.3895313892515355e38f, scale = 6.646139978924579e35f; };
// v within +- m, NaN kept
__device__ __forceinline__ float clamp_nan(float v, float m) {
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(m));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(-m));
  return v;
}
// 16 payload values times their scale, within T's range
template <class T>
__device__ __forceinline__ void restore16(const u128& w, float scale, float* f) {
  e4m3_16_to_float(make_uint4((uint32_t)w.x, (uint32_t)(w.x >> 32), (uint32_t)w.y, (uint32_t)(w.y >> 32)), f);
  scale16(f, scale);
  if (!(fabsf(scale) <= MaxOf<T>::scale)) {
    asm volatile("");
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = clamp_nan(f[i], MaxOf<T>::value);
  }
}

// Where a thread of the row-block kernels works: eight lanes share a block of 128, 16 elements each, and a CTA of 256
// threads has 32 groups of U neighbouring blocks: of 32 rows where there are that many (their scales are neighbours in
// memory), else of one row.  The grid has a column of CTAs for each 32 rows (or row) where it may be that high, else CTAs
// find their place by a division; 64-bit divisions and one block a thread cost as much as the work on the block.
struct RowGrid {
  int64_t rows, cols;
  uint32_t across;      // CTAs across a row
  bool flat;            // one row of CTAs
};
template <int U>
__host__ inline cudaError_t row_grid(int64_t rows, int64_t cols, RowGrid* g, dim3* grid) {
  const int64_t groups = (cols + 128 * U - 1) / (128 * U), across = rows >= 32 ? groups : (groups + 31) / 32,
                down = rows >= 32 ? (rows + 31) / 32 : rows;
  if (across * down >= 0x7fffffffll) return cudaErrorInvalidValue;
  *g = {rows, cols, (uint32_t)across, down > 65535};
  *grid = g->flat ? dim3((unsigned)(across * down)) : dim3((unsigned)across, (unsigned)down);
  return cudaSuccess;
}
template <int U>
struct Place {
  int64_t row, c0;      // the lane's first span; the others are 128 elements on
  uint32_t kb;          // its block
  int64_t left;         // elements of the row from that block on, 0 if there is no such row
  __device__ __forceinline__ explicit Place(const RowGrid& g) {
    const int gr = threadIdx.x >> 3;
    uint32_t down = blockIdx.y, at = blockIdx.x;
    if (g.flat) {
      down = blockIdx.x / g.across;
      at = blockIdx.x - down * g.across;
    }
    if (g.rows >= 32) {
      row = (int64_t)down * 32 + gr;
      kb = at * U;
    } else {
      row = down;
      kb = (at * 32 + gr) * U;
    }
    const int64_t b0 = (int64_t)kb * 128;
    c0 = b0 + (threadIdx.x & 7) * 16;
    left = row < g.rows ? g.cols - b0 : 0;
  }
  // elements of span u that exist, and whether its block has any
  __device__ __forceinline__ int n(int u) const {
    return (int)min((int64_t)16, max((int64_t)0, left - (128 * u + (int)(threadIdx.x & 7) * 16)));
  }
  __device__ __forceinline__ bool live(int u) const { return left > 128 * u; }
};

// fp32 bits of the largest finite magnitudes of the row blocks that this lane's spans are parts of, all lanes of the warp
// together; true if something in them was not finite.
template <class T, int VEC, int U>
__device__ __forceinline__ bool row_tops(const Span16<T, VEC>* v, uint32_t* top) {
  auto reduce = [&] {
#pragma unroll
    for (int d = 1; d < 8; d <<= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) top[u] = max(top[u], __shfl_xor_sync(0xffffffffu, top[u], d));
  };
  Mags<T> m;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    m.clear();
    m.template fold<false>(v[u].v);
    top[u] = m.top();
  }
  reduce();
  uint32_t all = top[0];
#pragma unroll
  for (int u = 1; u < U; ++u) all = max(all, top[u]);
  const bool special = __any_sync(0xffffffffu, all >= kInfBits);
  if (special) {
    asm volatile("");   // rare, as above
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m.clear();
      m.template fold<true>(v[u].v);
      top[u] = m.top();
    }
    reduce();
  }
  return special;
}
// Encodes the 16 values of this lane as part of its row block.  All lanes of the warp take part.
template <class T, int VEC>
__device__ __forceinline__ uint4 encode_row16(const Span16<T, VEC>& v, float* f, uint32_t* exp_out) {
  uint32_t top;
  only_finite16(f, row_tops<T, VEC, 1>(&v, &top));
  *exp_out = fp8_scale_exp(top);
  return e4m3_16(f, fp8_inverse(*exp_out));
}

}  // namespace mt
