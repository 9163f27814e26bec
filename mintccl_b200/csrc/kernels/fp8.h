// Arguments of the kernels for e4m3 tensors with one fp32 scale per block of 128: encoding, decoding, activations whose
// input is kept in 8 bits, and the product.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mt {

// Payload and scales of one encoding.  Scale of block (i, j): scale[i * s_row + j * s_col].
struct Fp8Out {
  uint8_t* data;   // null: not wanted
  float* scale;
  int64_t s_row, s_col;
};

struct Fp8QuantArgs {
  const void* x;           // [rows, cols], rows `ldx` elements apart, columns adjacent
  int64_t ldx, ldq;        // ldq: bytes between payload rows, a multiple of 16; payloads start on 16-byte boundaries
  int64_t rows, cols;
  int32_t vec;             // how rows of x may be read: 2 in 32-byte vectors, 1 in 16-byte ones, 0 by elements
  Fp8Out row, col, tile;   // blocks of 1 x 128, 128 x 1, 128 x 128
};
cudaError_t launch_fp8_quant(int dtype, const Fp8QuantArgs& a, cudaStream_t s);

struct Fp8DequantArgs {
  const uint8_t* data;
  const float* scale;
  void* out;               // [rows, cols], rows `ldo` elements apart
  int64_t ldq, ldo, rows, cols, s_row, s_col;
  int32_t rshift, cshift;  // 7: blocks of 128 along that dimension, 0: of one
  int32_t vec;             // as above, for both sides
};
cudaError_t launch_fp8_dequant(int dtype, const Fp8DequantArgs& a, cudaStream_t s);

// y = silu(h) or silu(h) * u, inputs kept in row blocks; and the gradients from what was kept.
struct Fp8ActArgs {
  const void *h, *u;       // u: null without a gate.  Forward only
  const void* dy;          // backward only
  void *y, *dh, *du;       // y: forward's result; backward: the activation again (null: not wanted)
  Fp8Out kh, ku;           // row blocks of h and u
  int64_t ldh, ldu, lddy, ldy, lddh, lddu, ldq;
  int64_t rows, cols;
  int32_t vec;
};
cudaError_t launch_fp8_act_forward(int dtype, const Fp8ActArgs& a, cudaStream_t s);
cudaError_t launch_fp8_act_backward(int dtype, const Fp8ActArgs& a, cudaStream_t s);

// C[M, N] = sum over blocks kb of 128 along K: sa(m, kb) * sb(n / 128, kb) * A[m, kb] . B[n, kb]
struct Fp8GemmArgs {
  CUtensorMap a, b;
  const float *sa, *sb;
  int64_t sa_m, sa_k, sb_n, sb_k;   // strides of the scales in elements
  void* c;
  int64_t ldc;                      // elements
  int32_t M, N, K;
  int32_t out_dtype;                // DType of C: fp32, fp16 or bf16
  int32_t vec_out;                  // rows of C start on 16-byte boundaries
  uint64_t timeout_ns;
};
// bn: columns of a tile, 128, or 256 with pair and pow2.  pair: 256 rows each, on CTA pairs (nctas even).  Else 128 rows
// each; split (1, 2, 4 or 8): the CTAs that share a tile's blocks along K, at most as many as there are blocks; nctas =
// split * tiles if it is not 1.
// pow2: all scales are powers of two (looked at with pair only).
cudaError_t launch_fp8_gemm(int bn, bool pair, bool pow2, int split, bool ta, bool tb, const Fp8GemmArgs& a, int nctas, cudaStream_t s);
// *expired = 1 if a wait of the product expired on the current device since the last call (waits for the device).
cudaError_t fp8_gemm_error(int* expired);
cudaError_t launch_fp8_gemm_expire(cudaStream_t s);   // a kernel whose wait expires

}  // namespace mt
