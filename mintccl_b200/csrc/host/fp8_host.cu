// Host side of the operators on e4m3 tensors with one fp32 scale per block of 128: checks of arguments, TMA descriptors,
// choice of tiles, launches.
#include <cuda.h>
#include <cuda_runtime.h>
#include <string.h>

#include <atomic>

#include <string>

#include "../kernels/fp8.h"
#include "comm_internal.h"

using mthost::fail;

namespace {

int elem_size(int dtype) { return dtype == 0 ? 4 : dtype == 1 || dtype == 2 ? 2 : 0; }

// No exception leaves a C entry point.
template <class F>
int guarded(F f) noexcept {
  try {
    return f();
  } catch (...) {
    return -1;
  }
}
int launched(cudaError_t e, const char* what) {
  return e == cudaSuccess ? 0 : fail(std::string(what) + ": " + cudaGetErrorString(e));
}

// The widest vectors in which rows `ld` elements apart may be accessed: 2 (32 bytes), 1 (16) or 0 (elements).
int vec_of(const void* p, int64_t ld, int esz) {
  const uint64_t bits = (uint64_t)(uintptr_t)p | (uint64_t)(ld * esz);
  return bits % 32 == 0 ? 2 : bits % 16 == 0 ? 1 : 0;
}
int narrower(int a, int b) { return a < b ? a : b; }

// SMs of the current device, asked for once.
int sms_here() {
  static std::atomic<int> known[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev > 63) return mthost::sm_count(dev);
  int n = known[dev].load(std::memory_order_relaxed);
  if (!n) known[dev].store(n = mthost::sm_count(dev), std::memory_order_relaxed);
  return n;
}

// Columns of a tile of 256 rows where the tensor core applies the scales.  In 10 ns: a wave of 256 columns takes 35 a block of
// 128 along K and 300 beside, and the last one 150 until its only accumulator is stored; a wave of 128 columns 22 and 136.
// Measured (us, 256 / 128 columns, when the rule was made): 8192 x 1792 x 4096 51.0 / 56.1, 8192 x 4096 x 4096 99.8 / 116.0, 8192 x 4096 x 1792 50.5 /
// 59.2, 1792 x 4096 x 8192 51.0 / 61.0, 1024 x 4096 x 4096 16.8 / 19.2, 8192 x 512 x 8192 37.7 / 45.4, 2048 x 2048 x 2048
// 14.1 / 13.2, 1024 x 14336 x 512 21.0 / 20.3.
int pow2_columns(int64_t row_tiles, int64_t N, int64_t blocks, int64_t clusters) {
  auto waves = [&](int bn) { return (row_tiles * ((N + bn - 1) / bn) + clusters - 1) / clusters; };
  return waves(256) * (35 * blocks + 300) + 150 <= waves(128) * (22 * blocks + 136) ? 256 : 128;
}

int check_matrix(int64_t rows, int64_t cols, int64_t ldq, int dtype) {
  if (rows <= 0 || cols <= 0) return fail("rows and columns must be positive");
  if (!elem_size(dtype)) return fail("dtype must be fp32, fp16 or bf16");
  if (ldq < cols || ldq % 16) return fail("payload rows must be a multiple of 16 bytes apart");
  return 0;
}
int check_pair(const void* data, const void* scale) {
  if (!data != !scale) return fail("a payload goes with its scales");
  if ((uintptr_t)data & 15) return fail("payloads must be 16-byte aligned");
  return 0;
}
mt::Fp8Out row_blocks(void* data, void* scale, int64_t rows) { return {(uint8_t*)data, (float*)scale, 1, rows}; }

}  // namespace

extern "C" {

int mt_fp8_quantize(void* stream, int dtype, const void* x, int64_t ldx, int64_t rows, int64_t cols, int64_t ldq,
                    void* row_data, void* row_scale, void* col_data, void* col_scale, void* tile_data, void* tile_scale) {
  return guarded([&]() -> int {
    if (check_matrix(rows, cols, ldq, dtype) || check_pair(row_data, row_scale) || check_pair(col_data, col_scale) ||
        check_pair(tile_data, tile_scale))
      return -1;
    if (!x || ldx < 0 || (!row_data && !col_data && !tile_data)) return fail("nothing to encode");
    mt::Fp8QuantArgs a;
    memset(&a, 0, sizeof(a));
    a.x = x;
    a.ldx = ldx;
    a.ldq = ldq;
    a.rows = rows;
    a.cols = cols;
    a.vec = vec_of(x, ldx, elem_size(dtype));
    a.row = row_blocks(row_data, row_scale, rows);
    a.col = {(uint8_t*)col_data, (float*)col_scale, cols, 1};
    a.tile = {(uint8_t*)tile_data, (float*)tile_scale, (cols + 127) / 128, 1};
    return launched(mt::launch_fp8_quant(dtype, a, (cudaStream_t)stream), "fp8 encoding");
  });
}

int mt_fp8_dequantize(void* stream, int dtype, const void* data, int64_t ldq, const void* scale, int64_t s_row, int64_t s_col,
                      int64_t rows, int64_t cols, int row_block, int col_block, void* out, int64_t ldo) {
  return guarded([&]() -> int {
    if (check_matrix(rows, cols, ldq, dtype) || check_pair(data, scale)) return -1;
    if (!data || !out || ldo < cols) return fail("bad operands");
    if ((row_block != 1 && row_block != 128) || (col_block != 1 && col_block != 128)) return fail("blocks are of 1 or 128");
    mt::Fp8DequantArgs a;
    memset(&a, 0, sizeof(a));
    a.data = (const uint8_t*)data;
    a.scale = (const float*)scale;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.rows = rows;
    a.cols = cols;
    a.s_row = s_row;
    a.s_col = s_col;
    a.rshift = row_block == 128 ? 7 : 0;
    a.cshift = col_block == 128 ? 7 : 0;
    a.vec = vec_of(out, ldo, elem_size(dtype));
    return launched(mt::launch_fp8_dequant(dtype, a, (cudaStream_t)stream), "fp8 decoding");
  });
}

int mt_fp8_act_forward(void* stream, int dtype, const void* h, int64_t ldh, const void* u, int64_t ldu, int64_t rows, int64_t cols,
                       void* y, int64_t ldy, int64_t ldq, void* h_data, void* h_scale, void* u_data, void* u_scale) {
  return guarded([&]() -> int {
    if (check_matrix(rows, cols, ldq, dtype) || check_pair(h_data, h_scale) || check_pair(u_data, u_scale)) return -1;
    if (!h || !y || !h_data || ldh < 0 || ldy < cols || !u != !u_data || (u && ldu < 0)) return fail("bad operands");
    const int esz = elem_size(dtype);
    mt::Fp8ActArgs a;
    memset(&a, 0, sizeof(a));
    a.h = h;
    a.u = u;
    a.y = y;
    a.ldh = ldh;
    a.ldu = ldu;
    a.ldy = ldy;
    a.ldq = ldq;
    a.rows = rows;
    a.cols = cols;
    a.kh = row_blocks(h_data, h_scale, rows);
    a.ku = row_blocks(u_data, u_scale, rows);
    a.vec = narrower(vec_of(h, ldh, esz), vec_of(y, ldy, esz));
    if (u) a.vec = narrower(a.vec, vec_of(u, ldu, esz));
    return launched(mt::launch_fp8_act_forward(dtype, a, (cudaStream_t)stream), "fp8 activation");
  });
}

int mt_fp8_act_backward(void* stream, int dtype, int64_t ldq, const void* h_data, const void* h_scale, int64_t h_srow, int64_t h_scol,
                        const void* u_data, const void* u_scale, int64_t u_srow, int64_t u_scol, const void* dy, int64_t lddy,
                        int64_t rows, int64_t cols, void* dh, void* du, void* y) {
  return guarded([&]() -> int {
    if (check_matrix(rows, cols, ldq, dtype) || check_pair(h_data, h_scale) || check_pair(u_data, u_scale)) return -1;
    if (!h_data || !dy || !dh || lddy < 0 || !u_data != !du) return fail("bad operands");
    const int esz = elem_size(dtype);
    mt::Fp8ActArgs a;
    memset(&a, 0, sizeof(a));
    a.dy = dy;
    a.y = y;
    a.dh = dh;
    a.du = du;
    a.kh = {(uint8_t*)h_data, (float*)h_scale, h_srow, h_scol};
    a.ku = {(uint8_t*)u_data, (float*)u_scale, u_srow, u_scol};
    a.lddy = lddy;
    a.ldy = a.lddh = a.lddu = cols;
    a.ldq = ldq;
    a.rows = rows;
    a.cols = cols;
    a.vec = narrower(vec_of(dy, lddy, esz), vec_of(dh, cols, esz));
    if (du) a.vec = narrower(a.vec, vec_of(du, cols, esz));
    if (y) a.vec = narrower(a.vec, vec_of(y, cols, esz));
    return launched(mt::launch_fp8_act_backward(dtype, a, (cudaStream_t)stream), "fp8 activation gradient");
  });
}

static int gemm(void* stream, const void* A, int64_t lda, const void* sa, int64_t sa_m, int64_t sa_k, const void* B, int64_t ldb,
                const void* sb, int64_t sb_n, int64_t sb_k, void* C, int64_t ldc, int dtype, int64_t M, int64_t N, int64_t K,
                int ta, int tb, int nctas, bool pow2) {
  return guarded([&]() -> int {
    if (M <= 0 || N <= 0 || K <= 0 || M > 0x7fff0000ll || N > 0x7fff0000ll || K > 0x7fff0000ll) return fail("bad GEMM shape");
    if (ta && !tb) return fail("ta goes with tb");
    if (!A || !B || !sa || !sb || !C || !elem_size(dtype) || ldc < N) return fail("bad GEMM operands");
    if (lda < (ta ? M : K) || ldb < (tb ? N : K)) return fail("rows of an operand overlap");
    const int sms = nctas > 0 ? nctas : sms_here();
    // Pairs where single CTAs would need more than one wave.  Fewer tiles than half the SMs: CTAs share a tile along K, at
    // least eight blocks each; adding up and the skew of the CTAs cost about 2 us, a block 0.25.  Measured (us, 1 / 2 / 4 / 8
    // CTAs a tile): 1 x 4096 x 4096 12.6 / 10.2 / 8.9, 128 x 1024 x 8192 21.3 / 15.5 / 11.5 / 10.2, 64 x 64 x 8192 22.1 / 15.4 /
    // 10.6 / 8.1, 1001 x 1111 x 2050 13.0 / 11.0; 128 x 4096 x 1792 (14 blocks) 8.6 / 9.3 / 9.0.
    const int64_t nt = (N + 127) / 128, singles = (M + 127) / 128 * nt, blocks = (K + 127) / 128;
    const bool pair = M > 128 && sms > 1 && singles > sms;
    const int bn = pair && pow2 ? pow2_columns((M + 255) / 256, N, blocks, sms / 2) : 128;
    const int64_t tiles = pair ? (M + 255) / 256 * ((N + bn - 1) / bn) : singles;
    int split = 1;
    while (!pair && split < 8 && tiles * split * 2 <= sms && split * 16 <= blocks) split *= 2;
    if (tiles > 0x3fffffffll) return fail("GEMM shape: too many tiles");
    mt::Fp8GemmArgs a;
    memset(&a, 0, sizeof(a));
    // K-major: boxes of 128 K x the CTA's rows; stored transposed: its columns x 128 K rows
    if (ta ? mthost::make_u8_map(&a.a, A, K, M, lda, 128) : mthost::make_u8_map(&a.a, A, M, K, lda, 128)) return -1;
    if (tb ? mthost::make_u8_map(&a.b, B, K, N, ldb, 128, pair ? bn / 2 : 128) : mthost::make_u8_map(&a.b, B, N, K, ldb, pair ? bn / 2 : 128)) return -1;
    a.sa = (const float*)sa;
    a.sb = (const float*)sb;
    a.sa_m = sa_m;
    a.sa_k = sa_k;
    a.sb_n = sb_n;
    a.sb_k = sb_k;
    a.c = C;
    a.ldc = ldc;
    a.M = (int32_t)M;
    a.N = (int32_t)N;
    a.K = (int32_t)K;
    a.out_dtype = dtype;
    a.vec_out = vec_of(C, ldc, elem_size(dtype)) > 0;
    a.timeout_ns = 4000000000ull;
    const int units = pair ? sms / 2 : sms, used = (int)(tiles < units ? tiles : units);
    const int grid = pair ? 2 * used : split > 1 ? split * (int)tiles : used;
    if (launched(mt::launch_fp8_gemm(bn, pair, pow2, split, ta != 0, tb != 0, a, grid, (cudaStream_t)stream), "fp8 gemm"))
      return -1;
    mthost::stat_add(mthost::ST_GEMM, (uint64_t)(2.0 * M * N * K));
    return 0;
  });
}

int mt_gemm_fp8(void* stream, const void* A, int64_t lda, const void* sa, int64_t sa_m, int64_t sa_k, const void* B, int64_t ldb,
                const void* sb, int64_t sb_n, int64_t sb_k, void* C, int64_t ldc, int dtype, int64_t M, int64_t N, int64_t K,
                int ta, int tb, int nctas) {
  return gemm(stream, A, lda, sa, sa_m, sa_k, B, ldb, sb, sb_n, sb_k, C, ldc, dtype, M, N, K, ta, tb, nctas, false);
}

static int packed(void* stream, int op, const int64_t* v) {
  if (!v) return fail("no arguments");
  auto p = [&](int i) { return (void*)(uintptr_t)v[i]; };
  switch (op) {
    case MT_FP8_QUANTIZE:
      return mt_fp8_quantize(stream, (int)v[0], p(1), v[2], v[3], v[4], v[5], p(6), p(7), p(8), p(9), p(10), p(11));
    case MT_FP8_DEQUANTIZE:
      return mt_fp8_dequantize(stream, (int)v[0], p(1), v[2], p(3), v[4], v[5], v[6], v[7], (int)v[8], (int)v[9], p(10), v[11]);
    case MT_FP8_ACT_FORWARD:
      return mt_fp8_act_forward(stream, (int)v[0], p(1), v[2], p(3), v[4], v[5], v[6], p(7), v[8], v[9], p(10), p(11), p(12), p(13));
    case MT_FP8_ACT_BACKWARD:
      return mt_fp8_act_backward(stream, (int)v[0], v[1], p(2), p(3), v[4], v[5], p(6), p(7), v[8], v[9], p(10), v[11], v[12], v[13],
                                 p(14), p(15), p(16));
    case MT_FP8_GEMM:
      return gemm(stream, p(0), v[1], p(2), v[3], v[4], p(5), v[6], p(7), v[8], v[9], p(10), v[11], (int)v[12], v[13], v[14], v[15],
                  (int)v[16], (int)v[17], (int)v[18], v[19] != 0);
    case MT_FP8_LINEAR_FORWARD: {
      const int64_t T = v[3], K = v[4], N = v[8], ldq = (K + 15) / 16 * 16;
      if (mt_fp8_quantize(stream, (int)v[0], p(1), v[2], T, K, ldq, p(9), p(10), nullptr, nullptr, p(11), p(12))) return -1;
      if (v[6] && mt_fp8_quantize(stream, (int)v[5], p(6), v[7], N, K, v[14], nullptr, nullptr, nullptr, nullptr, p(13), p(15))) return -1;
      return gemm(stream, p(9), ldq, p(10), 1, T, p(13), v[14], p(15), v[16], v[17], p(18), N, (int)v[0], T, N, K, 0, 0, 0, v[19] != 0);
    }
    case MT_FP8_LINEAR_BACKWARD: {
      const int64_t T = v[3], N = v[4], K = v[5], ldq = (N + 15) / 16 * 16, ldx = (K + 15) / 16 * 16;
      const bool want_x = v[13] != 0, want_w = v[18] != 0, pow2 = v[20] != 0;
      if (mt_fp8_quantize(stream, (int)v[0], p(1), v[2], T, N, ldq, want_x ? p(6) : nullptr, want_x ? p(7) : nullptr,
                          want_w ? p(14) : nullptr, want_w ? p(15) : nullptr, nullptr, nullptr))
        return -1;
      if (want_x && gemm(stream, p(6), ldq, p(7), 1, T, p(8), v[9], p(10), v[12], v[11], p(13), K, (int)v[0], T, K, N, 0, 1, 0, pow2))
        return -1;
      if (want_w && gemm(stream, p(14), ldq, p(15), 1, N, p(16), ldx, p(17), 1, (K + 127) / 128, p(18), K, (int)v[19], N, K, T, 1, 1, 0, pow2))
        return -1;
      return 0;
    }
    default: return fail("unknown operation");
  }
}

int mt_fp8_packed(void* stream, int op, const int64_t* v) {
  return guarded([&]() -> int { return packed(stream, op, v); });
}

int mt_gemm_fp8_error(void) {
  return guarded([&]() -> int {
    int expired = 0;
    return launched(mt::fp8_gemm_error(&expired), "fp8 gemm status") ? -1 : expired;
  });
}

int mt_test_gemm_fp8_expire(void* stream) {
  return guarded([&]() -> int { return launched(mt::launch_fp8_gemm_expire((cudaStream_t)stream), "launch"); });
}

}  // extern "C"
