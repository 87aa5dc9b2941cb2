// nc_lowbit.h — the 8-bit layer operators: formats, launch contexts and device helpers.
//
// Three code formats (nc_code_format):
//   NC_CODES_ROW    int8 codes, one float scale per row: s = max(fl(amax / 127), 2^-126),
//                   q = the integer nearest to x / s (ties to even), value = q s.
//   NC_CODES_GROUP  int8 codes, one byte per 32 neighbouring columns: the step is the power of
//                   two 2^(byte - 127), the least one with 127 steps >= the group's amax.
//   NC_CODES_RELU   uint8 codes of max(x, 0), one byte per 32 columns: code 0 says x <= 0 (so the
//                   code is ReLU's derivative too), code c > 0 stands for (c - 1) steps, 254
//                   steps >= amax.
// A group or row that holds an infinity or a NaN gets byte 255 (scale NaN) and codes that stand
// for 0 steps: all its values are NaN, so the fault stays visible.  A step is a power of two
// so that every value (at most 8 significant bits) is exact in float, bfloat16 and half: the
// weight gradient multiplies the checkpoint's values without a rounding of their own.
// Codes are stored in rows of code_stride bytes, a multiple of 128, with codes of 0 behind the
// last column, so the matrix kernels read whole 128-byte slices of every row.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "nc_device.h"
#include "nc_internal.h"

namespace nc {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int CODE_GROUP = 32;   // columns that share a step
constexpr int CODE_ALIGN = 128;  // code rows: bytes
constexpr int ROW_ALIGN = 64;    // padded 16-bit rows: elements (128 bytes)

__host__ __device__ inline int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// ---- elementwise: codes, padded 16-bit copies, three-plane splits, transposes, sums --------------
struct CodeCtx {
  int32_t dtype, format;   // nc_dtype of x / values, nc_code_format (-1: no codes)
  int64_t rows, cols;
  const void* x;           // [rows][x_stride] elements
  int64_t x_stride;
  uint8_t* codes;          // [rows][code_stride]
  int64_t code_stride;
  void* scales;            // ROW: float [rows]; else uint8 [rows][code_stride / 32]
  void* values;            // decode: [rows][x_stride]
  // encode of the layer's input: what the matrix kernel reads besides
  int32_t relu;            // max(x, 0) in the 16-bit copy / planes
  uint16_t* copy;          // 16-bit x: [rows][copy_stride]; float x: three bfloat16 planes of that
  int64_t copy_stride;     // elements, a multiple of 64
  int64_t plane;           // elements between planes
};
int launch_encode(const CodeCtx& c, hipStream_t s);   // ROW, or groups (+ copy), or copy alone
int launch_decode(const CodeCtx& c, hipStream_t s);

// dst[c][r] = src[r][c], rows padded with zeros to dst_stride (a multiple of 64); float: three planes
struct TransposeCtx {
  int32_t dtype;
  int64_t rows, cols;
  const void* src;
  int64_t src_stride;
  uint16_t* dst;
  int64_t dst_stride, plane;
};
int launch_transpose(const TransposeCtx& c, hipStream_t s);

// ---- C[m][n] = sum over plane pairs of A_p[m][:] . B_p[n][:] (both row-major along the sum) --------
struct LowGemm {
  const uint8_t* A;        // rows of lda bytes: int8 codes or 16-bit elements, 128-byte slices
  const uint8_t* B;
  int64_t lda, ldb;        // bytes
  int64_t plane_a, plane_b;  // bytes between planes (segments > 1)
  int64_t M, N;
  int32_t slices;          // 128-byte slices of a row
  int32_t segments;        // 1, or 6: the plane pairs of a float product
  int32_t mode;            // LOW_I8 / LOW_BF16 / LOW_F16
  int32_t out_dtype, bias_dtype, relu;
  void* out;               // [M][ldc] elements
  int64_t ldc;
  const void* bias;        // [N] or NULL
  const float* row_scale;  // LOW_I8: [M], [N]
  const float* col_scale;
  const uint8_t* mask;     // output zeroed where the code [m][n] is 0, or NULL
  int64_t ldm;
};
enum LowMode { LOW_I8 = 0, LOW_BF16, LOW_F16 };
int launch_low_gemm(const LowGemm& g, hipStream_t s);

// ---- dW[n][k] = sum_m dY[m][n] value(code[m][k]) --------------------------------------------------
struct LowWgrad {
  const uint16_t* dy;      // planes x [M][ldy]: 16-bit elements, rows 16-byte aligned
  int64_t ldy, plane;      // elements
  int32_t planes;          // 1 or 3
  int32_t f16, relu;       // element type (else bfloat16), code format (RELU else GROUP)
  const uint8_t* codes;
  const uint8_t* steps;
  int64_t code_stride;
  int64_t M, N, K;
  float* part;             // [splits][N][K]
  int32_t splits;
  int64_t rows_per;        // rows of a split, a multiple of 64
};
int launch_low_wgrad(const LowWgrad& g, hipStream_t s);
void low_wgrad_splits(int64_t M, int64_t N, int64_t K, int32_t& splits, int64_t& rows_per);

// out[e] = sum_s part[s][e] in order, as dtype
int launch_sum_parts(const float* part, int64_t n, int32_t splits, void* out, int32_t dtype, hipStream_t s);
// part[slice][c] = sums of x's columns over a slice of rows
int launch_col_sums(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t stride, int32_t slices,
                    float* part, hipStream_t s);

// ---- device helpers -------------------------------------------------------------------------------
__device__ __forceinline__ float bf16_f32(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
__device__ __forceinline__ uint16_t f32_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }

template <int DT>
__device__ __forceinline__ float elem_f32(uint16_t b) {
  return DT == NC_BF16 ? bf16_f32(b) : (float)__builtin_bit_cast(_Float16, b);
}
template <int DT>
__device__ __forceinline__ uint16_t f32_elem(float x) {  // round to nearest even
  return DT == NC_BF16 ? f32_bf16(x) : __builtin_bit_cast(uint16_t, (_Float16)x);
}

// x = p[0] + p[1] + p[2] in bfloat16, each the rounding of what is left: 24 significant bits at
// least for |x| >= 2^-100.  A finite x whose rounding would overflow is cut instead; an
// infinity or NaN goes into the first plane alone.
__device__ __forceinline__ void split3(float x, uint16_t (&p)[3]) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const uint32_t mag = u & 0x7fffffffu;
  p[0] = f32_bf16(x);
  if (mag >= 0x7f7f8000u) {  // would round to infinity, or is not finite
    const bool nan = mag > 0x7f800000u;
    p[0] = nan ? 0x7fc0 : (uint16_t)(u >> 16);
    if (mag >= 0x7f800000u) {
      p[1] = p[2] = 0;
      return;
    }
  }
  const float r1 = x - bf16_f32(p[0]);
  p[1] = f32_bf16(r1);
  p[2] = f32_bf16(r1 - bf16_f32(p[1]));
}

// biased exponent of a group's step from the bits of its amax (magnitude bits)
__device__ __forceinline__ int step_byte(uint32_t amax, bool relu) {
  if (amax >= 0x7f800000u) return 255;
  int e = (int)((amax + 0x1ffffu) >> 23);  // + 1 when the mantissa is over 127/64
  e = (e > 254 ? 254 : e) - (relu ? 7 : 6);
  return e < 1 ? 1 : e;
}

}  // namespace nc
