// nc_lowbit.h — the 8-bit layer operators: formats, launch contexts and device helpers.
//
// Three code formats (nc_code_format):
//   NC_CODES_ROW    int8 codes, one float scale per row: s = max(fl(amax fl(1 / 127)), 2^-126),
//                   q = the integer nearest to x / s (ties to even), value = q s.
//   NC_CODES_GROUP  int8 codes, one byte per 32 neighbouring columns: the step is the power of
//                   two 2^(byte - 127), the least one with 127 steps >= the group's amax.
//   NC_CODES_RELU   uint8 codes of max(x, 0), one byte per 32 columns: code 0 says x <= 0 (so the
//                   code is ReLU's derivative too), code c > 0 stands for (c - 1) steps, 254
//                   steps >= amax.
// A group or row that holds an infinity or a NaN gets byte 255 (scale NaN) and codes that stand
// for 0 steps: all its values are NaN, so the fault stays visible.  A step is a power of two
// so that every value (at most 8 significant bits) is exact in float and bfloat16, and in half for a
// checkpoint of half values, but one: the code nearest to a magnitude over 65024 (RELU: 65280) stands for
// 65536, which as half is the largest number, 65504, itself within half a step of that magnitude.  The
// weight gradient multiplies the checkpoint's values without another rounding of their own.
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

// ---- elementwise: codes, padded 16-bit copies, float planes, transposes, sums ----------------------
struct CodeCtx {
  int32_t dtype, format;   // nc_dtype of x / values, nc_code_format (-1: no codes)
  int64_t rows, cols;
  const void* x;           // [rows][x_stride] elements
  int64_t x_stride;
  uint8_t* codes;          // [rows][code_stride]
  int64_t code_stride;
  void* scales;            // ROW: float [rows]; else uint8 [rows][code_stride / 32]
  void* values;            // decode: [rows][x_stride]
  int64_t zero_rows;       // decode: rows of zeros behind them
  // encode of the layer's input: what the matrix kernel reads besides
  int32_t relu;            // max(x, 0) in the 16-bit copy
  uint16_t* copy;          // 16-bit x: [rows][copy_stride]
  int64_t copy_stride;     // elements, a multiple of 64
};
int launch_encode(const CodeCtx& c, hipStream_t s);   // ROW, or groups (+ copy), or copy alone
int launch_decode(const CodeCtx& c, hipStream_t s);

// a float matrix as two half planes [rows][dst_stride] (a multiple of 64), each row by a power of two of its own
// (split2): 2^(141 - exponent)
struct SplitCtx {
  int64_t rows, cols;
  const float* x;
  int64_t x_stride;
  uint16_t* dst;
  int64_t dst_stride, plane;  // elements
  int32_t* exponent;       // [rows]
};
int launch_split(const SplitCtx& c, hipStream_t s);

// dst[c][r] = src[r][c], rows padded with zeros to dst_stride (a multiple of 64); float: split planes of it
constexpr int TOP_ROWS = 256;
struct TransposeCtx {
  int32_t dtype;
  int64_t rows, cols;
  const void* src;
  int64_t src_stride;
  uint16_t* dst;
  int64_t dst_stride, plane;
  int32_t* exponent;       // float: [cols]
  uint32_t* tops;          // float: scratch [ceil(rows / TOP_ROWS)][cols]
};
int launch_transpose(const TransposeCtx& c, hipStream_t s);

// ---- C[m][n] = sum_k A[m][k] B[n][k] (both row-major along the sum) --------------------------------
struct LowGemm {
  const uint8_t* A;        // rows of lda bytes: int8 codes or 16-bit elements, 128-byte slices
  const uint8_t* B;
  int64_t lda, ldb;        // bytes
  int64_t plane_b;         // bytes between B's two planes (LOW_F32)
  int64_t M, N;
  int32_t slices;          // 128-byte slices of a row (LOW_F32: of 32 columns)
  int32_t mode;            // LOW_I8 / LOW_BF16 / LOW_F16
  int32_t out_dtype, bias_dtype, relu;
  void* out;               // [M][ldc] elements
  int64_t ldc;
  const void* bias;        // [N] or NULL
  const float* row_scale;  // LOW_I8: [M]
  const float* col_scale;  // LOW_I8: [N]
  const int32_t* exponent; // LOW_F32: [N], of B's rows
  const uint8_t* mask;     // output zeroed where the code [m][n] is 0, or NULL
  int64_t ldm;
  // LOW_F32: A is float [M][lda / 4] with K columns, split into planes while it is staged (B: two planes,
  // slices of 32 columns); a_relu: of max(A, 0); codes: its 8-bit checkpoint is written besides
  int64_t K;
  int32_t a_relu;
  uint8_t* codes;
  uint8_t* steps;
  int64_t code_stride;
  // a sum cut into `splits` parts, part[split][M][N] (float, LOW_I8: int32), when the tiles are few
  int32_t splits;
  float* part;
};
enum LowMode { LOW_I8 = 0, LOW_BF16, LOW_F16, LOW_F32 };
int launch_low_gemm(const LowGemm& g, hipStream_t s);
// LOW_I8 for few rows or few columns: x (of x_dtype, [M][x_stride]) encoded within the kernel, or -1: given codes
struct LowSmall {
  LowGemm g;               // A: the codes (x_dtype = -1)
  int32_t x_dtype;
  const void* x;
  int64_t x_stride;
};
bool low_small_encodes(int64_t M, int64_t N, int64_t K);
int launch_low_small(const LowSmall& a, hipStream_t s);
int low_gemm_splits(int mode, int64_t M, int64_t N, int64_t K);

// ---- dW[n][k] = sum_m dY[m][n] value(code[m][k]) --------------------------------------------------
struct LowWgrad {
  const void* dy;          // [M][ldy] of dtype; 16-bit rows are 16-byte aligned
  int64_t ldy;             // elements
  int32_t dtype, relu;     // nc_dtype; code format (RELU else GROUP)
  const uint8_t* codes;
  const uint8_t* steps;
  int64_t code_stride;
  const uint16_t* x;       // the codes' values, [round_up(M, 64)][code_stride], zeros behind row M; or NULL
  int64_t M, N, K;
  float* part;             // [splits][N][K]
  float* sums;             // [splits][pieces][N]: the columns' sums of dY
  int32_t pieces;
  void* dw;                // splits = 1: dW itself, of dtype; else NULL
  void* db;                // one part: the sums themselves; else NULL
  int32_t want_dw, want_db;
  int32_t splits;
  int64_t rows_per;        // rows of a split, a multiple of 64
};
int launch_low_wgrad(const LowWgrad& g, hipStream_t s);
bool low_wgrad_decodes(int dtype, int64_t M, int64_t N, int64_t K);  // whether it takes x
void low_wgrad_splits(int dtype, int64_t M, int64_t N, int64_t K, bool want_dw, int32_t& splits, int32_t& pieces,
                      int64_t& rows_per);

// out[e] = sum_s part[s][e], in order, as dtype, for two matrices in one launch; out = NULL: none
struct SumParts {
  const float* part[2];
  int64_t n[2];
  int32_t parts[2];
  void* out[2];
};
int launch_sum_parts(const SumParts& a, int32_t dtype, hipStream_t s);

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

__device__ __forceinline__ float relu_keep_nan(float x) { return x <= 0.f ? 0.f : x; }  // (of -0: +0)

// x = x0 + x1 + x2, exactly, in bfloat16: each plane is what is left cut to its upper half (8 significant
// bits, 24 in all; the third is whole by then).  Of 8 values: a plane is 4 words.  Behind an infinity the planes are 0.
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
}
__device__ __forceinline__ float cut_bf16(float x) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u);
}
__device__ __forceinline__ void split3(const float (&x)[8], uint4 (&plane)[3]) {
  float r[8], top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    r[e] = x[e];
    top = __builtin_fmaxf(top, __builtin_fabsf(x[e]));
  }
  const bool infinite = __any(top == __builtin_inff());  // (a wave's own: seldom)
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    plane[k] = uint4{upper_halves(r[0], r[1]), upper_halves(r[2], r[3]), upper_halves(r[4], r[5]), upper_halves(r[6], r[7])};
    if (k < 2)
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = r[e] - cut_bf16(r[e]);
    if (k == 0 && infinite)
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = __builtin_fabsf(x[e]) == __builtin_inff() ? 0.f : r[e];
  }
}

// x scale = x0 + x1 in half, |x scale| < 2^15: x0 the nearest, x1 what is left, rounded.  x1 is given times 2^UP: within
// 2^-22 of |x|, or 2^-(25 + UP) / scale for small ones.  Of 8 values: a plane is 4 words.  An infinity leaves an infinity and a
// NaN, which split2_infinite replaces.  (Written as fused multiply-adds that end in half: one instruction an element and plane.)
template <int UP>
__device__ __forceinline__ void split2(const float (&x)[8], float scale, uint4 (&plane)[2]) {
  uint32_t w[2][4];
  constexpr float up = (float)(1 << UP);
  const float scaled = scale * up;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float v = x[2 * j + k];
      const _Float16 h = (_Float16)__builtin_fmaf(v, scale, 0.f);
      const _Float16 l = (_Float16)(UP ? __builtin_fmaf(-(float)h, up, v * scaled) : __builtin_fmaf(v, scale, -(float)h));
      w[0][j] = k ? w[0][j] | (uint32_t)__builtin_bit_cast(uint16_t, h) << 16 : __builtin_bit_cast(uint16_t, h);
      w[1][j] = k ? w[1][j] | (uint32_t)__builtin_bit_cast(uint16_t, l) << 16 : __builtin_bit_cast(uint16_t, l);
    }
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) plane[p] = uint4{w[p][0], w[p][1], w[p][2], w[p][3]};
}
// the planes of infinities: 0 and the infinity, so that its products are what the formula's are (a wave takes this
// branch where it holds one)
__device__ __forceinline__ void split2_infinite(const float (&x)[8], uint4 (&plane)[2]) {
  uint32_t h[4] = {plane[0].x, plane[0].y, plane[0].z, plane[0].w}, l[4] = {plane[1].x, plane[1].y, plane[1].z, plane[1].w};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool inf = __builtin_fabsf(x[e]) == __builtin_inff();
    const uint32_t keep = inf ? (e & 1 ? 0xffffu : 0xffff0000u) : ~0u;
    const uint32_t v = inf ? (x[e] > 0.f ? 0x7c00u : 0xfc00u) << (e & 1 ? 16 : 0) : 0u;
    h[e / 2] &= keep;
    l[e / 2] = (l[e / 2] & keep) | v;
  }
  plane[0] = uint4{h[0], h[1], h[2], h[3]};
  plane[1] = uint4{l[0], l[1], l[2], l[3]};
}
// biased exponent of the largest magnitude, for scales (times 2^UP) that are normal floats too: zero and what is below
// 2^(UP - 112) count as 15 + UP, infinities as 254
template <int UP>
__device__ __forceinline__ int top_exponent(uint32_t top) { return min(max((int)(top >> 23), 15 + UP), 254); }
// 2^(to - e): what has exponent e is below 2^(to - 126)
__device__ __forceinline__ float scale_to(int to, int e) { return __builtin_bit_cast(float, (uint32_t)(127 + to - e) << 23); }

// biased exponent of a group's step from the bits of its amax (magnitude bits)
__device__ __forceinline__ int step_byte(uint32_t amax, bool relu) {
  const int e = min((int)((amax + 0x1ffffu) >> 23), 254) - (relu ? 7 : 6);  // + 1 when the mantissa is over 127/64
  return amax >= 0x7f800000u ? 255 : max(e, 1);
}

// 16 (8) bytes at any element's address: one instruction, whose address need not be a multiple of its size
template <typename T>
__device__ __forceinline__ T load_any(const void* p) {
  T v;
  __builtin_memcpy(&v, p, sizeof(T));
  return v;
}
template <typename T>
__device__ __forceinline__ void store_any(void* p, T v) {
  __builtin_memcpy(p, &v, sizeof(T));
}
// v[j] = v[j + s], 0 <= s < 8, for the values that are there
template <int BIT>
__device__ __forceinline__ void shift_by(float (&v)[8], bool on) {
#pragma unroll
  for (int j = 0; j < 8 - BIT; ++j) {
    const float there = v[j + BIT], here = v[j];  // (values: a choice of places would put the array into memory)
    v[j] = on ? there : here;
  }
}
__device__ __forceinline__ void shift8(float (&v)[8], int s) {
  shift_by<4>(v, (s & 4) != 0);
  shift_by<2>(v, (s & 2) != 0);
  shift_by<1>(v, (s & 1) != 0);
}

// 8 columns [8 c, 8 c + 8) of a row as float, from any address; clear8 puts zeros for those behind the last.  WIDE:
// rows of at least 8 columns, whose last chunk is loaded as the row's last 8 and moved to its place by clear8, away
// from the loads (what waits for a load keeps the next one from being asked for).
template <int DT>
__device__ __forceinline__ void load8_at(const void* x, int64_t at, float (&v)[8]) {
  if (DT == NC_F32) {
    const float* p = reinterpret_cast<const float*>(x) + at;
    const float4 a = load_any<float4>(p), b = load_any<float4>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = load_any<uint4>(reinterpret_cast<const uint16_t*>(x) + at);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = elem_f32<DT>((uint16_t)w[j]);
      v[2 * j + 1] = elem_f32<DT>((uint16_t)(w[j] >> 16));
    }
  }
}
template <int DT, bool WIDE>
__device__ __forceinline__ void load8(const void* x, int64_t off, int64_t c, int64_t cols, float (&v)[8]) {
  if (WIDE) {
    load8_at<DT>(x, off + (8 * c < cols - 8 ? 8 * c : cols - 8), v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t k = 8 * c + j, at = off + (k < cols ? k : cols - 1);
      v[j] = DT == NC_F32 ? reinterpret_cast<const float*>(x)[at] : elem_f32<DT>(reinterpret_cast<const uint16_t*>(x)[at]);
    }
  }
}
template <bool WIDE>
__device__ __forceinline__ void clear8(int64_t c, int64_t cols, float (&v)[8]) {
  if (WIDE && cols % 8 == 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 8 * c < cols ? v[j] : 0.f;
  } else {
    if (WIDE) shift8(v, 8 * c > cols - 8 ? (int)(8 * c - cols) & 7 : 0);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 8 * c + j < cols ? v[j] : 0.f;
  }
}
inline bool wide8(int64_t cols) { return cols >= 8; }

// the low bytes of 8 words
__device__ __forceinline__ uint2 pack8(const uint32_t (&q)[8]) {
  uint2 r;
  r.x = __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u) | __builtin_amdgcn_perm(q[3], q[2], 0x04000c0cu);
  r.y = __builtin_amdgcn_perm(q[5], q[4], 0x0c0c0400u) | __builtin_amdgcn_perm(q[7], q[6], 0x04000c0cu);
  return r;
}

__device__ __forceinline__ uint32_t mag_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// The code is the integer nearest to the exact quotient x / s: t = rint(x rcp) is at most one off
// next to a half, and the remainder x - t s (exact in a fused multiply-add there: its grid is half an
// ulp of s and it is below s) says on which side of s / 2 the quotient lies.
__device__ __forceinline__ int row_code(float x, float s, float rcp) {
  float t = __builtin_rintf(x * rcp);
  const float r = __builtin_fmaf(-t, s, x), h = 0.5f * s;
  const bool odd = ((int)t & 1) != 0;
  if (r > h || (r == h && odd)) t += 1.f;
  else if (r < -h || (r == -h && odd)) t -= 1.f;
  return (int)__builtin_fminf(__builtin_fmaxf(t, -127.f), 127.f);
}

// a row's scale from its amax (magnitude bits): the product with the rounded 1 / 127, as a float tensor divided by a
// number comes out on this hardware (torch does so), so that codes made there and here are the same.  5 % of rows get
// a neighbour of the rounded quotient, which moves a code only where x / s is next to a half.
__device__ __forceinline__ float row_scale(uint32_t top) {
  return __builtin_fmaxf(__builtin_bit_cast(float, top) * (1.f / 127.f), 0x1p-126f);
}
__device__ __forceinline__ uint2 row_codes(const float (&v)[8], bool bad, float s, float rcp) {
  uint32_t q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = bad ? 0u : (uint32_t)row_code(v[e], s, rcp);
  return pack8(q);
}

// the codes of 8 columns and the step byte of their group, whose other columns the three lanes beside
// (lane ^ 1, 2, 3) hold; RELU: the columns are max(x, 0) already.
// v inv + 1.5 2^23 rounds v / step to an integer, ties to even, in the float's low bits.  The bounds are for
// an amax near the largest float, which no step reaches, and for NaN, of which the median takes the lower.
template <bool RELU>
__device__ __forceinline__ uint2 group_codes(const float (&v)[8], int& sb) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, RELU ? __builtin_bit_cast(uint32_t, v[e]) : mag_bits(v[e]));
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true));  // lane ^ 1
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4e, 0xf, 0xf, true));  // lane ^ 2
  sb = step_byte(top, RELU);
  const float inv = sb == 255 ? 0.f : __builtin_bit_cast(float, (uint32_t)(254 - sb) << 23);
  constexpr float ONE = 12582912.f;
  uint32_t q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = __builtin_amdgcn_fmed3f(__builtin_fmaf(v[e], inv, ONE), RELU ? ONE : ONE - 127.f, ONE + (RELU ? 254.f : 127.f));
    const uint32_t k = __builtin_bit_cast(uint32_t, t);
    q[e] = RELU ? (v[e] <= 0.f ? 0u : k + 1u) : k;
  }
  uint2 w = pack8(q);
  if (!RELU && sb == 255) w = uint2{0u, 0u};
  return w;
}

}  // namespace nc
