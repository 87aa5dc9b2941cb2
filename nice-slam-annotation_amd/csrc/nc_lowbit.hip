// nc_lowbit.hip — codes of the 8-bit layer operators and the copies that their matrix kernels read.
//
// Everything here is one pass over its input and bound by memory: a thread takes 8 neighbouring
// columns (16 or 32 bytes in, 8 bytes of codes out).
#include "nc_lowbit.h"

namespace nc {

static inline unsigned blocks_of(int64_t n, int b) { return (unsigned)((n + b - 1) / b); }

// 8 columns [8 c, 8 c + 8) of a row as float, 0 behind the last one
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* x, int64_t off, int64_t c, int64_t cols, float (&v)[8]) {
  if (DT == NC_F32) {
    const float* p = reinterpret_cast<const float*>(x) + off + 8 * c;
    if (VEC && 8 * c + 8 <= cols) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 8 * c + j < cols ? p[j] : 0.f;
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(x) + off + 8 * c;
    if (VEC && 8 * c + 8 <= cols) {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = elem_f32<DT>((uint16_t)w[j]);
        v[2 * j + 1] = elem_f32<DT>((uint16_t)(w[j] >> 16));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 8 * c + j < cols ? elem_f32<DT>(p[j]) : 0.f;
    }
  }
}

template <int DT, bool VEC>
__device__ __forceinline__ void store8(void* x, int64_t off, int64_t c, int64_t cols, const float (&v)[8]) {
  if (DT == NC_F32) {
    float* p = reinterpret_cast<float*>(x) + off + 8 * c;
    if (VEC && 8 * c + 8 <= cols) {
      reinterpret_cast<float4*>(p)[0] = float4{v[0], v[1], v[2], v[3]};
      reinterpret_cast<float4*>(p)[1] = float4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (8 * c + j < cols) p[j] = v[j];
    }
  } else {
    uint16_t* p = reinterpret_cast<uint16_t*>(x) + off + 8 * c;
    uint16_t e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = f32_elem<DT>(v[j]);
    if (VEC && 8 * c + 8 <= cols) {
      uint4 a;
      a.x = e[0] | (uint32_t)e[1] << 16;
      a.y = e[2] | (uint32_t)e[3] << 16;
      a.z = e[4] | (uint32_t)e[5] << 16;
      a.w = e[6] | (uint32_t)e[7] << 16;
      *reinterpret_cast<uint4*>(p) = a;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (8 * c + j < cols) p[j] = e[j];
    }
  }
}

__device__ __forceinline__ uint2 pack8(const int (&q)[8]) {
  uint2 r;
  r.x = (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | (uint32_t)(q[3] & 255) << 24;
  r.y = (q[4] & 255) | (q[5] & 255) << 8 | (q[6] & 255) << 16 | (uint32_t)(q[7] & 255) << 24;
  return r;
}

// ---- rows with one scale ---------------------------------------------------------------------------
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

__device__ __forceinline__ uint32_t mag_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// NT threads (64 or 1024) own a row; C > 0: its 8-column chunks t, t + NT, ... stay in registers
// (C of them a thread), C = 0: any length, read twice (the second time from the cache).
template <int DT, bool VEC, int NT, int C>
__global__ void __launch_bounds__(NT == 64 ? 256 : NT) k_encode_rows(const CodeCtx a) {
  constexpr int RPW = NT == 64 ? 4 : 1;  // rows a workgroup
  __shared__ uint32_t red[16];
  const int t = NT == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const int64_t r = (int64_t)blockIdx.x * RPW + (NT == 64 ? (threadIdx.x >> 6) : 0);
  if (NT == 64 && r >= a.rows) return;  // whole waves; no barrier in this variant
  const int64_t off = r * a.x_stride, chunks = a.code_stride / 8;
  float v[C > 0 ? C : 1][8];
  uint32_t top = 0;
  if (C > 0) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int64_t c = t + (int64_t)NT * j;
      if (c < chunks) load8<DT, VEC>(a.x, off, c, a.cols, v[j]);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, mag_bits(v[j][e]));
    }
  } else {
    for (int64_t c = t; 8 * c < a.cols; c += NT) {
      load8<DT, VEC>(a.x, off, c, a.cols, v[0]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, mag_bits(v[0][e]));
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  if (NT > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) top = max(top, red[w]);
  }
  const bool bad = top >= 0x7f800000u;
  const float s = __builtin_fmaxf(__builtin_bit_cast(float, top) / 127.f, 0x1p-126f);
  const float rcp = 1.f / s;
  if (t == 0) reinterpret_cast<float*>(a.scales)[r] = bad ? __builtin_nanf("") : s;
  uint2* out = reinterpret_cast<uint2*>(a.codes + r * a.code_stride);
  if (C > 0) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int64_t c = t + (int64_t)NT * j;
      if (c >= chunks) break;
      int q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = bad ? 0 : row_code(v[j][e], s, rcp);
      out[c] = pack8(q);
    }
  } else {
    for (int64_t c = t; c < chunks; c += NT) {
      load8<DT, VEC>(a.x, off, c, a.cols, v[0]);
      int q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = bad ? 0 : row_code(v[0][e], s, rcp);
      out[c] = pack8(q);
    }
  }
}

// ---- groups with one step, and the copies for the matrix kernels ----------------------------------------
// A thread takes one chunk of 8 columns; 4 neighbouring lanes are a group of 32 (rows hold a multiple
// of 4 chunks and workgroups of 256 threads start on one, so a group never crosses a row or a wave).
// FMT: -1 no codes; OUT: 0 none, 1 a 16-bit copy (max(x, 0) when relu), 2 three bfloat16 planes.
template <int DT, bool VEC, int FMT, int OUT>
__global__ void __launch_bounds__(256) k_encode_groups(const CodeCtx a, int64_t row_chunks, int64_t total) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;  // a multiple of 4: whole groups
  const int64_t r = id / row_chunks, c = id - r * row_chunks;
  float v[8];
  load8<DT, VEC>(a.x, r * a.x_stride, c, a.cols, v);
  constexpr bool RELU = FMT == NC_CODES_RELU;
  if (FMT >= 0) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t m = mag_bits(v[e]);
      top = max(top, RELU && !(v[e] > 0.f) && !(v[e] != v[e]) ? 0u : m);
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    const int sb = step_byte(top, RELU);
    const float inv = __builtin_bit_cast(float, (uint32_t)(254 - (sb < 254 ? sb : 253)) << 23);
    int q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = __builtin_rintf(v[e] * inv);
      if (RELU) {
        const int k = sb == 255 ? 0 : (int)__builtin_fminf(__builtin_fmaxf(t, 0.f), 254.f);
        q[e] = v[e] > 0.f || v[e] != v[e] ? 1 + k : 0;
      } else {
        q[e] = sb == 255 ? 0 : (int)__builtin_fminf(__builtin_fmaxf(t, -127.f), 127.f);
      }
    }
    if (8 * c < a.code_stride) {
      *reinterpret_cast<uint2*>(a.codes + r * a.code_stride + 8 * c) = pack8(q);
      if ((c & 3) == 0) reinterpret_cast<uint8_t*>(a.scales)[r * (a.code_stride / CODE_GROUP) + (c >> 2)] = (uint8_t)sb;
    }
  }
  if (OUT > 0 && 8 * c < a.copy_stride) {
    if (a.relu) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] > 0.f || v[e] != v[e] ? v[e] : 0.f;
    }
    if (OUT == 1) {
      store8<DT == NC_F32 ? NC_BF16 : DT, true>(a.copy, r * a.copy_stride, c, a.copy_stride, v);  // exact: v is of that type
    } else {
      uint16_t p[8][3];
#pragma unroll
      for (int e = 0; e < 8; ++e) split3(v[e], p[e]);
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        uint4 w;
        w.x = p[0][k] | (uint32_t)p[1][k] << 16;
        w.y = p[2][k] | (uint32_t)p[3][k] << 16;
        w.z = p[4][k] | (uint32_t)p[5][k] << 16;
        w.w = p[6][k] | (uint32_t)p[7][k] << 16;
        *reinterpret_cast<uint4*>(a.copy + k * a.plane + r * a.copy_stride + 8 * c) = w;
      }
    }
  }
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(256) k_decode(const CodeCtx a, int64_t row_chunks, int64_t total) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int64_t r = id / row_chunks, c = id - r * row_chunks;
  const uint2 w = *reinterpret_cast<const uint2*>(a.codes + r * a.code_stride + 8 * c);
  float s;
  if (a.format == NC_CODES_ROW) {
    s = reinterpret_cast<const float*>(a.scales)[r];
  } else {
    const uint32_t b = reinterpret_cast<const uint8_t*>(a.scales)[r * (a.code_stride / CODE_GROUP) + (c >> 2)];
    s = b == 255u ? __builtin_nanf("") : __builtin_bit_cast(float, b << 23);
  }
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = ((e < 4 ? w.x : w.y) >> (8 * (e & 3))) & 255u;
    const int q = a.format == NC_CODES_RELU ? (b > 0 ? (int)b - 1 : 0) : (int)(int8_t)b;
    v[e] = (float)q * s;
  }
  store8<DT, VEC>(a.values, r * a.x_stride, c, a.cols, v);
}

// ---- transpose into padded 16-bit rows: 64 x 64 tiles through LDS -------------------------------------
template <int DT>
__global__ void __launch_bounds__(256) k_transpose(const TransposeCtx a) {
  __shared__ float tile[64][65];
  const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int rr = e >> 6, cc = e & 63;
    const int64_t r = r0 + rr, c = c0 + cc;
    float v = 0.f;
    if (r < a.rows && c < a.cols)
      v = DT == NC_F32 ? reinterpret_cast<const float*>(a.src)[r * a.src_stride + c]
                       : elem_f32<DT>(reinterpret_cast<const uint16_t*>(a.src)[r * a.src_stride + c]);
    tile[rr][cc] = v;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int cc = e >> 6, rr = e & 63;
    const int64_t r = r0 + rr, c = c0 + cc;
    if (c >= a.cols) continue;  // r < dst_stride: whole tiles of 64
    uint16_t* d = a.dst + c * a.dst_stride + r;
    if (DT == NC_F32) {
      uint16_t p[3];
      split3(tile[rr][cc], p);
      d[0] = p[0];
      d[a.plane] = p[1];
      d[2 * a.plane] = p[2];
    } else {
      d[0] = f32_elem<DT>(tile[rr][cc]);
    }
  }
}

// ---- sums in a fixed order ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) k_sum_parts(const float* part, int64_t n, int32_t splits, void* out, int32_t dtype) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  float t = 0.f;
  for (int k = 0; k < splits; ++k) t += part[k * n + e];
  if (dtype == NC_F32) reinterpret_cast<float*>(out)[e] = t;
  else reinterpret_cast<uint16_t*>(out)[e] = dtype == NC_BF16 ? f32_elem<NC_BF16>(t) : f32_elem<NC_F16>(t);
}

// 64 columns x 4 row lanes; a slice's rows in four interleaved float sums, then those
template <int DT>
__global__ void __launch_bounds__(256) k_col_sums(const void* x, int64_t rows, int64_t cols, int64_t stride, int64_t per,
                                                  float* part) {
  __shared__ float red[4][64];
  const int cl = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + cl;
  const int64_t rb = (int64_t)blockIdx.y * per, re = rb + per < rows ? rb + per : rows;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < cols) {
    auto at = [&](int64_t r) {
      return DT == NC_F32 ? reinterpret_cast<const float*>(x)[r * stride + c]
                          : elem_f32<DT>(reinterpret_cast<const uint16_t*>(x)[r * stride + c]);
    };
    int64_t r = rb + w;
    for (; r + 12 < re; r += 16) {
#pragma unroll
      for (int u = 0; u < 4; ++u) t[u] += at(r + 4 * u);
    }
    for (; r < re; r += 4) t[0] += at(r);
  }
  red[w][cl] = (t[0] + t[1]) + (t[2] + t[3]);
  __syncthreads();
  if (w == 0 && c < cols) part[blockIdx.y * cols + c] = (red[0][cl] + red[1][cl]) + (red[2][cl] + red[3][cl]);
}

// ---- launchers ---------------------------------------------------------------------------------------
static bool vec_rows(const void* p, int64_t stride, int dtype) {
  const int64_t b = dtype == NC_F32 ? 4 : 2;
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * b) % 16 == 0;
}

template <int DT, bool VEC>
static int encode_rows(const CodeCtx& c, hipStream_t s) {
  const int64_t k = c.code_stride;
  const dim3 waves(blocks_of(c.rows, 4)), rows((unsigned)c.rows);
  if (k <= 512) hipLaunchKernelGGL((k_encode_rows<DT, VEC, 64, 1>), waves, dim3(256), 0, s, c);
  else if (k <= 1024) hipLaunchKernelGGL((k_encode_rows<DT, VEC, 64, 2>), waves, dim3(256), 0, s, c);
  else if (k <= 8192) hipLaunchKernelGGL((k_encode_rows<DT, VEC, 1024, 1>), rows, dim3(1024), 0, s, c);
  else hipLaunchKernelGGL((k_encode_rows<DT, VEC, 1024, 0>), rows, dim3(1024), 0, s, c);
  return (int)hipGetLastError();
}

template <int DT, bool VEC, int FMT>
static int encode_groups(const CodeCtx& c, hipStream_t s) {
  int64_t width = FMT >= 0 ? c.code_stride : 0;
  if (c.copy && c.copy_stride > width) width = c.copy_stride;
  const int64_t rc = width / 8, total = rc * c.rows;
  const dim3 g(blocks_of(total, 256));
  if (!c.copy) {
    if (FMT >= 0) hipLaunchKernelGGL((k_encode_groups<DT, VEC, FMT, 0>), g, dim3(256), 0, s, c, rc, total);
  } else {
    hipLaunchKernelGGL((k_encode_groups<DT, VEC, FMT, DT == NC_F32 ? 2 : 1>), g, dim3(256), 0, s, c, rc, total);
  }
  return (int)hipGetLastError();
}

template <int DT, bool VEC>
static int encode(const CodeCtx& c, hipStream_t s) {
  switch (c.format) {
    case NC_CODES_ROW: return encode_rows<DT, VEC>(c, s);
    case NC_CODES_GROUP: return encode_groups<DT, VEC, NC_CODES_GROUP>(c, s);
    case NC_CODES_RELU: return encode_groups<DT, VEC, NC_CODES_RELU>(c, s);
  }
  return encode_groups<DT, VEC, -1>(c, s);
}

int launch_encode(const CodeCtx& c, hipStream_t s) {
  if (c.rows <= 0) return 0;
  const bool v = vec_rows(c.x, c.x_stride, c.dtype);
  switch (c.dtype) {
    case NC_F32: return v ? encode<NC_F32, true>(c, s) : encode<NC_F32, false>(c, s);
    case NC_F16: return v ? encode<NC_F16, true>(c, s) : encode<NC_F16, false>(c, s);
    case NC_BF16: return v ? encode<NC_BF16, true>(c, s) : encode<NC_BF16, false>(c, s);
  }
  return (int)hipErrorInvalidValue;
}

int launch_decode(const CodeCtx& c, hipStream_t s) {
  if (c.rows <= 0) return 0;
  const bool v = vec_rows(c.values, c.x_stride, c.dtype);
  const int64_t rc = (c.cols + 7) / 8, total = rc * c.rows;
  const dim3 g(blocks_of(total, 256)), b(256);
  switch (c.dtype) {
    case NC_F32:
      if (v) hipLaunchKernelGGL((k_decode<NC_F32, true>), g, b, 0, s, c, rc, total);
      else hipLaunchKernelGGL((k_decode<NC_F32, false>), g, b, 0, s, c, rc, total);
      break;
    case NC_F16:
      if (v) hipLaunchKernelGGL((k_decode<NC_F16, true>), g, b, 0, s, c, rc, total);
      else hipLaunchKernelGGL((k_decode<NC_F16, false>), g, b, 0, s, c, rc, total);
      break;
    case NC_BF16:
      if (v) hipLaunchKernelGGL((k_decode<NC_BF16, true>), g, b, 0, s, c, rc, total);
      else hipLaunchKernelGGL((k_decode<NC_BF16, false>), g, b, 0, s, c, rc, total);
      break;
    default: return (int)hipErrorInvalidValue;
  }
  return (int)hipGetLastError();
}

int launch_transpose(const TransposeCtx& c, hipStream_t s) {
  if (c.rows <= 0 || c.cols <= 0) return 0;
  const dim3 g(blocks_of(c.dst_stride, 64), blocks_of(c.cols, 64));
  switch (c.dtype) {
    case NC_F32: hipLaunchKernelGGL((k_transpose<NC_F32>), g, dim3(256), 0, s, c); break;
    case NC_F16: hipLaunchKernelGGL((k_transpose<NC_F16>), g, dim3(256), 0, s, c); break;
    case NC_BF16: hipLaunchKernelGGL((k_transpose<NC_BF16>), g, dim3(256), 0, s, c); break;
    default: return (int)hipErrorInvalidValue;
  }
  return (int)hipGetLastError();
}

int launch_sum_parts(const float* part, int64_t n, int32_t splits, void* out, int32_t dtype, hipStream_t s) {
  if (n <= 0) return 0;
  hipLaunchKernelGGL(k_sum_parts, dim3(blocks_of(n, 256)), dim3(256), 0, s, part, n, splits, out, dtype);
  return (int)hipGetLastError();
}

int launch_col_sums(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t stride, int32_t slices,
                    float* part, hipStream_t s) {
  if (cols <= 0 || slices <= 0) return 0;
  const int64_t per = (rows + slices - 1) / slices;
  const dim3 g(blocks_of(cols, 64), (unsigned)slices);
  switch (dtype) {
    case NC_F32: hipLaunchKernelGGL((k_col_sums<NC_F32>), g, dim3(256), 0, s, x, rows, cols, stride, per, part); break;
    case NC_F16: hipLaunchKernelGGL((k_col_sums<NC_F16>), g, dim3(256), 0, s, x, rows, cols, stride, per, part); break;
    case NC_BF16: hipLaunchKernelGGL((k_col_sums<NC_BF16>), g, dim3(256), 0, s, x, rows, cols, stride, per, part); break;
    default: return (int)hipErrorInvalidValue;
  }
  return (int)hipGetLastError();
}

}  // namespace nc
