// nc_lowbit.hip — codes of the 8-bit layer operators and the copies that their matrix kernels read.
//
// Everything here is one pass over its input and bound by memory: a thread takes 8 neighbouring
// columns (16 or 32 bytes in, 8 bytes of codes out).  Measured: rows of 16384 x 4096 bfloat16 to codes 42 us (4.8
// TB/s), codes to values 31 us (6.5, the codes in the cache); groups of 100000 x 256 float 19 us (6.8, most of it in
// the cache); the copy with codes of 8192 x 4096 bfloat16 28 us.
#include "nc_lowbit.h"

#include <type_traits>

namespace nc {

static inline unsigned blocks_of(int64_t n, int b) { return (unsigned)((n + b - 1) / b); }

template <int DT>
__device__ __forceinline__ void store8(void* x, int64_t off, int64_t c, int64_t cols, const float (&v)[8]) {
  if (DT == NC_F32) {
    float* p = reinterpret_cast<float*>(x) + off + 8 * c;
    if (8 * c + 8 <= cols) {
      store_any(p, float4{v[0], v[1], v[2], v[3]});
      store_any(p + 4, float4{v[4], v[5], v[6], v[7]});
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
    if (8 * c + 8 <= cols) {
      store_any(p, uint4{e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                         e[6] | (uint32_t)e[7] << 16});
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (8 * c + j < cols) p[j] = e[j];
    }
  }
}

// ---- rows with one scale ---------------------------------------------------------------------------
// Rows of up to 512 columns: LPR lanes (16, 32 or 64) own a row, R rows each, all loads first.
template <int DT, bool VEC, int LPR, int R>
__global__ void __launch_bounds__(256) k_encode_short_rows(const CodeCtx a) {
  const int c = threadIdx.x % LPR;
  const int64_t r0 = ((int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR) * R, chunks = a.code_stride / 8;
  float v[R][8];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int64_t r = r0 + j < a.rows ? r0 + j : a.rows - 1;
    load8<DT, VEC>(a.x, r * a.x_stride, c, a.cols, v[j]);
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    uint32_t top = 0;
    clear8<VEC>(c, a.cols, v[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, mag_bits(v[j][e]));
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    const bool bad = top >= 0x7f800000u;
    const float s = row_scale(top);
    const uint2 w = row_codes(v[j], bad, s, 1.f / s);
    if (r0 + j >= a.rows) continue;
    if (c == 0) reinterpret_cast<float*>(a.scales)[r0 + j] = bad ? __builtin_nanf("") : s;
    if (c < chunks) reinterpret_cast<uint2*>(a.codes + (r0 + j) * a.code_stride)[c] = w;
  }
}

// NT threads (64, 256 or 1024) own a row; C > 0: its 8-column chunks t, t + NT, ... stay in registers
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
      load8<DT, VEC>(a.x, off, c, a.cols, v[j]);
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
      clear8<VEC>(t + (int64_t)NT * j, a.cols, v[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, mag_bits(v[j][e]));
    }
  } else {
    for (int64_t c = t; 8 * c < a.cols; c += NT) {
      load8<DT, VEC>(a.x, off, c, a.cols, v[0]);
      clear8<VEC>(c, a.cols, v[0]);
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
  const float s = row_scale(top);
  const float rcp = 1.f / s;
  if (t == 0) reinterpret_cast<float*>(a.scales)[r] = bad ? __builtin_nanf("") : s;
  uint2* out = reinterpret_cast<uint2*>(a.codes + r * a.code_stride);
  if (C > 0) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int64_t c = t + (int64_t)NT * j;
      if (c >= chunks) break;
      out[c] = row_codes(v[j], bad, s, rcp);
    }
  } else {
    for (int64_t c = t; c < chunks; c += NT) {
      load8<DT, VEC>(a.x, off, c, a.cols, v[0]);
      clear8<VEC>(c, a.cols, v[0]);
      out[c] = row_codes(v[0], bad, s, rcp);
    }
  }
}

// ---- groups with one step, and the copies for the matrix kernels ----------------------------------------
// A thread takes one chunk of 8 columns; 4 neighbouring lanes are a group of 32 (rows hold a multiple
// of 4 chunks and workgroups of 256 threads start on one, so a group never crosses a row or a wave).
// FMT: -1 no codes; COPY: a 16-bit copy (max(x, 0) when relu).
template <int DT, bool VEC, int FMT, bool COPY>
__global__ void __launch_bounds__(256) k_encode_groups(const CodeCtx a, int64_t row_chunks, int64_t total) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;  // a multiple of 4: whole groups
  const int64_t r = id / row_chunks, c = id - r * row_chunks;
  float v[8];
  load8<DT, VEC>(a.x, r * a.x_stride, c, a.cols, v);
  clear8<VEC>(c, a.cols, v);
  constexpr bool RELU = FMT == NC_CODES_RELU;
  if (RELU || a.relu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = relu_keep_nan(v[e]);
  }
  if (FMT >= 0) {
    int sb;
    const uint2 w = group_codes<RELU>(v, sb);
    if (8 * c < a.code_stride) {
      *reinterpret_cast<uint2*>(a.codes + r * a.code_stride + 8 * c) = w;
      if ((c & 3) == 0) reinterpret_cast<uint8_t*>(a.scales)[r * (a.code_stride / CODE_GROUP) + (c >> 2)] = (uint8_t)sb;
    }
  }
  if (COPY && 8 * c < a.copy_stride) store8<DT>(a.copy, r * a.copy_stride, c, a.copy_stride, v);  // exact: v is of that type
}

template <int DT>
__global__ void __launch_bounds__(256) k_decode(const CodeCtx a, int64_t row_chunks, int64_t total) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int64_t r = id / row_chunks, c = id - r * row_chunks;
  if (r >= a.rows) {
    const float zero[8] = {};
    store8<DT>(a.values, r * a.x_stride, c, a.cols, zero);
    return;
  }
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
    // as half, the one group code beyond its largest number ends there (nc_lowbit.h)
    if (DT == NC_F16 && a.format != NC_CODES_ROW && __builtin_fabsf(v[e]) == 65536.f) v[e] = __builtin_copysignf(65504.f, v[e]);
  }
  store8<DT>(a.values, r * a.x_stride, c, a.cols, v);
}

// ---- float matrices in two half planes --------------------------------------------------------------------
// a wave a row, read twice (the second time from the cache)
template <bool VEC>
__global__ void __launch_bounds__(256) k_split(const SplitCtx a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= a.rows) return;
  const int64_t off = r * a.x_stride;
  uint32_t top = 0;
  for (int64_t c = lane; 8 * c < a.cols; c += 64) {
    float v[8];
    load8<NC_F32, VEC>(a.x, off, c, a.cols, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, mag_bits(v[e]));  // (columns behind the last are copies)
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  const int e = top_exponent<0>(top);
  if (lane == 0) a.exponent[r] = e;
  for (int64_t c = lane; 8 * c < a.dst_stride; c += 64) {
    float v[8];
    load8<NC_F32, VEC>(a.x, off, c, a.cols, v);
    clear8<VEC>(c, a.cols, v);
    uint4 p[2];
    split2<0>(v, scale_to(141, e), p);
    if (top >= 0x7f800000u) split2_infinite(v, p);
#pragma unroll
    for (int k = 0; k < 2; ++k) *reinterpret_cast<uint4*>(a.dst + k * a.plane + r * a.dst_stride + 8 * c) = p[k];
  }
}

// the largest magnitude of each column in every TOP_ROWS rows: 64 columns a workgroup, a quarter of the rows a wave
__global__ void __launch_bounds__(256) k_tops(const TransposeCtx a) {
  __shared__ uint32_t red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane, cc = c < a.cols ? c : a.cols - 1;
  const int64_t r0 = (int64_t)blockIdx.y * TOP_ROWS + wave * (TOP_ROWS / 4);
  const float* x = reinterpret_cast<const float*>(a.src) + cc;
  uint32_t top = 0;
  for (int k = 0; k < TOP_ROWS / 4; k += 16) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = x[(r0 + k + j < a.rows ? r0 + k + j : a.rows - 1) * a.src_stride];
#pragma unroll
    for (int j = 0; j < 16; ++j) top = max(top, mag_bits(v[j]));
  }
  red[wave][lane] = top;
  __syncthreads();
  if (wave == 0 && c < a.cols) a.tops[blockIdx.y * a.cols + c] = max(max(red[0][lane], red[1][lane]), max(red[2][lane], red[3][lane]));
}

// ---- transpose into padded 16-bit rows: 64 x 64 tiles through LDS -------------------------------------
// A lane loads 16 bytes of its row and writes them down a column of the tile:
// a wave's 64 lanes are a column's 64 elements, side by side in LDS.  Then 8 lanes write a row of the
// result, 16 bytes each (float: to each plane).  4096 x 4096 bfloat16 12 us (5.6 TB/s); 31 with 2 bytes a lane.
template <int DT>
__global__ void __launch_bounds__(256) k_transpose(const TransposeCtx a) {
  using E = typename std::conditional<DT == NC_F32, float, uint16_t>::type;
  constexpr int EC = 16 / sizeof(E), CH = 64 / EC / 4;  // elements a chunk, chunks a thread
  __shared__ __attribute__((aligned(16))) E tile[64][64 + EC];
  const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool in = r0 + lane < a.rows;
  const E* src = reinterpret_cast<const E*>(a.src) + (in ? r0 + lane : a.rows - 1) * a.src_stride;
  E v[CH][EC];
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int64_t c = c0 + EC * (wave + 4 * j);
    if (c + EC <= a.cols) {  // (a wave's lanes all)
      const uint4 w = load_any<uint4>(src + c);
      __builtin_memcpy(v[j], &w, 16);
    } else {
#pragma unroll
      for (int e = 0; e < EC; ++e) v[j][e] = src[c + e < a.cols ? c + e : a.cols - 1];
    }
  }
#pragma unroll
  for (int j = 0; j < CH; ++j)
#pragma unroll
    for (int e = 0; e < EC; ++e) tile[EC * (wave + 4 * j) + e][lane] = in ? v[j][e] : E(0);
  __shared__ uint32_t red[4][64];
  if (DT == NC_F32) {  // the columns' exponents
    const int64_t c = c0 + lane < a.cols ? c0 + lane : a.cols - 1, parts = (a.rows + TOP_ROWS - 1) / TOP_ROWS;
    uint32_t top = 0;
    for (int64_t k = wave; k < parts; k += 4) top = max(top, a.tops[k * a.cols + c]);
    red[wave][lane] = top;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int at = j * 256 + threadIdx.x, cc = at >> 3, r8 = 8 * (at & 7);
    if (c0 + cc >= a.cols) continue;  // r0 + r8 < dst_stride: whole tiles of 64
    uint16_t* d = a.dst + (c0 + cc) * a.dst_stride + r0 + r8;
    if constexpr (DT == NC_F32) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = tile[cc][r8 + e];
      const uint32_t top = max(max(red[0][cc], red[1][cc]), max(red[2][cc], red[3][cc]));
      const int e = top_exponent<0>(top);
      if (r0 + r8 == 0) a.exponent[c0 + cc] = e;
      uint4 p[2];
      split2<0>(x, scale_to(141, e), p);
      if (top >= 0x7f800000u) split2_infinite(x, p);
#pragma unroll
      for (int k = 0; k < 2; ++k) *reinterpret_cast<uint4*>(d + k * a.plane) = p[k];
    } else {
      *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(&tile[cc][r8]);
    }
  }
}

// ---- sums in a fixed order ---------------------------------------------------------------------------
// 4 neighbouring elements a thread.  The 128 parts of 220000 x 256 x 256 take 9 us; one load at a time, 25 more.
template <int DT>
__global__ void __launch_bounds__(256) k_sum_parts(const SumParts a, unsigned first_blocks) {
  const int w = blockIdx.x >= first_blocks ? 1 : 0;
  const int64_t n = a.n[w], last = n > 4 ? n - 4 : 0;
  int64_t e = ((int64_t)(blockIdx.x - (w ? first_blocks : 0)) * 256 + threadIdx.x) * 4;
  if (e >= n) return;
  const float* p = a.part[w];
  if (n < 4) {  // the last 4 are written twice where n is no multiple; fewer go one by one
    for (; e < n; ++e) {
      float t = 0.f;
      for (int k = 0; k < a.parts[w]; ++k) t += p[k * n + e];
      if (DT == NC_F32) reinterpret_cast<float*>(a.out[w])[e] = t;
      else reinterpret_cast<uint16_t*>(a.out[w])[e] = f32_elem<DT>(t);
    }
    return;
  }
  e = e < last ? e : last;
  p += e;
  floatx4 t = zero4();
  int k = a.parts[w];
  for (; k >= 8; k -= 8, p += 8 * n) {  // 8 loads in flight, added in order
    floatx4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = load_any<floatx4>(p + j * n);
#pragma unroll
    for (int j = 0; j < 8; ++j) t += v[j];
  }
  for (; k > 0; --k, p += n) t += load_any<floatx4>(p);
  if (DT == NC_F32) {
    store_any(reinterpret_cast<float*>(a.out[w]) + e, t);
  } else {
    const uint16_t o[4] = {f32_elem<DT>(t[0]), f32_elem<DT>(t[1]), f32_elem<DT>(t[2]), f32_elem<DT>(t[3])};
    store_any(reinterpret_cast<uint16_t*>(a.out[w]) + e, uint2{o[0] | (uint32_t)o[1] << 16, o[2] | (uint32_t)o[3] << 16});
  }
}

// ---- launchers ---------------------------------------------------------------------------------------
template <int DT, bool VEC>
static int encode_rows(const CodeCtx& c, hipStream_t s) {
  // A wave a row needs no barrier (16384 x 4096 bfloat16: 49 us; 79 us with 1024 threads a row); few rows get
  // 256 threads each for a shorter way through a row.  Short rows go several to a wave, so that enough
  // loads are in flight.
  const int64_t k = c.code_stride;
  const bool few = c.rows < 512;
  const dim3 waves(blocks_of(c.rows, 4)), rows((unsigned)c.rows), b(256);
  if (k <= 128) {
    if (few) hipLaunchKernelGGL((k_encode_short_rows<DT, VEC, 16, 1>), dim3(blocks_of(c.rows, 16)), b, 0, s, c);
    else hipLaunchKernelGGL((k_encode_short_rows<DT, VEC, 16, 4>), dim3(blocks_of(c.rows, 64)), b, 0, s, c);
  } else if (k <= 256) {
    if (few) hipLaunchKernelGGL((k_encode_short_rows<DT, VEC, 32, 1>), dim3(blocks_of(c.rows, 8)), b, 0, s, c);
    else hipLaunchKernelGGL((k_encode_short_rows<DT, VEC, 32, 4>), dim3(blocks_of(c.rows, 32)), b, 0, s, c);
  } else if (k <= 512) {
    if (few) hipLaunchKernelGGL((k_encode_short_rows<DT, VEC, 64, 1>), dim3(blocks_of(c.rows, 4)), b, 0, s, c);
    else hipLaunchKernelGGL((k_encode_short_rows<DT, VEC, 64, 4>), dim3(blocks_of(c.rows, 16)), b, 0, s, c);
  }
  else if (k <= 1024 && !few) hipLaunchKernelGGL((k_encode_rows<DT, VEC, 64, 2>), waves, dim3(256), 0, s, c);
  else if (k <= 2048 && few) hipLaunchKernelGGL((k_encode_rows<DT, VEC, 256, 1>), rows, dim3(256), 0, s, c);
  else if (k <= 2048) hipLaunchKernelGGL((k_encode_rows<DT, VEC, 64, 4>), waves, dim3(256), 0, s, c);
  else if (k <= 4096 && !few) hipLaunchKernelGGL((k_encode_rows<DT, VEC, 64, 8>), waves, dim3(256), 0, s, c);
  else if (k <= 8192) hipLaunchKernelGGL((k_encode_rows<DT, VEC, 256, 4>), rows, dim3(256), 0, s, c);
  else hipLaunchKernelGGL((k_encode_rows<DT, VEC, 1024, 0>), rows, dim3(1024), 0, s, c);
  return (int)hipGetLastError();
}

template <int DT, bool VEC, int FMT>
static int encode_groups(const CodeCtx& c, hipStream_t s) {
  int64_t width = FMT >= 0 ? c.code_stride : 0;
  if (c.copy && c.copy_stride > width) width = c.copy_stride;
  const int64_t rc = width / 8, total = rc * c.rows;
  const dim3 g(blocks_of(total, 256));
  if (c.copy) {
    if constexpr (DT == NC_F32) return (int)hipErrorInvalidValue;  // float inputs are read as they are
    else hipLaunchKernelGGL((k_encode_groups<DT, VEC, FMT, true>), g, dim3(256), 0, s, c, rc, total);
  } else {
    if constexpr (FMT < 0) return (int)hipErrorInvalidValue;
    else hipLaunchKernelGGL((k_encode_groups<DT, VEC, FMT, false>), g, dim3(256), 0, s, c, rc, total);
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
  const bool v = wide8(c.cols);
  switch (c.dtype) {
    case NC_F32: return v ? encode<NC_F32, true>(c, s) : encode<NC_F32, false>(c, s);
    case NC_F16: return v ? encode<NC_F16, true>(c, s) : encode<NC_F16, false>(c, s);
    case NC_BF16: return v ? encode<NC_BF16, true>(c, s) : encode<NC_BF16, false>(c, s);
  }
  return (int)hipErrorInvalidValue;
}

int launch_decode(const CodeCtx& c, hipStream_t s) {
  if (c.rows <= 0) return 0;
  const int64_t rc = (c.cols + 7) / 8, total = rc * (c.rows + c.zero_rows);
  const dim3 g(blocks_of(total, 256)), b(256);
  switch (c.dtype) {
    case NC_F32: hipLaunchKernelGGL(k_decode<NC_F32>, g, b, 0, s, c, rc, total); break;
    case NC_F16: hipLaunchKernelGGL(k_decode<NC_F16>, g, b, 0, s, c, rc, total); break;
    case NC_BF16: hipLaunchKernelGGL(k_decode<NC_BF16>, g, b, 0, s, c, rc, total); break;
    default: return (int)hipErrorInvalidValue;
  }
  return (int)hipGetLastError();
}

int launch_split(const SplitCtx& c, hipStream_t s) {
  if (c.rows <= 0 || c.cols <= 0) return 0;
  if (wide8(c.cols)) hipLaunchKernelGGL((k_split<true>), dim3(blocks_of(c.rows, 4)), dim3(256), 0, s, c);
  else hipLaunchKernelGGL((k_split<false>), dim3(blocks_of(c.rows, 4)), dim3(256), 0, s, c);
  return (int)hipGetLastError();
}

template <int DT>
static int transpose(const TransposeCtx& c, hipStream_t s) {
  if (DT == NC_F32) hipLaunchKernelGGL(k_tops, dim3(blocks_of(c.cols, 64), blocks_of(c.rows, TOP_ROWS)), dim3(256), 0, s, c);
  const dim3 g(blocks_of(c.dst_stride, 64), blocks_of(c.cols, 64));
  hipLaunchKernelGGL(k_transpose<DT>, g, dim3(256), 0, s, c);
  return (int)hipGetLastError();
}

int launch_transpose(const TransposeCtx& c, hipStream_t s) {
  if (c.rows <= 0 || c.cols <= 0) return 0;
  switch (c.dtype) {
    case NC_F32: return transpose<NC_F32>(c, s);
    case NC_F16: return transpose<NC_F16>(c, s);
    case NC_BF16: return transpose<NC_BF16>(c, s);
  }
  return (int)hipErrorInvalidValue;
}

template <int DT>
static int sum_parts(const SumParts& a, hipStream_t s) {
  const unsigned first = blocks_of(a.out[0] ? a.n[0] : 0, 1024), all = first + blocks_of(a.out[1] ? a.n[1] : 0, 1024);
  if (all == 0) return 0;
  hipLaunchKernelGGL(k_sum_parts<DT>, dim3(all), dim3(256), 0, s, a, first);
  return (int)hipGetLastError();
}

int launch_sum_parts(const SumParts& a, int32_t dtype, hipStream_t s) {
  switch (dtype) {
    case NC_F32: return sum_parts<NC_F32>(a, s);
    case NC_F16: return sum_parts<NC_F16>(a, s);
    case NC_BF16: return sum_parts<NC_BF16>(a, s);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace nc
