// nc_lowgemm.hip — the matrix products of the 8-bit layer operators on the gfx950 matrix cores.
//
// k_low_gemm    C[m][n] = sum_k A[m][k] B[n][k]: int8 codes (v_mfma_i32_16x16x64_i8, exact sums) or
//               16-bit elements (v_mfma_f32_16x16x32_bf16 / _f16, float sums).  A float product is six
//               products of bfloat16 planes (split3: x = x0 + x1 + x2): x0 y0 + x0 y1 + x1 y0 + x0 y2 +
//               x1 y1 + x2 y0; what is left out is below 2^-25 of |x y|.
// k_low_wgrad   dW[n][k] = sum_m dY[m][n] V[m][k], V the values of an 8-bit checkpoint, decoded while a
//               tile is staged (a code times a power of two is exact in 16 bits), both operands
//               read transposed from LDS (ds_read_b64_tr_b16).
#include "nc_lowbit.h"

namespace nc {

#define NC_GLOBAL(p) ((const __attribute__((address_space(1))) void*)(p))
#define NC_LDS(p) ((__attribute__((address_space(3))) void*)(p))

// every matrix result is read by vector instructions next: wait states for the longest of the
// instructions used here (see mfma16_drain in nc_device.h for the shortest count that held)
__device__ __forceinline__ void matrix_drain() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// loads into LDS are counted as memory loads of the wave that issued them: each wave waits for its
// own before the barrier
__device__ __forceinline__ void staged_barrier() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// workgroups to tiles: those that the hardware deals to one chiplet (w mod 8) take a run of
// neighbouring tiles, so that the operands of the run are shared in that chiplet's L2
__device__ __forceinline__ int64_t chiplet_order(int64_t w, int64_t n) {
  const int64_t x = w & 7, k = w >> 3, base = n >> 3, more = n & 7;
  return x * base + (x < more ? x : more) + k;
}

constexpr int SLICE = 128;  // bytes of a row staged at a time
// LDS tile: rows of 128 bytes, 16-byte chunk c of row r at c ^ ((r >> 1) & 7): the 16 lanes that
// ds_read_b128 serves together then touch 16 distinct 16-byte slots of the 64 banks
__device__ __forceinline__ int swz(int row, int chunk) { return chunk ^ ((row >> 1) & 7); }

template <int MODE>
struct Mac;
template <>
struct Mac<LOW_I8> {
  typedef intx4 Acc;
  static __device__ __forceinline__ Acc zero() { return intx4{0, 0, 0, 0}; }
  static __device__ __forceinline__ Acc mac(uint4 a, uint4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(intx4, a), __builtin_bit_cast(intx4, b), c, 0, 0, 0);
  }
};
template <>
struct Mac<LOW_BF16> {
  typedef floatx4 Acc;
  static __device__ __forceinline__ Acc zero() { return zero4(); }
  static __device__ __forceinline__ Acc mac(uint4 a, uint4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mac<LOW_F16> {
  typedef floatx4 Acc;
  static __device__ __forceinline__ Acc zero() { return zero4(); }
  static __device__ __forceinline__ Acc mac(uint4 a, uint4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  }
};

__device__ __forceinline__ float load_bias(const void* b, int dtype, int64_t n) {
  if (dtype == NC_F32) return reinterpret_cast<const float*>(b)[n];
  const uint16_t e = reinterpret_cast<const uint16_t*>(b)[n];
  return dtype == NC_BF16 ? elem_f32<NC_BF16>(e) : elem_f32<NC_F16>(e);
}

// 4 neighbouring outputs [m][n .. n + 3]
__device__ __forceinline__ void store4(const LowGemm& g, int64_t m, int64_t n, const float (&v)[4]) {
  const bool whole = n + 4 <= g.N;
  if (g.out_dtype == NC_F32) {
    float* p = reinterpret_cast<float*>(g.out) + m * g.ldc + n;
    if (whole && (reinterpret_cast<uintptr_t>(p) & 15) == 0) *reinterpret_cast<float4*>(p) = float4{v[0], v[1], v[2], v[3]};
    else
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < g.N) p[j] = v[j];
  } else {
    uint16_t* p = reinterpret_cast<uint16_t*>(g.out) + m * g.ldc + n;
    uint16_t e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = g.out_dtype == NC_BF16 ? f32_elem<NC_BF16>(v[j]) : f32_elem<NC_F16>(v[j]);
    if (whole && (reinterpret_cast<uintptr_t>(p) & 7) == 0)
      *reinterpret_cast<uint2*>(p) = uint2{e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16};
    else
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < g.N) p[j] = e[j];
  }
}

// BM x BN tile, WM x WN waves, each (BM / WM) x (BN / WN) in blocks of 16 x 16.  The instruction
// takes B's rows as its first operand: lane (i, q) then holds, for row m = i of the block, the four
// neighbouring columns n = 4 q + 0..3.
template <int MODE, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) k_low_gemm(const LowGemm g, int64_t mt, int64_t nt) {
  constexpr int W = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int STAGE = (BM + BN) * SLICE;
  constexpr int LA = BM / 8 / W, LB = BN / 8 / W;  // 8-row loads a wave
  static_assert(BM % (8 * W) == 0 && BN % (8 * W) == 0, "whole loads a wave");
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, q = lane >> 4;
  const int64_t tile = chiplet_order(blockIdx.x, mt * nt);
  const int64_t tm = tile / nt, tn = tile - tm * nt;
  const int64_t m0 = tm * BM, n0 = tn * BN;
  // staging: lane l of a load puts chunk position l & 7 of row l >> 3
  uint32_t oa[LA], ob[LB];
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int r = (wave * LA + j) * 8 + (lane >> 3);
    const int64_t rr = m0 + r < g.M ? r : g.M - 1 - m0;  // rows behind the last: its copies, not stored
    oa[j] = (uint32_t)(rr * g.lda) + 16 * swz(r, lane & 7);
  }
#pragma unroll
  for (int j = 0; j < LB; ++j) {
    const int r = (wave * LB + j) * 8 + (lane >> 3);
    const int64_t rr = n0 + r < g.N ? r : g.N - 1 - n0;
    ob[j] = (uint32_t)(rr * g.ldb) + 16 * swz(r, lane & 7);
  }
  const uint8_t* A = g.A + m0 * g.lda;
  const uint8_t* B = g.B + n0 * g.ldb;
  const int total = g.slices * g.segments;
  auto stage = [&](int t) {
    unsigned char* s = lds + (t & 1) * STAGE;
    int sl = t, seg = 0;
    while (sl >= g.slices) { sl -= g.slices; ++seg; }
    // plane pairs, the largest product last: (2,0) (1,1) (0,2) (1,0) (0,1) (0,0)
    const int pa = g.segments > 1 ? (0x001012 >> (4 * seg)) & 3 : 0;
    const int pb = g.segments > 1 ? (0x010210 >> (4 * seg)) & 3 : 0;
    const uint8_t* a = A + pa * g.plane_a + (int64_t)sl * SLICE;
    const uint8_t* b = B + pb * g.plane_b + (int64_t)sl * SLICE;
#pragma unroll
    for (int j = 0; j < LA; ++j)
      __builtin_amdgcn_global_load_lds(NC_GLOBAL(a + oa[j]), NC_LDS(s + (wave * LA + j) * 1024), 16, 0, 0);
#pragma unroll
    for (int j = 0; j < LB; ++j)
      __builtin_amdgcn_global_load_lds(NC_GLOBAL(b + ob[j]), NC_LDS(s + BM * SLICE + (wave * LB + j) * 1024), 16, 0, 0);
  };
  typename Mac<MODE>::Acc acc[FM][FN];
#pragma unroll
  for (int u = 0; u < FM; ++u)
#pragma unroll
    for (int v = 0; v < FN; ++v) acc[u][v] = Mac<MODE>::zero();
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
  const int c0 = 16 * swz(i, q), c1 = 16 * swz(i, 4 + q);  // wm, wn and 16 u leave the swizzle as it is
  stage(0);
  for (int t = 0; t < total; ++t) {
    staged_barrier();  // slice t is in LDS, slice t - 1 is used up
    if (t + 1 < total) stage(t + 1);
    const unsigned char* As = lds + (t & 1) * STAGE;
    const unsigned char* Bs = As + BM * SLICE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 a[FM], b[FN];
#pragma unroll
      for (int u = 0; u < FM; ++u) a[u] = *reinterpret_cast<const uint4*>(As + (wm + 16 * u + i) * SLICE + (h ? c1 : c0));
#pragma unroll
      for (int v = 0; v < FN; ++v) b[v] = *reinterpret_cast<const uint4*>(Bs + (wn + 16 * v + i) * SLICE + (h ? c1 : c0));
#pragma unroll
      for (int u = 0; u < FM; ++u)
#pragma unroll
        for (int v = 0; v < FN; ++v) acc[u][v] = Mac<MODE>::mac(b[v], a[u], acc[u][v]);
    }
  }
  matrix_drain();
#pragma unroll
  for (int u = 0; u < FM; ++u) {
    const int64_t m = m0 + wm + 16 * u + i;
    if (m >= g.M) continue;
    const float rs = MODE == LOW_I8 ? g.row_scale[m] : 1.f;
#pragma unroll
    for (int v = 0; v < FN; ++v) {
      const int64_t n = n0 + wn + 16 * v + 4 * q;
      if (n >= g.N) continue;
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = n + j < g.N;
        float x = (float)acc[u][v][j];
        if (MODE == LOW_I8) x = x * (rs * (in ? g.col_scale[n + j] : 0.f));
        if (g.bias && in) x += load_bias(g.bias, g.bias_dtype, n + j);
        if (g.relu) x = x > 0.f || x != x ? x : 0.f;
        if (g.mask && in && g.mask[m * g.ldm + n + j] == 0) x = 0.f;
        o[j] = x;
      }
      store4(g, m, n, o);
    }
  }
}

template <int MODE, int BM, int BN, int WM, int WN>
static int run_low_gemm(const LowGemm& g, hipStream_t s) {
  const int64_t mt = (g.M + BM - 1) / BM, nt = (g.N + BN - 1) / BN;
  constexpr int lds = 2 * (BM + BN) * SLICE;
  hipLaunchKernelGGL((k_low_gemm<MODE, BM, BN, WM, WN>), dim3((unsigned)(mt * nt)), dim3(64 * WM * WN), lds, s, g, mt, nt);
  return (int)hipGetLastError();
}

int launch_low_gemm(const LowGemm& g, hipStream_t s) {
  if (g.M <= 0 || g.N <= 0) return 0;
  switch (g.mode) {
    case LOW_I8: return run_low_gemm<LOW_I8, 128, 128, 2, 2>(g, s);
    case LOW_BF16: return run_low_gemm<LOW_BF16, 128, 128, 2, 2>(g, s);
    case LOW_F16: return run_low_gemm<LOW_F16, 128, 128, 2, 2>(g, s);
  }
  return (int)hipErrorInvalidValue;
}

// ---- weight gradient -----------------------------------------------------------------------------------
// A workgroup sums its rows [rb, re) of dY and codes into a BN x BK tile of dW.  A stage is MS rows of
// both operands in LDS as 16-bit elements, row-major (the sum's index m is the row).  ds_read_b64_tr_b16
// hands lane (i, q) four rows of column i: rows 4 q + 0..3 of a 4-row x 16-column block, so two of them
// make the 8 sum indices of a lane's operand: m = 4 q + e and 16 + 4 q + e, the same for both operands.
// Rows of BN (BK) elements are cut into 32-byte units; unit u of row m lies at u ^ (m & 7): the 8 rows
// that 32 lanes read together then cover all 64 banks.
__device__ const uint4 g_zero_row[2] = {};  // what rows behind the last one read

__device__ __forceinline__ shortx4 tr_read(const unsigned char* p) {
  typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)p);
}

// 16 codes of one row and group -> 16 elements of 16 bits; step is a power of two: exact
template <bool F16, bool RELU>
__device__ __forceinline__ void decode16(uint4 c, float step, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t o[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = RELU ? w[j] : w[j] ^ 0x80808080u;  // signed codes as code + 128
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = (float)((b >> (8 * e)) & 255u);
      v[e] = RELU ? __builtin_fmaxf(__builtin_fmaf(f, step, -step), 0.f) : __builtin_fmaf(f, step, -128.f * step);
      if (step != step) v[e] = step;  // a NaN group (fmax would drop it)
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (F16) {
        o[2 * j + e] = f32_elem<NC_F16>(v[2 * e]) | (uint32_t)f32_elem<NC_F16>(v[2 * e + 1]) << 16;
      } else {  // exact in bfloat16: the upper halves
        o[2 * j + e] = __builtin_bit_cast(uint32_t, v[2 * e]) >> 16 | (__builtin_bit_cast(uint32_t, v[2 * e + 1]) & 0xffff0000u);
      }
    }
  }
  lo = uint4{o[0], o[1], o[2], o[3]};
  hi = uint4{o[4], o[5], o[6], o[7]};
}

template <int NP, bool F16, bool RELU, int BN, int BK, int MS, int WN, int WK>
__global__ void __launch_bounds__(64 * WN * WK) k_low_wgrad(const LowWgrad g) {
  constexpr int W = WN * WK, T = 64 * W;
  constexpr int FN = BN / WN / 16, FK = BK / WK / 16;
  constexpr int YROW = 2 * BN, XROW = 2 * BK;               // bytes of a staged row
  constexpr int YSTAGE = MS * YROW, XSTAGE = MS * XROW, STAGE = NP * YSTAGE + XSTAGE;
  constexpr int YL = NP * YSTAGE / 1024 / W;                // 1-KB loads a wave
  constexpr int XL = MS * BK / 16 / T;                      // 16-code loads a thread
  static_assert(NP * YSTAGE % (1024 * W) == 0 && MS * BK % (16 * T) == 0 && YL > 0 && XL > 0, "whole loads");
  static_assert(BN >= 128 && BK >= 128, "rows of at least 8 units of 32 bytes");
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q = lane >> 4, j16 = lane & 15;
  const int64_t n0 = (int64_t)blockIdx.x * BN, k0 = (int64_t)blockIdx.y * BK;
  const int64_t rb = (int64_t)blockIdx.z * g.rows_per;
  const int64_t re = rb + g.rows_per < g.M ? rb + g.rows_per : g.M;
  const int64_t ychunks = (g.N + 7) / 8, xchunks = g.code_stride / 16, steps_row = g.code_stride / CODE_GROUP;
  const int total = (int)((re - rb + MS - 1) / MS);

  auto stage_y = [&](int t) {
    unsigned char* s = lds + (t & 1) * STAGE;
#pragma unroll
    for (int l = 0; l < YL; ++l) {
      const int at = (wave * YL + l) * 64 + lane;  // 16-byte position in the planes' tiles
      const int p = at / (YSTAGE / 16), in = at % (YSTAGE / 16);
      const int row = in / (YROW / 16), pos = in % (YROW / 16);
      int64_t c = n0 / 8 + (pos ^ ((row & 7) << 1));
      c = c < ychunks ? c : ychunks - 1;  // columns behind the last: not stored
      const int64_t m = rb + (int64_t)t * MS + row;
      const void* src = m < re ? (const void*)(g.dy + p * g.plane + m * g.ldy + 8 * c) : (const void*)g_zero_row;
      __builtin_amdgcn_global_load_lds(NC_GLOBAL(src), NC_LDS(s + (wave * YL + l) * 1024), 16, 0, 0);
    }
  };
  uint4 xc[XL];
  uint32_t xs[XL];
  auto load_x = [&](int t) {
#pragma unroll
    for (int l = 0; l < XL; ++l) {
      const int at = l * T + threadIdx.x, row = at / (BK / 16);
      int64_t c = k0 / 16 + at % (BK / 16);
      c = c < xchunks ? c : xchunks - 1;
      const int64_t m = rb + (int64_t)t * MS + row;
      if (m < re) {
        xc[l] = *reinterpret_cast<const uint4*>(g.codes + m * g.code_stride + 16 * c);
        xs[l] = g.steps[m * steps_row + (c >> 1)];
      } else {
        xc[l] = uint4{0u, 0u, 0u, 0u};
        xs[l] = 1u;
      }
    }
  };
  auto store_x = [&](int t) {
    unsigned char* s = lds + (t & 1) * STAGE + NP * YSTAGE;
#pragma unroll
    for (int l = 0; l < XL; ++l) {
      const int at = l * T + threadIdx.x, row = at / (BK / 16), u = at % (BK / 16);
      const float step = xs[l] == 255u ? __builtin_nanf("") : __builtin_bit_cast(float, xs[l] << 23);
      uint4 lo, hi;
      decode16<F16, RELU>(xc[l], step, lo, hi);
      uint4* d = reinterpret_cast<uint4*>(s + row * XROW + 32 * (u ^ (row & 7)));
      d[0] = lo;
      d[1] = hi;
    }
  };

  floatx4 acc[FN][FK];
#pragma unroll
  for (int u = 0; u < FN; ++u)
#pragma unroll
    for (int v = 0; v < FK; ++v) acc[u][v] = zero4();
  const int wn = (wave / WK) * (BN / WN), wk = (wave % WK) * (BK / WK);
  const int tr = 4 * q + (j16 >> 2), tc = 8 * (j16 & 3);  // row and byte in the 32-byte unit of a lane's transposed read
  if (total > 0) {
    stage_y(0);
    load_x(0);
    store_x(0);
  }
  for (int t = 0; t < total; ++t) {
    staged_barrier();
    if (t + 1 < total) {
      stage_y(t + 1);
      load_x(t + 1);
    }
    const unsigned char* Y = lds + (t & 1) * STAGE;
    const unsigned char* X = Y + NP * YSTAGE;
#pragma unroll
    for (int ms = 0; ms < MS; ms += 32) {
      uint4 b[FK];
#pragma unroll
      for (int v = 0; v < FK; ++v) {
        const unsigned char* p = X + (ms + tr) * XROW + 32 * ((wk / 16 + v) ^ (tr & 7)) + tc;
        const shortx4 x0 = tr_read(p), x1 = tr_read(p + 16 * XROW);
        b[v] = uint4{__builtin_bit_cast(uint2, x0).x, __builtin_bit_cast(uint2, x0).y, __builtin_bit_cast(uint2, x1).x,
                     __builtin_bit_cast(uint2, x1).y};
      }
#pragma unroll
      for (int pl = NP - 1; pl >= 0; --pl) {
#pragma unroll
        for (int u = 0; u < FN; ++u) {
          const unsigned char* p = Y + pl * YSTAGE + (ms + tr) * YROW + 32 * ((wn / 16 + u) ^ (tr & 7)) + tc;
          const shortx4 y0 = tr_read(p), y1 = tr_read(p + 16 * YROW);
          const uint4 a = uint4{__builtin_bit_cast(uint2, y0).x, __builtin_bit_cast(uint2, y0).y,
                                __builtin_bit_cast(uint2, y1).x, __builtin_bit_cast(uint2, y1).y};
#pragma unroll
          for (int v = 0; v < FK; ++v) acc[u][v] = Mac<F16 ? LOW_F16 : LOW_BF16>::mac(b[v], a, acc[u][v]);
        }
      }
    }
    if (t + 1 < total) store_x(t + 1);  // the other half of LDS: last read before this pass's barrier
  }
  matrix_drain();
  float* part = g.part + (int64_t)blockIdx.z * g.N * g.K;
  const int i = j16;
#pragma unroll
  for (int u = 0; u < FN; ++u) {
    const int64_t n = n0 + wn + 16 * u + i;
    if (n >= g.N) continue;
#pragma unroll
    for (int v = 0; v < FK; ++v) {
      const int64_t k = k0 + wk + 16 * v + 4 * q;
      float* p = part + n * g.K + k;
      if (k + 4 <= g.K && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        *reinterpret_cast<floatx4*>(p) = acc[u][v];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < g.K) p[e] = acc[u][v][e];
      }
    }
  }
}

constexpr int WG_N = 128, WG_K = 128;

void low_wgrad_splits(int64_t M, int64_t N, int64_t K, int32_t& splits, int64_t& rows_per) {
  const int64_t tiles = ((N + WG_N - 1) / WG_N) * ((K + WG_K - 1) / WG_K);
  int64_t want = (512 + tiles - 1) / tiles, most = (M + 255) / 256;
  if (want > most) want = most;
  if (want < 1) want = 1;
  rows_per = round_up((M + want - 1) / want, 64);
  if (rows_per < 64) rows_per = 64;
  splits = (int32_t)((M + rows_per - 1) / rows_per);
  if (splits < 1) splits = 1;
}

template <int NP, bool F16, bool RELU>
static int run_low_wgrad(const LowWgrad& g, hipStream_t s) {
  constexpr int MS = NP == 3 ? 32 : 64;
  constexpr int lds = 2 * (NP * MS * 2 * WG_N + MS * 2 * WG_K);
  const dim3 grid((unsigned)((g.N + WG_N - 1) / WG_N), (unsigned)((g.K + WG_K - 1) / WG_K), (unsigned)g.splits);
  hipLaunchKernelGGL((k_low_wgrad<NP, F16, RELU, WG_N, WG_K, MS, 2, 2>), grid, dim3(256), lds, s, g);
  return (int)hipGetLastError();
}

int launch_low_wgrad(const LowWgrad& g, hipStream_t s) {
  if (g.N <= 0 || g.K <= 0) return 0;
  if (g.planes == 3) return g.relu ? run_low_wgrad<3, false, true>(g, s) : run_low_wgrad<3, false, false>(g, s);
  if (g.f16) return g.relu ? run_low_wgrad<1, true, true>(g, s) : run_low_wgrad<1, true, false>(g, s);
  return g.relu ? run_low_wgrad<1, false, true>(g, s) : run_low_wgrad<1, false, false>(g, s);
}

}  // namespace nc
