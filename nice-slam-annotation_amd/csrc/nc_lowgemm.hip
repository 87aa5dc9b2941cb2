// nc_lowgemm.hip — the matrix products of the 8-bit layer operators on the gfx950 matrix cores.
//
// k_low_gemm    C[m][n] = sum_k A[m][k] B[n][k]: int8 codes (v_mfma_i32_16x16x64_i8, exact sums) or
//               16-bit elements (v_mfma_f32_16x16x32_bf16 / _f16, float sums).
// k_low_gemm_f  the same for float A: three products of half planes with scales (split2).  A is split while it is
//               staged, and its 8-bit checkpoint written besides.
// k_low_small   the int8 product of few rows or short sums, x encoded within it.
// k_low_wgrad   dW[n][k] = sum_m dY[m][n] V[m][k], V the values of an 8-bit checkpoint, decoded while a
//               tile is staged or written out before (a code times a power of two is exact in 16 bits), both
//               operands read transposed from LDS (ds_read_b64_tr_b16); db[n] = sum_m dY[m][n] beside it.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "nc_lowbit.h"

namespace nc {

// every matrix result is read by vector instructions next: wait states for the longest of the
// instructions used here (see mfma16_drain in nc_device.h for the shortest count that held)
__device__ __forceinline__ void matrix_drain() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// 16 bytes a lane from base + offset into LDS at `to` + 16 lane (wave-uniform).  Written as an
// instruction of its own because the compiler, which cannot tell the two halves of the double buffer
// apart, would wait for every such load before the next LDS read; it has no result register, and
// the kernels wait for it (vmcnt) before the barrier after which its bytes are read.
__device__ __forceinline__ void load_lds16(const void* base, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void load_lds4(const void* base, uint32_t offset, uint32_t to) {  // 4 bytes a lane
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(offset), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// waits until at most N of the wave's vector memory loads are in flight
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void staged_barrier() {
  wait_loads<0>();
  __syncthreads();
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// a barrier for LDS alone: __syncthreads() would also wait for every store in flight
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
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
  typedef int Elem;
  static __device__ __forceinline__ Acc zero() { return intx4{0, 0, 0, 0}; }
  static __device__ __forceinline__ Acc mac(uint4 a, uint4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(intx4, a), __builtin_bit_cast(intx4, b), c, 0, 0, 0);
  }
};
template <>
struct Mac<LOW_BF16> {
  typedef floatx4 Acc;
  typedef float Elem;
  static __device__ __forceinline__ Acc zero() { return zero4(); }
  static __device__ __forceinline__ Acc mac(uint4 a, uint4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mac<LOW_F16> {
  typedef floatx4 Acc;
  typedef float Elem;
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

// 4 neighbouring outputs [m][n .. n + 3], one store where all are there
template <int DT>
__device__ __forceinline__ void store4(const LowGemm& g, int64_t m, int64_t n, const float (&v)[4]) {
  if (DT == NC_F32) {
    float* p = reinterpret_cast<float*>(g.out) + m * g.ldc + n;
    if (n + 4 <= g.N) {
      store_any(p, float4{v[0], v[1], v[2], v[3]});
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < g.N) p[j] = v[j];
    }
  } else {
    uint16_t* p = reinterpret_cast<uint16_t*>(g.out) + m * g.ldc + n;
    uint16_t e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = f32_elem<DT>(v[j]);
    if (n + 4 <= g.N) {
      store_any(p, uint2{e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16});
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < g.N) p[j] = e[j];
    }
  }
}
// a row's or channel's scale = mantissa 2^exponent.  The mantissas' product is a normal number also where that of the
// scales is subnormal or infinite, so y is rounded as often as with scales near 1.
struct Scale {
  float mantissa;
  int exponent;
};
__device__ __forceinline__ Scale split_scale(float s) { return {__builtin_amdgcn_frexp_mantf(s), __builtin_amdgcn_frexp_expf(s)}; }
__device__ __forceinline__ Scale operator*(Scale a, Scale b) { return {a.mantissa * b.mantissa, a.exponent + b.exponent}; }
// from 2^-60 to 2^60: the product of two is a normal number itself
__device__ __forceinline__ bool near_scale(float s) { return s >= 0x1p-60f && s <= 0x1p60f; }

// one column's result of a sum
template <int MODE, bool NEAR = false>
__device__ __forceinline__ float finish(const LowGemm& g, float x, Scale scale, float bias, uint32_t code) {
  if (MODE == LOW_I8) x = x * scale.mantissa;
  if (MODE == LOW_I8 && !NEAR) x = __builtin_ldexpf(x, scale.exponent);
  if (g.bias) x += bias;
  if (g.relu) x = relu_keep_nan(x);
  if (MODE != LOW_I8 && code == 0) x = 0.f;
  return x;
}

// A wave's FM x FN blocks of sums at [m0][n0]: 16 rows at a time through its own piece of LDS (cw,
// 16 (64 FN + 16) bytes), so that they leave in whole lines.  Everything that the epilogue reads is read
// first: a store counts as a memory access in flight like a load, so a load behind stores waits for
// them.  Rows and columns behind the last read the last's.
template <int MODE, int DT, int FM, int FN, typename Acc>
__device__ __forceinline__ void store_tile(const LowGemm& g, unsigned char* cw, int lane, const Acc (&acc)[FM][FN], int64_t m0,
                                           int64_t n0) {
  constexpr int CROW = 64 * FN + 16;               // bytes of a row, padded
  constexpr int LPR = 4 * FN, RPI = 64 / LPR;      // lanes a row, rows at once
  const int i = lane & 15, q = lane >> 4;
  const int64_t n = n0 + 4 * (lane % LPR);
  float* part = g.splits > 1 ? g.part + (int64_t)blockIdx.y * g.M * g.N : nullptr;
  float cs[4], cb[4];
  float rs[MODE == LOW_I8 ? FM : 1][16 / RPI];
  uint32_t mask[FM][16 / RPI];
  bool near = true;
  if (!part) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t nn = n + j < g.N ? n + j : g.N - 1;
      cs[j] = MODE == LOW_I8 ? g.col_scale[nn] : 1.f;
      cb[j] = g.bias ? load_bias(g.bias, g.bias_dtype, nn) : 0.f;
    }
    if (MODE == LOW_I8) {
      near = near_scale(g.col_scale[n0 + lane % (16 * FN) < g.N ? n0 + lane % (16 * FN) : g.N - 1]);
#pragma unroll
      for (int r = 0; r < 16 * FM; r += 64) near &= near_scale(g.row_scale[m0 + r + lane < g.M ? m0 + r + lane : g.M - 1]);
    }
#pragma unroll
    for (int u = 0; u < FM; ++u)
#pragma unroll
      for (int k = 0; k < 16 / RPI; ++k) {
        const int64_t m = m0 + 16 * u + k * RPI + lane / LPR, mm = m < g.M ? m : g.M - 1;
        if (MODE == LOW_I8) rs[u][k] = g.row_scale[mm];
        else mask[u][k] = g.mask ? *reinterpret_cast<const uint32_t*>(g.mask + mm * g.ldm + (n < g.ldm ? n : 0)) : ~0u;
      }
  }
  // the plain product of the scales takes two instructions less for an output (500000 x 256 x 256 coded: 144.5 us, 146.9)
  auto rows = [&](auto kind) {
    constexpr bool NEAR = decltype(kind)::value;
#pragma unroll
    for (int u = 0; u < FM; ++u) {
#pragma unroll
      for (int v = 0; v < FN; ++v) *reinterpret_cast<Acc*>(cw + i * CROW + 64 * v + 16 * q) = acc[u][v];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int k = 0; k < 16 / RPI; ++k) {
        const int row = k * RPI + lane / LPR;
        const int64_t m = m0 + 16 * u + row;
        const Acc c = *reinterpret_cast<const Acc*>(cw + row * CROW + 16 * (lane % LPR));
        if (m >= g.M || n >= g.N) continue;
        if (part) {
          float* p = part + m * g.N + n;
          if (n + 4 <= g.N) {
            store_any(p, c);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (n + j < g.N) reinterpret_cast<typename Mac<MODE>::Elem*>(p)[j] = c[j];
          }
        } else {
          float o[4];
          const float r = MODE == LOW_I8 ? rs[u][k] : 1.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const Scale sc = NEAR ? Scale{r * cs[j], 0} : split_scale(r) * split_scale(cs[j]);
            o[j] = finish<MODE, NEAR>(g, (float)c[j], sc, cb[j], (mask[u][k] >> (8 * j)) & 255u);
          }
          store4<DT>(g, m, n, o);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  };
  if (MODE != LOW_I8 || __all(near)) rows(std::true_type{});
  else rows(std::false_type{});
}

// the parts of a cut sum, in order, and the epilogue: 4 neighbouring columns a thread
template <int MODE, int DT>
__global__ void __launch_bounds__(256) k_low_finish(const LowGemm g, int64_t quads) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= g.M * quads) return;
  const int64_t m = id / quads, n = 4 * (id - m * quads);
  float o[4], cb[4];
  Scale cs[4];
  const Scale rs = split_scale(MODE == LOW_I8 ? g.row_scale[m] : 1.f);
  const uint32_t mask = MODE != LOW_I8 && g.mask ? *reinterpret_cast<const uint32_t*>(g.mask + m * g.ldm + n) : ~0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t nn = n + j < g.N ? n + j : g.N - 1;
    cs[j] = split_scale(MODE == LOW_I8 ? g.col_scale[nn] : 1.f) * rs;
    cb[j] = g.bias ? load_bias(g.bias, g.bias_dtype, nn) : 0.f;
  }
  typedef Mac<MODE == LOW_I8 ? LOW_I8 : LOW_BF16> M;
  typedef typename M::Acc Acc;
  Acc t = M::zero();
  const float* p = g.part + m * g.N + n;
  const bool whole = n + 4 <= g.N;
  auto part = [&](int k) {
    const typename M::Elem* e = reinterpret_cast<const typename M::Elem*>(p + k * (g.M * g.N));
    if (whole) return load_any<Acc>(e);
    Acc v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = e[n + j < g.N ? j : 0];  // columns behind the last: not stored
    return v;
  };
  int k = 0;
  for (; k + 4 <= g.splits; k += 4) {  // 4 loads in flight, added in order
    const Acc a = part(k), b = part(k + 1), c = part(k + 2), d = part(k + 3);
    t += a;
    t += b;
    t += c;
    t += d;
  }
  for (; k < g.splits; ++k) t += part(k);
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = finish<MODE>(g, (float)t[j], cs[j], cb[j], (mask >> (8 * j)) & 255u);
  store4<DT>(g, m, n, o);
}

// BM x BN tile, WM x WN waves, each (BM / WM) x (BN / WN) in blocks of 16 x 16.  The instruction
// takes B's rows as its first operand: lane (i, q) then holds, for row m = i of the block, the four
// neighbouring columns n = 4 q + 0..3.
// A slice is worked off in phases of 4 x FN blocks; while a phase multiplies, the next one's operands
// are read from LDS.  Before the last phase a barrier says that the slice is read and the next one
// has arrived; the slice after that goes into the freed half then, a whole slice ahead of its use.
// Measured, M x K x N: int8 16384 x 4096 x 4096 232 - 241 us = 2.3 POP/s (a library's int8 product on this card: 2.47),
// bfloat16 8192 x 4096 x 4096 205 - 217 us = 1.3 PFLOP/s (1.57).  The matrix cores are busy 55 - 62 % of the cycles at the 2.0 - 2.2
// GHz that their power leaves.  4 waves of 128 x 128 read a third less from LDS, but a wave alone on its SIMD waits
// for every read: int8 392 us.  Half slices (64 bytes of a row) five deep: 255 us; memory prefers whole lines.
template <int MODE, int DT, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) k_low_gemm(const LowGemm g, int64_t mt, int64_t nt) {
  constexpr int W = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int STAGE = (BM + BN) * SLICE;
  constexpr int LA = BM / 8 / W, LB = BN / 8 / W;  // 8-row loads a wave
  constexpr int NG = FM / 4, PH = 2 * NG;          // phases of a slice
  constexpr int CROW = 64 * FN + 16;               // bytes of a row of the epilogue's block, padded
  static_assert(BM % (8 * W) == 0 && BN % (8 * W) == 0 && FM % 4 == 0, "whole loads a wave, whole phases");
  static_assert(W * 16 * CROW <= 2 * STAGE, "the epilogue's blocks fit the buffers");
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
  const int first = (int)((int64_t)g.slices * blockIdx.y / g.splits);  // this part's slices
  const int total = (int)((int64_t)g.slices * (blockIdx.y + 1) / g.splits) - first;
  const uint32_t lds0 = lds_address(lds);
  const uint8_t* a_next = A + (int64_t)first * SLICE;  // of the next stage() call
  const uint8_t* b_next = B + (int64_t)first * SLICE;
  auto stage = [&](int half) {
    const uint8_t* a = a_next;
    const uint8_t* b = b_next;
    a_next += SLICE;
    b_next += SLICE;
    const uint32_t s = lds0 + half * STAGE;
#pragma unroll
    for (int j = 0; j < LA; ++j) load_lds16(a, oa[j], s + (wave * LA + j) * 1024);
#pragma unroll
    for (int j = 0; j < LB; ++j) load_lds16(b, ob[j], s + BM * SLICE + (wave * LB + j) * 1024);
  };
  typename Mac<MODE>::Acc acc[FM][FN];
#pragma unroll
  for (int u = 0; u < FM; ++u)
#pragma unroll
    for (int v = 0; v < FN; ++v) acc[u][v] = Mac<MODE>::zero();
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
  // wm, wn and 16 u leave the swizzle as it is
  const unsigned char* fa = lds + (wm + i) * SLICE + 16 * swz(i, q);
  const unsigned char* fb = lds + BM * SLICE + (wn + i) * SLICE + 16 * swz(i, q);
  const int other = 16 * swz(i, 4 + q) - 16 * swz(i, q);  // to the slice's second half
  uint4 a[2][4], b[2][FN];
  auto read = [&](int half, int p) {  // phase p's operands of the slice in `half`
    const int h = p / NG, gr = p % NG;
    const unsigned char* pa = fa + half * STAGE + (h ? other : 0) + gr * 64 * SLICE;
#pragma unroll
    for (int u = 0; u < 4; ++u) a[p & 1][u] = *reinterpret_cast<const uint4*>(pa + 16 * u * SLICE);
    if (gr == 0) {
      const unsigned char* pb = fb + half * STAGE + (h ? other : 0);
#pragma unroll
      for (int v = 0; v < FN; ++v) b[h][v] = *reinterpret_cast<const uint4*>(pb + 16 * v * SLICE);
    }
  };
  stage(0);
  if (total > 1) {
    stage(1);
    wait_loads<LA + LB>();
  } else {
    wait_loads<0>();
  }
  __syncthreads();
  read(0, 0);
  auto multiply = [&](int p) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int v = 0; v < FN; ++v) {
        auto& c = acc[(p % NG) * 4 + u][v];
        c = Mac<MODE>::mac(b[p / NG][v], a[p & 1][u], c);
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int t = 0; t + 1 < total; ++t) {
#pragma unroll
    for (int p = 0; p < PH; ++p) {
      if (p + 1 < PH) {
        read(t & 1, p + 1);
      } else {
        staged_barrier();
        if (t + 2 < total) stage(t & 1);
        read((t + 1) & 1, 0);
      }
      multiply(p);
    }
  }
#pragma unroll
  for (int p = 0; p < PH; ++p) {  // the last slice
    if (p + 1 < PH) read((total - 1) & 1, p + 1);
    multiply(p);
  }
  matrix_drain();
  __syncthreads();  // the last slice is read: its memory takes the results
  store_tile<MODE, DT, FM, FN>(g, lds + wave * 16 * CROW, lane, acc, m0 + wm, n0 + wn);
}

// ---- float A ------------------------------------------------------------------------------------------
// The same pipeline over slices of 32 columns, as three products of half planes: x = (x0 + x1) / scale
// (split2), C = x0 y0 + x0 y1 + x1 y0.  B's scale is a power of two of its row, A's one of its row so far: it puts
// the first 32 columns' largest below 2^12 and stays until one reaches 2^15, when the row's sums are scaled
// down with it (seldom after the first slices).  Both are undone in the epilogue.  A's x1 is held times 2^11 and
// multiplied by y0 2^-11, made of y0 as it arrives: a half has no digits below 2^-24, and x1 would lose its own there.
// A value of A keeps 22 bits down to 2^-25 of the largest before it in its row (its floor is 2^-47 of that), one of B
// down to 2^-17 of the largest in its row (2^-38); the product left out is below 2^-22: 2^-20.4 of |x y| at most, about
// 2^-23 on average.  Off the exact result by 1.9e-7 at 200 x 93 x 256 (a plain float product: 2.9e-7), 3.6e-7 at
// 2048 x 1024 x 4096 (1.1e-6); 2000 x 256 x 256 with one input of 10^6 beside those of 1: 1.9e-7 (x1 without its 2^11
// 6e-6, a plain product 2.9e-7; the 2^11 cost 2 - 3 % of a product).  Six products of exact bfloat16 planes, 2.5e-7 and
// 5.1e-7 there for the longer chain of sums, are twice the work for matrix cores that are bound by their
// power: 4096 x 4096 x 4096 740 us on a card where these took 385, before the 2^11.
// Planes lie in LDS as rows of 64 bytes, 16-byte chunk c of row r at c ^ F((r >> 2) & 3), F = (0, 2, 3, 1):
// conflict-free for ds_read_b128 (the third weight plane's layout of nc_device.h).  A's floats go into a piece of
// LDS of their own, where each lane finds the 8 columns that it asked for; it reads them, asks for those two
// slices on, splits them and writes the planes.  B's planes have room for three slices and are asked for three
// ahead (two, and A's floats with them half a slice before their use: 409 us).  4 neighbouring lanes hold a
// group of 32 columns, so the workgroups of the first column tile write the checkpoint's codes in passing.
// A slice goes block by block of 16 rows: its 3 FN products while the next one's planes are read; the last block's
// products take turns with the reads of the next slice's B.
// A layer's sums are short (8 slices for 256 inputs), so a workgroup goes through its tiles as one stream of
// slices: the next tile's first slices are on their way while a tile ends, and its results leave from
// registers and are not waited for.
// An infinity of A or B has the planes 0 and infinity (split2_infinite): products with it alone.
// RELU: of max(A, 0); MASK: the output is masked by codes and has no bias (each would take 16 registers).
// Measured, M x K x N: 220000 x 256 x 256 148 us (450 MB: 91 us at a copy's rate; all workgroups store at once, and
// loads behind stores wait for them), 4096 x 4096 x 4096 464 - 473 us = 0.88 PFLOP/s of plane products.
constexpr int A_UP = 11;  // bits of a half: x1 2^11 is as large as x0
template <int BM, int BN, int WM, int WN, bool VEC, bool RELU, bool MASK>
__global__ void __launch_bounds__(64 * WM * WN) k_low_gemm_f(const LowGemm g, int32_t tiles, int32_t nt) {
  constexpr int W = WM * WN, T = 64 * W, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int APL = BM * 64, BPL = BN * 64;      // bytes of a plane's slice
  constexpr int B0 = 4 * APL;                      // two slices of A's planes, then three of B's
  constexpr int XA = BM * 4 / T;                   // chunks of A a thread
  constexpr int LA = XA * (VEC ? 2 : 8);           // loads of A a wave
  constexpr int LB = 2 * BPL / 1024 / W;           // 1-KB loads of B a wave
  constexpr int RAW = B0 + 6 * BPL, EXPS = RAW + W * XA * 2048;  // A's floats, then its exponents [2][BM]
  static_assert(BM * 4 % T == 0 && 2 * BPL % (1024 * W) == 0, "whole chunks a thread, whole loads a wave");
  static_assert(FM % 2 == 0 && FN % 2 == 0, "pairs");
  extern __shared__ __attribute__((aligned(256))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, q = lane >> 4;
  const int first = (int)((int64_t)g.slices * blockIdx.y / g.splits);
  const int total = (int)((int64_t)g.slices * (blockIdx.y + 1) / g.splits) - first;
  const int mine = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  const int steps = mine * total;
  const uint32_t lds0 = lds_address(lds);
  unsigned char* raw = lds + RAW + wave * (XA * 2048);  // this wave's floats
  int32_t* const exps = reinterpret_cast<int32_t*>(lds + EXPS);
  const int pads = (int)(g.code_stride / CODE_GROUP) - g.slices;  // code groups behind the last slice
  auto tile_at = [&](int k, int64_t& m0, int64_t& n0) {
    const uint32_t t = (uint32_t)chiplet_order(blockIdx.x + k * gridDim.x, tiles), tm = t / (uint32_t)nt;
    m0 = (int64_t)tm * BM;
    n0 = (int64_t)(t - tm * (uint32_t)nt) * BN;
  };

  // what is loaded next, tile and slice: A's floats run two slices ahead, B's planes three
  int ak = 0, as = 0, bk = 0, bs = 0;
  int64_t am0 = 0, an0 = 0;
  uint32_t oa[XA], ob[LB];
  const uint8_t* a_next = nullptr;
  const uint8_t* b_next = nullptr;
  auto enter_a = [&]() {
    tile_at(ak, am0, an0);
#pragma unroll
    for (int l = 0; l < XA; ++l) {
      const int r = (l * T + (int)threadIdx.x) >> 2;
      const int64_t rr = am0 + r < g.M ? r : g.M - 1 - am0;  // rows behind the last: its copies, not stored
      oa[l] = (uint32_t)(rr * g.lda);
    }
    a_next = g.A + am0 * g.lda;
    if (g.codes && an0 == 0 && first == 0) {
      for (int e = threadIdx.x; e < BM * pads; e += T) {
        const int64_t m = am0 + e / pads, gr = g.slices + e % pads;
        if (m >= g.M) break;
        uint4* c = reinterpret_cast<uint4*>(g.codes + m * g.code_stride + gr * CODE_GROUP);
        c[0] = c[1] = uint4{0u, 0u, 0u, 0u};
        g.steps[m * (g.code_stride / CODE_GROUP) + gr] = 1;
      }
    }
  };
  auto enter_b = [&]() {
    int64_t m0, n0;
    tile_at(bk, m0, n0);
#pragma unroll
    for (int j = 0; j < LB; ++j) {
      const int at = (wave * LB + j) * 16 + (lane >> 2), r = at % BN;  // a row of a plane
      const int64_t rr = n0 + r < g.N ? r : g.N - 1 - n0;
      ob[j] = (uint32_t)(rr * g.ldb) + hchunk3(r, lane & 3);
    }
    b_next = g.B + n0 * g.ldb + (int64_t)first * 64;
  };
  // what the floats in LDS are: tile and slice, and whether their codes are written
  int64_t xm0 = 0;
  int xt = 0;
  bool xcode = false, xnew = false;  // xnew: a tile's first slice
  int xe[XA];                        // the exponents that the rows' scales are made of
  auto load_a = [&]() {
    xnew = as == 0;
    xm0 = am0;
    xt = first + as;
    xcode = g.codes && an0 == 0;
    const uint32_t to = lds0 + RAW + wave * (XA * 2048);
#pragma unroll
    for (int l = 0; l < XA; ++l) {
      const int c = 8 * (4 * xt + (int)(threadIdx.x & 3)), k = (int)g.K;
      if (VEC) {
        const uint32_t at = oa[l] + 4 * (uint32_t)(c < k - 8 ? c : k - 8);  // the last chunk: the row's last 8, moved and cleared later
        load_lds16(a_next, at, to + l * 2048);
        load_lds16(a_next, at + 16, to + l * 2048 + 1024);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          load_lds4(a_next, oa[l] + 4 * (uint32_t)(c + e < k ? c + e : k - 1), to + l * 2048 + e * 256);
      }
    }
    if (++as == total) {
      as = 0;
      if (++ak < mine) enter_a();
    }
  };
  auto load_b = [&](int third) {
#pragma unroll
    for (int j = 0; j < LB; ++j) {
      const int pl = (wave * LB + j) * 16 / BN;
      load_lds16(b_next + pl * g.plane_b, ob[j], lds0 + B0 + third * (2 * BPL) + (wave * LB + j) * 1024);
    }
    b_next += 64;
    if (++bs == total) {
      bs = 0;
      if (++bk < mine) enter_b();
    }
  };
  float xs[XA][8];
  auto fetch_a = [&]() {
#pragma unroll
    for (int l = 0; l < XA; ++l) {
      float(&x)[8] = xs[l];
      if (VEC) {
        const float4 lo = *reinterpret_cast<const float4*>(raw + l * 2048 + 16 * lane);
        const float4 hi = *reinterpret_cast<const float4*>(raw + l * 2048 + 1024 + 16 * lane);
        x[0] = lo.x; x[1] = lo.y; x[2] = lo.z; x[3] = lo.w;
        x[4] = hi.x; x[5] = hi.y; x[6] = hi.z; x[7] = hi.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = *reinterpret_cast<const float*>(raw + l * 2048 + e * 256 + 4 * lane);
      }
    }
  };
  // more: the floats after next are asked for as soon as these are read
  auto store_a = [&](int half, bool more) {
    unsigned char* s = lds + half * (2 * APL);
    wait_lds();
    const int64_t m0 = xm0;
    const int t = xt;
    const bool code = xcode, fresh_row = xnew;
    xcode = false;  // a step behind the last one stores the same planes again, which nobody reads
    if (more) load_a();
#pragma unroll
    for (int l = 0; l < XA; ++l) {
      const int at = l * T + threadIdx.x, r = at >> 2, c = at & 3;
      float(&x)[8] = xs[l];
      if ((t + 1) * 32 > (int)g.K) clear8<VEC>((int64_t)t * 4 + c, g.K, x);
      if (RELU)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = relu_keep_nan(x[e]);
      if (code) {
        int sb;
        const uint2 w = group_codes<RELU>(x, sb);
        if (m0 + r < g.M) {
          *reinterpret_cast<uint2*>(g.codes + m0 * g.code_stride + (uint32_t)(r * (int)g.code_stride + 32 * t + 8 * c)) = w;
          const int sr = (int)(g.code_stride / CODE_GROUP);
          if (c == 0) (g.steps + m0 * sr)[(uint32_t)(r * sr + t)] = (uint8_t)sb;
        }
      }
      float top = 0.f;  // (NaN counts as nothing: it is one in the planes)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = __builtin_fmaxf(top, __builtin_fabsf(x[e]));
      uint32_t bits = __builtin_bit_cast(uint32_t, top);
      bits = max(bits, (uint32_t)__builtin_amdgcn_mov_dpp((int)bits, 0xb1, 0xf, 0xf, true));  // lane ^ 1
      bits = max(bits, (uint32_t)__builtin_amdgcn_mov_dpp((int)bits, 0x4e, 0xf, 0xf, true));  // lane ^ 2
      const int e = top_exponent<A_UP>(bits);
      xe[l] = fresh_row || e > xe[l] + 3 ? e : xe[l];
      if (c == 0) exps[half * BM + r] = xe[l];
      uint4 p[2];
      split2<A_UP>(x, scale_to(138, xe[l]), p);
      if (__any(bits == 0x7f800000u)) split2_infinite(x, p);
#pragma unroll
      for (int k = 0; k < 2; ++k) *reinterpret_cast<uint4*>(s + k * APL + r * 64 + hchunk3(r, c)) = p[k];
    }
  };
  floatx4 acc[FM][FN];
#pragma unroll
  for (int u = 0; u < FM; ++u)
#pragma unroll
    for (int v = 0; v < FN; ++v) acc[u][v] = zero4();
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
  const unsigned char* fa = lds + (wm + i) * 64 + hchunk3(i, q);  // wm, wn and 16 u leave the chunk order as it is
  const unsigned char* fb = lds + B0 + (wn + i) * 64 + hchunk3(i, q);
  uint4 a[2][2], b[2][FN];  // a[block & 1][plane], b[plane][block]
  uint4 down[FN];           // b[0] 2^-A_UP
  int ea[FM], next_ea[FM];  // exponents of the sums, of the next slice's rows
  bool fresh = true;        // the sums are zero
  auto read_a = [&](int half, int u) {
#pragma unroll
    for (int p = 0; p < 2; ++p) a[u & 1][p] = *reinterpret_cast<const uint4*>(fa + half * (2 * APL) + p * APL + 16 * u * 64);
  };
  auto read_b = [&](int third, int v) {
#pragma unroll
    for (int p = 0; p < 2; ++p) b[p][v] = *reinterpret_cast<const uint4*>(fb + third * (2 * BPL) + p * BPL + 16 * v * 64);
  };
  auto read_exps = [&](int half) {
#pragma unroll
    for (int u = 0; u < FM; ++u) next_ea[u] = exps[half * BM + wm + 16 * u + i];
  };
  auto rescale = [&]() {  // the sums in the units of the slice to come
    bool differ = false;
#pragma unroll
    for (int u = 0; u < FM; ++u) differ = differ || ea[u] != next_ea[u];
    if (!fresh && __any(differ)) {
      matrix_drain();
#pragma unroll
      for (int u = 0; u < FM; ++u)
#pragma unroll
        for (int v = 0; v < FN; ++v)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[u][v][j] = __builtin_ldexpf(acc[u][v][j], ea[u] - next_ea[u]);
      matrix_drain();
    }
#pragma unroll
    for (int u = 0; u < FM; ++u) ea[u] = next_ea[u];
    fresh = false;
  };
  auto multiply = [&](int u, int v0) {  // blocks (u, v0) and (u, v0 + 1); the smallest products first
    __builtin_amdgcn_sched_barrier(0);
    if (u == 0)
#pragma unroll
      for (int v = v0; v < v0 + 2; ++v)
        down[v] = __builtin_bit_cast(uint4, __builtin_bit_cast(half8, b[0][v]) * (_Float16)(1.f / (1 << A_UP)));
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int v = v0; v < v0 + 2; ++v) {
        const int p = u == 0 ? (k + 1) % 3 : k;
        acc[u][v] = Mac<LOW_F16>::mac(p == 0 ? down[v] : b[p == 1][v], a[u & 1][p == 0], acc[u][v]);
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  enter_a();
  enter_b();
  load_a();
  load_b(0);
  if (steps > 1) {
    load_b(1);
    wait_loads<LB>();
  } else {
    wait_loads<0>();
  }
  fetch_a();
  store_a(0, steps > 1);
  if (steps > 2) load_b(2);
  lds_barrier();
  read_a(0, 0);
#pragma unroll
  for (int v = 0; v < FN; ++v) read_b(0, v);
  read_exps(0);
  float* const to = g.splits > 1 ? g.part + (int64_t)blockIdx.y * g.M * g.N : reinterpret_cast<float*>(g.out);
  const int64_t ldo = g.splits > 1 ? g.N : g.ldc;
  const bool biased = g.bias && g.splits == 1;
  constexpr int RESULTS = FM * FN;  // stores of a whole tile's results
  int s = 0;
  bool left = false;  // RESULTS stores were issued after the loads that the next slice waits for: they stay in flight
  int third = 0;  // of B, where this slice's was
  auto slice = [&](auto arrived) {
    const int h = s & 1, next = third == 2 ? 0 : third + 1;
    rescale();
#pragma unroll
    for (int u = 0; u + 1 < FM; ++u) {
      read_a(h, u + 1);
      const bool split = u == (FM > 2 ? 1 : 0);
      if (split) {
        // the next slice's floats, and with them its B, which was asked for before; behind them only the B after
        // next and a tile's results are in flight
        if (s + 2 >= steps) wait_loads<0>();
        else if (left) wait_loads<LB + RESULTS>();
        else wait_loads<LB>();
        left = false;
        fetch_a();
      }
#pragma unroll
      for (int v = 0; v < FN; v += 2) multiply(u, v);
      if (split) {
        arrived();
        store_a(h ^ 1, s + 2 < steps);
      }
    }
    lds_barrier();
    if (s + 3 < steps) load_b(third);
    read_a(h ^ 1, 0);
#pragma unroll
    for (int v = 0; v < FN; v += 2) {
      multiply(FM - 1, v);
      read_b(next, v);
      read_b(next, v + 1);
    }
    read_exps(h ^ 1);
    third = next;
    ++s;
  };
  for (int k = 0; k < mine; ++k) {
    for (int n = 1; n < total; ++n) slice([] {});
    int64_t m0, n0;
    tile_at(k, m0, n0);
    float cb[FN][4];  // what the results need, a slice ahead; without a branch (what a branch loads is waited for at its end)
    int ec[FN][4];
    uint32_t mask[FM][FN];
    int ln = lane;
    asm volatile("" : "+v"(ln));  // computed here: kept, it would take registers that the products need
    const int row = wm + (ln & 15), col = wn + 4 * (ln >> 4);
    const float* bias = reinterpret_cast<const float*>(biased ? g.bias : g.exponent);
#pragma unroll
    for (int v = 0; v < FN; ++v)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = (int)n0 + col + 16 * v + j, n = c < (int)g.N ? c : (int)g.N - 1;
        ec[v][j] = g.exponent[n];
        if (!MASK) cb[v][j] = bias[n];
      }
    if (MASK) {
      const uint8_t* base = g.mask + m0 * g.ldm;
#pragma unroll
      for (int u = 0; u < FM; ++u) {
        const int last = (int)(g.M - 1 - m0 < BM ? g.M - 1 - m0 : BM);
        const uint32_t r = (uint32_t)(row + 16 * u < last ? row + 16 * u : last) * (uint32_t)g.ldm;
#pragma unroll
        for (int v = 0; v < FN; ++v) {
          const int c = (int)n0 + col + 16 * v;
          mask[u][v] = *reinterpret_cast<const uint32_t*>(base + (r + (c < (int)g.ldm ? (uint32_t)c : 0u)));
        }
      }
    }
    slice([&] {  // here by now: taken before the next loads, so that nothing is waited for between the stores
#pragma unroll
      for (int v = 0; v < FN; ++v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(ec[v][j]));
        if (!MASK)
#pragma unroll
          for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(cb[v][j]));
        if (MASK)
#pragma unroll
          for (int u = 0; u < FM; ++u) asm volatile("" : "+v"(mask[u][v]));
      }
    });
    matrix_drain();
    if (!MASK && !biased)
#pragma unroll
      for (int v = 0; v < FN; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j) cb[v][j] = 0.f;
#pragma unroll
    for (int u = 0; u < FM; ++u)
#pragma unroll
      for (int v = 0; v < FN; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // (a cut sum: the mask of each part, no bias)
          const float o = __builtin_ldexpf(acc[u][v][j], ea[u] + ec[v][j] - 279);  // 138 + 141
          acc[u][v][j] = !MASK ? o + cb[v][j] : ((mask[u][v] >> (8 * j)) & 255u) ? o : 0.f;
        }
    fresh = true;
    left = m0 + BM <= g.M && n0 + BN <= g.N;  // (a tile cut off by the matrix's end stores less)
    int at = lane;
    asm volatile("" : "+v"(at));
    if (left) {  // offsets in a tile fit 32 bits: row strides are at most 2^22
      float* const base = to + m0 * ldo + n0;
      const uint32_t o = 4 * ((uint32_t)(wm + (at & 15)) * (uint32_t)ldo + (uint32_t)(wn + 4 * (at >> 4)));
#pragma unroll
      for (int u = 0; u < FM; ++u)
#pragma unroll
        for (int v = 0; v < FN; ++v)
          store_any(reinterpret_cast<unsigned char*>(base) + (o + 64u * u * (uint32_t)ldo) + 64 * v, acc[u][v]);
    } else {
#pragma unroll
      for (int u = 0; u < FM; ++u) {
        const int64_t m = m0 + wm + 16 * u + (at & 15);
#pragma unroll
        for (int v = 0; v < FN; ++v) {
          const int64_t n = n0 + wn + 16 * v + 4 * (at >> 4);
          if (m >= g.M || n >= g.N) continue;
          float* p = to + m * ldo + n;
          if (n + 4 <= g.N) {
            store_any(p, acc[u][v]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (n + j < g.N) p[j] = acc[u][v][j];
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < FM; ++u)
#pragma unroll
      for (int v = 0; v < FN; ++v) acc[u][v] = zero4();
  }
}

// ---- launches ------------------------------------------------------------------------------------------
// once for each kernel and device
template <typename K>
static int allow_lds(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (bytes <= 65536) return 0;
  if (const int e = (int)hipGetDevice(&dev)) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return 0;
  const int e = (int)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (!e) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <int MODE, int DT>
static int finish_parts(const LowGemm& g, hipStream_t s) {
  if (g.splits <= 1) return (int)hipGetLastError();
  const int64_t quads = (g.N + 3) / 4, n = g.M * quads;
  hipLaunchKernelGGL((k_low_finish<MODE, DT>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, g, quads);
  return (int)hipGetLastError();
}

template <int MODE, int DT, int BM, int BN, int WM, int WN>
static int run_low_gemm(const LowGemm& g, hipStream_t s) {
  const int64_t mt = (g.M + BM - 1) / BM, nt = (g.N + BN - 1) / BN;
  constexpr int lds = 2 * (BM + BN) * SLICE;
  auto kernel = k_low_gemm<MODE, DT, BM, BN, WM, WN>;
  static std::atomic<uint64_t> done{0};
  if (const int e = allow_lds(kernel, lds, done)) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(mt * nt), (unsigned)g.splits), dim3(64 * WM * WN), lds, s, g, mt, nt);
  return finish_parts<MODE, DT>(g, s);
}

template <int BM, int BN, int WM, int WN, bool VEC, bool RELU, bool MASK>
static int run_low_gemm_f(const LowGemm& g, hipStream_t s) {
  const int64_t mt = (g.M + BM - 1) / BM, nt = (g.N + BN - 1) / BN, tiles = mt * nt;
  constexpr int lds = 256 * BM + 384 * BN + 128 * BM + 8 * BM, per_cu = 163840 / lds;  // resident workgroups
  auto kernel = k_low_gemm_f<BM, BN, WM, WN, VEC, RELU, MASK>;
  static std::atomic<uint64_t> done{0};
  if (const int e = allow_lds(kernel, lds, done)) return e;
  const int64_t fill = 256 * per_cu;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles < fill ? tiles : fill), (unsigned)g.splits), dim3(64 * WM * WN), lds, s, g,
                     (int32_t)tiles, (int32_t)nt);
  return finish_parts<LOW_F32, NC_F32>(g, s);
}

// Tiles and cuts of the sum.  256 compute units; a large tile reads less LDS for each product, a small one (or
// a cut sum) fills the units when the output is small.  M x K x N in us (S, M, L: tiles; x4: cuts):
//   float     8192 x 1024 x 1024 S 110, M 78, L 67;  4096 x 1024 x 1024 S 61, M 44, L x2 51;  1024 x 4096 x 4096 M 148,
//             L x2 136;  2048 x 4096 x 1024 S 115, M x2 90, L x4 79;  8192 x 8192 x 256 S 234, L x4 145;  2000 x 2000 x 500
//             S x2 41, M x4 33;  500 x 1024 x 1024 S x4 22, M x8 23;  65536 x 1024 x 64 S 82, M 95, L 115
//   bfloat16  8192 x 1024 x 1024 S 32, M 28, L 37;  4096 x 1024 x 1024 S 19, M 22;  1024 x 4096 x 4096 S 61, M 58;
//             1000 x 1000 x 1000 S 14, S x2 17;  200 x 4096 x 256 S x12 12, x4 13
//   int8      8192 x 1024 x 1024 S 22, M 20, L 27;  4096 x 1024 x 1024 S 14, M 16;  65536 x 1024 x 64 S 17, M 20, L 27
enum LowTile { TILE_SMALL, TILE_MIDDLE, TILE_LARGE };
struct LowCut {
  LowTile tile;
  int splits;
};
static int64_t tiles_of(int64_t M, int64_t N, int bm, int bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); }

static LowCut low_cut(int mode, int64_t M, int64_t N, int64_t K) {
  const int64_t slices = (K * (mode == LOW_I8 ? 1 : mode == LOW_F32 ? 4 : 2) + SLICE - 1) / SLICE;
  const int64_t middle = N > 64 ? tiles_of(M, N, 128, 128) : 0;
  if (mode == LOW_F32) {
    const int64_t large = N > 128 ? tiles_of(M, N, 128, 256) : 0;
    if (large >= 192) return {TILE_LARGE, 1};
    auto cut = [&](int64_t tiles, int64_t most) { return tiles > 0 ? std::min(256 / tiles, slices / most) : 0; };
    if (large * cut(large, 32) >= 192) return {TILE_LARGE, (int)cut(large, 32)};
    if (middle >= 192) return {TILE_MIDDLE, 1};
    if (middle * cut(middle, 8) >= 192) return {TILE_MIDDLE, (int)cut(middle, 8)};
  } else {
    if (N > 128 && tiles_of(M, N, 256, 256) >= 192) return {TILE_LARGE, 1};
    if (middle >= (slices >= 32 ? 192 : 320)) return {TILE_MIDDLE, 1};
  }
  if (slices < 32) return {TILE_SMALL, 1};
  const int64_t cuts = std::min(512 / std::max<int64_t>(tiles_of(M, N, 64, 64), 1), slices / 8);  // 8 slices at least
  return {TILE_SMALL, (int)std::max<int64_t>(cuts, 1)};
}

int low_gemm_splits(int mode, int64_t M, int64_t N, int64_t K) { return low_cut(mode, M, N, K).splits; }

template <int MODE, int DT>
static int pick_low_gemm(const LowGemm& g, hipStream_t s) {
  switch (low_cut(MODE, g.M, g.N, g.K).tile) {
    case TILE_LARGE: return run_low_gemm<MODE, DT, 256, 256, 2, 4>(g, s);
    case TILE_MIDDLE: return run_low_gemm<MODE, DT, 128, 128, 2, 2>(g, s);
    default: return run_low_gemm<MODE, DT, 64, 64, 1, 4>(g, s);
  }
}

template <bool VEC, bool RELU, bool MASK>
static int pick_low_gemm_f(const LowGemm& g, hipStream_t s) {
  switch (low_cut(LOW_F32, g.M, g.N, g.K).tile) {
    case TILE_LARGE: return run_low_gemm_f<128, 256, 2, 4, VEC, RELU, MASK>(g, s);
    case TILE_MIDDLE: return run_low_gemm_f<128, 128, 4, 2, VEC, RELU, MASK>(g, s);
    default: return run_low_gemm_f<64, 64, 2, 2, VEC, RELU, MASK>(g, s);
  }
}

int launch_low_gemm(const LowGemm& g, hipStream_t s) {
  if (g.M <= 0 || g.N <= 0) return 0;
  switch (g.mode) {
    case LOW_I8:
      if (g.out_dtype == NC_F32) return pick_low_gemm<LOW_I8, NC_F32>(g, s);
      return g.out_dtype == NC_F16 ? pick_low_gemm<LOW_I8, NC_F16>(g, s) : pick_low_gemm<LOW_I8, NC_BF16>(g, s);
    case LOW_BF16: return pick_low_gemm<LOW_BF16, NC_BF16>(g, s);
    case LOW_F16: return pick_low_gemm<LOW_F16, NC_F16>(g, s);
    case LOW_F32: {
      const bool vec = wide8(g.K);
      if (g.mask && (g.a_relu || g.bias || g.relu)) return (int)hipErrorInvalidValue;  // no call has both
      if (vec) return g.mask ? pick_low_gemm_f<true, false, true>(g, s)
                    : g.a_relu ? pick_low_gemm_f<true, true, false>(g, s) : pick_low_gemm_f<true, false, false>(g, s);
      return g.mask ? pick_low_gemm_f<false, false, true>(g, s)
             : g.a_relu ? pick_low_gemm_f<false, true, false>(g, s) : pick_low_gemm_f<false, false, false>(g, s);
    }
  }
  return (int)hipErrorInvalidValue;
}

// ---- few rows, or few columns ------------------------------------------------------------------------------
// The int8 product where a launch costs more than its work, or where the weight's bytes are all there is
// to it.  4 waves; each streams 16 channels of the weight from memory into the instruction's first operand
// (lane (i, q): channel i, 16 bytes at 16 q of every 64), 8 loads ahead; the second operand is up to 16 MT
// rows of x codes.  WK = 4: the waves share 16 channels and a quarter of the sum each (few rows, long sums);
// WK = 1: 16 channels each (short sums).
// DX >= 0: x is encoded here, by every workgroup for itself, while the first weights are on their way: one
// launch instead of two, worth it up to 8192 values a workgroup.  1 x 8192 x 8192 bfloat16: 17.3 us, 3.9 TB/s of weight.
constexpr int SMALL_PAD = 16;  // bytes behind a row of codes in LDS: rows start 4 banks apart

template <int DX, bool VEC, int MT, int WK>
__global__ void __launch_bounds__(256) k_low_small(const LowSmall p) {
  const LowGemm& g = p.g;
  static_assert(WK == 4 || DX >= 0, "given codes: the sums' barriers are between the scales and their use");
  constexpr int RB = 16 * MT;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];  // x codes; then the waves' sums
  __shared__ float scale[RB];
  __shared__ uint32_t red[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, q = lane >> 4;
  const int kp = (int)g.ldb, row_bytes = kp + SMALL_PAD;
  const int64_t n0 = (int64_t)blockIdx.x * (WK == 4 ? 16 : 64) + (WK == 4 ? 0 : 16 * wave);
  const int64_t m0 = (int64_t)blockIdx.y * RB;
  const int rows = (int)(g.M - m0 < RB ? g.M - m0 : RB);
  const int ksteps = (int)((g.K + 63) / 64);  // code rows are padded to whole steps
  const int k0 = WK == 4 ? ksteps * wave / 4 : 0, k1 = WK == 4 ? ksteps * (wave + 1) / 4 : ksteps;
  const int64_t ch = n0 + i < g.N ? n0 + i : g.N - 1;
  const uint8_t* wrow = g.B + ch * g.ldb + 16 * q;
  constexpr int DEEP = 8;
  uint4 w[DEEP];
#pragma unroll
  for (int d = 0; d < DEEP; ++d) {
    const int k = k0 + d < k1 ? k0 + d : (k1 > 0 ? k1 - 1 : 0);
    w[d] = *reinterpret_cast<const uint4*>(wrow + 64 * k);
  }
  if (DX >= 0) {
    constexpr int C = 4;
    const int chunks = kp / 8;
    if (WK == 4 && rows < 4) {  // the workgroup takes a row: 256 C chunks
      for (int r = 0; r < rows; ++r) {
        float v[C][8];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < C; ++j) load8<DX, VEC>(p.x, (m0 + r) * p.x_stride, threadIdx.x + 256 * j, g.K, v[j]);
#pragma unroll
        for (int j = 0; j < C; ++j) {
          clear8<VEC>(threadIdx.x + 256 * j, g.K, v[j]);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, mag_bits(v[j][e]));
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        if (lane == 0) red[wave] = top;
        __syncthreads();
        top = max(max(red[0], red[1]), max(red[2], red[3]));
        __syncthreads();
        const bool bad = top >= 0x7f800000u;
        const float s = row_scale(top), rcp = 1.f / s;
        if (threadIdx.x == 0) scale[r] = bad ? __builtin_nanf("") : s;
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const int c = threadIdx.x + 256 * j;
          if (c < chunks) *reinterpret_cast<uint2*>(lds + r * row_bytes + 8 * c) = row_codes(v[j], bad, s, rcp);
        }
      }
    } else if (WK == 4) {  // a wave takes a row: 64 C chunks
      for (int r = wave; r < rows; r += 4) {
        float v[C][8];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < C; ++j) load8<DX, VEC>(p.x, (m0 + r) * p.x_stride, lane + 64 * j, g.K, v[j]);
#pragma unroll
        for (int j = 0; j < C; ++j) {
          clear8<VEC>(lane + 64 * j, g.K, v[j]);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, mag_bits(v[j][e]));
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        const bool bad = top >= 0x7f800000u;
        const float s = row_scale(top), rcp = 1.f / s;
        if (lane == 0) scale[r] = bad ? __builtin_nanf("") : s;
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (lane + 64 * j < chunks) *reinterpret_cast<uint2*>(lds + r * row_bytes + 8 * (lane + 64 * j)) = row_codes(v[j], bad, s, rcp);
      }
    } else {  // half a wave takes a row of up to 32 chunks, every eighth one, all loads first
      const int c = lane & 31, r0 = 2 * wave + (lane >> 5);
      float v[RB / 8][8];
#pragma unroll
      for (int j = 0; j < RB / 8; ++j) {
        const int r = r0 + 8 * j < rows ? r0 + 8 * j : rows - 1;
        load8<DX, VEC>(p.x, (m0 + r) * p.x_stride, c, g.K, v[j]);
      }
#pragma unroll
      for (int j = 0; j < RB / 8; ++j) {
        const int r = r0 + 8 * j;
        uint32_t top = 0;
        clear8<VEC>(c, g.K, v[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, mag_bits(v[j][e]));
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        const bool bad = top >= 0x7f800000u;
        const float s = row_scale(top), rcp = 1.f / s;
        if (r < rows) {
          if (c == 0) scale[r] = bad ? __builtin_nanf("") : s;
          if (c < chunks) *reinterpret_cast<uint2*>(lds + r * row_bytes + 8 * c) = row_codes(v[j], bad, s, rcp);
        }
      }
    }
    __syncthreads();
  } else if ((int)threadIdx.x < RB) {
    scale[threadIdx.x] = g.row_scale[m0 + ((int)threadIdx.x < rows ? (int)threadIdx.x : rows - 1)];
  }
  // x's operands: rows behind the last are others (LDS holds no more than `rows`), not stored
  const uint8_t* xrow[MT];
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    const int r = 16 * u + i < rows ? 16 * u + i : rows - 1;
    xrow[u] = DX >= 0 ? lds + r * row_bytes + 16 * q : g.A + (m0 + r) * g.lda + 16 * q;
  }
  intx4 acc[MT];
#pragma unroll
  for (int u = 0; u < MT; ++u) acc[u] = intx4{0, 0, 0, 0};
  for (int k = k0; k < k1; k += DEEP) {
    uint4 x[DX >= 0 ? 1 : DEEP][MT];
    if (DX < 0) {
#pragma unroll
      for (int d = 0; d < DEEP; ++d)
#pragma unroll
        for (int u = 0; u < MT; ++u) x[DX >= 0 ? 0 : d][u] = *reinterpret_cast<const uint4*>(xrow[u] + 64 * (k + d < k1 ? k + d : k1 - 1));
    }
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const uint4 wd = w[d];
      if (k + DEEP < k1) w[d] = *reinterpret_cast<const uint4*>(wrow + 64 * (k + DEEP + d < k1 ? k + DEEP + d : k1 - 1));
      if (k + d < k1) {
#pragma unroll
        for (int u = 0; u < MT; ++u) {
          const uint4 xd = DX >= 0 ? *reinterpret_cast<const uint4*>(xrow[u] + 64 * (k + d)) : x[DX >= 0 ? 0 : d][u];
          acc[u] = Mac<LOW_I8>::mac(wd, xd, acc[u]);
        }
      }
    }
  }
  matrix_drain();
  if (WK == 4) {  // the four sums of a block: wave u adds up block u of rows
    __syncthreads();
    intx4* part = reinterpret_cast<intx4*>(lds);
#pragma unroll
    for (int u = 0; u < MT; ++u) part[(wave * MT + u) * 64 + lane] = acc[u];
    __syncthreads();
    if (wave >= MT) return;
    intx4 t = part[wave * 64 + lane];
#pragma unroll
    for (int k = 1; k < 4; ++k) t += part[(k * MT + wave) * 64 + lane];
    acc[0] = t;
  }
  const int64_t n = n0 + 4 * q;
  if (n >= g.N) return;
  Scale cs[4];
  float cb[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t nn = n + j < g.N ? n + j : g.N - 1;
    cs[j] = split_scale(g.col_scale[nn]);
    cb[j] = g.bias ? load_bias(g.bias, g.bias_dtype, nn) : 0.f;
  }
#pragma unroll
  for (int u = 0; u < (WK == 4 ? 1 : MT); ++u) {
    const int r = 16 * (WK == 4 ? wave : u) + i;
    if (r >= rows) continue;
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = finish<LOW_I8>(g, (float)acc[u][j], split_scale(scale[r]) * cs[j], cb[j], 1u);
    if (g.out_dtype == NC_F32) store4<NC_F32>(g, m0 + r, n, o);
    else if (g.out_dtype == NC_F16) store4<NC_F16>(g, m0 + r, n, o);
    else store4<NC_BF16>(g, m0 + r, n, o);
  }
}

// Which products it takes with x to encode: up to 3 rows of 8192, 16 of 2048, or short sums (256) of at
// most 512 workgroups: beyond those every column tile's own encoding costs more than the launch that it
// saves (bfloat16, us, here | encoded once: 777 x 93 x 1001 14.9 | 16.5, 777 x 256 x 4096 19.2 | 17.6).
static bool short_sums(int64_t M, int64_t K) { return K <= 256 && M > 16; }
bool low_small_encodes(int64_t M, int64_t N, int64_t K) {
  if (short_sums(M, K)) return ((M + 63) / 64) * ((N + 63) / 64) <= 512;
  return (M < 4 && K <= 8192) || (M <= 16 && K <= 2048);
}

template <int DX, bool VEC, int MT, int WK>
static int run_low_small(const LowSmall& a, hipStream_t s) {
  const int rb = 16 * MT, rows = (int)(a.g.M < rb ? a.g.M : rb);
  int lds = DX >= 0 ? rows * (int)(a.g.ldb + SMALL_PAD) : 0;
  if (WK == 4 && lds < 4 * MT * 1024) lds = 4 * MT * 1024;
  const dim3 grid((unsigned)((a.g.N + (WK == 4 ? 15 : 63)) / (WK == 4 ? 16 : 64)), (unsigned)((a.g.M + rb - 1) / rb));
  hipLaunchKernelGGL((k_low_small<DX, VEC, MT, WK>), grid, dim3(256), lds, s, a);
  return (int)hipGetLastError();
}
template <int DX, bool VEC>
static int encode_low_small(const LowSmall& a, hipStream_t s) {
  if (short_sums(a.g.M, a.g.K)) return run_low_small<DX, VEC, 4, 1>(a, s);
  return run_low_small<DX, VEC, 1, 4>(a, s);
}

int launch_low_small(const LowSmall& a, hipStream_t s) {
  if (a.g.M <= 0 || a.g.N <= 0) return 0;
  const bool vec = a.x_dtype >= 0 && wide8(a.g.K);
  switch (a.x_dtype) {
    case NC_F32: return vec ? encode_low_small<NC_F32, true>(a, s) : encode_low_small<NC_F32, false>(a, s);
    case NC_F16: return vec ? encode_low_small<NC_F16, true>(a, s) : encode_low_small<NC_F16, false>(a, s);
    case NC_BF16: return vec ? encode_low_small<NC_BF16, true>(a, s) : encode_low_small<NC_BF16, false>(a, s);
  }
  if (a.g.M <= 16) return run_low_small<-1, false, 1, 4>(a, s);
  if (a.g.M <= 32) return run_low_small<-1, false, 2, 4>(a, s);
  return run_low_small<-1, false, 4, 4>(a, s);
}

// ---- weight gradient -----------------------------------------------------------------------------------
// A workgroup sums its rows [rb, re) of dY and codes into a BN x BK tile of dW.  A stage is MS rows of
// both operands in LDS as 16-bit elements, row-major (the sum's index m is the row).  ds_read_b64_tr_b16
// hands lane (i, q) four rows of column i: rows 4 q + 0..3 of a 4-row x 16-column block, so two of them
// make the 8 sum indices of a lane's operand: m = 4 q + e and 16 + 4 q + e, the same for both operands.
// Rows of BN (BK) elements are cut into 32-byte units; unit u of row m lies at u ^ (m & 7): the 8 rows
// that 32 lanes read together then cover all 64 banks.
// Measured, M x K x N: bfloat16 8192 x 4096 x 4096 239 us = 1.15 PFLOP/s with the values' decoding (11 us) and a call from Python,
// 220000 x 256 x 256 67 us; float 220000 x 256 x 256 100 us = 0.86 PFLOP/s of plane products, both with the sums of the parts.
__device__ __forceinline__ uint2 tr_read(uint32_t at) {
  typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)at));
}

// 16 codes of one row and group -> 16 elements of 16 bits: the values that k_decode gives too
template <bool F16, bool RELU>
__device__ __forceinline__ void decode16(uint4 c, float step, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t o[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // signed codes, -127 to 127, as code + 127 (no byte borrows from the next): 127 of the largest steps are a
    // finite float, 128 are not
    const uint32_t b = RELU ? w[j] : (w[j] ^ 0x80808080u) - 0x01010101u;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = (float)((b >> (8 * e)) & 255u);
      v[e] = __builtin_fmaf(f, step, RELU ? -step : -127.f * step);
      if (RELU) v[e] = relu_keep_nan(v[e]);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (F16) {  // exact in half, but 65536: a conversion toward 0 makes it 65504
        o[2 * j + e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(v[2 * e], v[2 * e + 1]));
      } else {  // exact in bfloat16: the upper halves
        o[2 * j + e] = upper_halves(v[2 * e], v[2 * e + 1]);
      }
    }
  }
  lo = uint4{o[0], o[1], o[2], o[3]};
  hi = uint4{o[4], o[5], o[6], o[7]};
}

constexpr int SUM_ROWS = 512;  // rows that one workgroup adds up for the bias gradient

// sums of the columns [n0, n0 + BN) of dY over rows [rb, re): a thread takes 8 columns of every R-th row, and
// the R sums of a column are added in order
template <int DT, int BN, int T>
__device__ __forceinline__ void put_col_sums(const LowWgrad& g, int64_t n0, int64_t piece, const float (&t)[8], float* red) {
  constexpr int C8 = BN / 8, R = T / C8;
  const int c = threadIdx.x % C8, w = threadIdx.x / C8;
  __syncthreads();  // the buffers are read
#pragma unroll
  for (int e = 0; e < 8; ++e) red[w * BN + 8 * c + e] = t[e];
  __syncthreads();
  for (int e = threadIdx.x; e < BN; e += T) {
    float sum = 0.f;
    for (int k = 0; k < R; ++k) sum += red[k * BN + e];
    if (n0 + e >= g.N) continue;
    if (!g.db) g.sums[piece * g.N + n0 + e] = sum;
    else if (DT == NC_F32) reinterpret_cast<float*>(g.db)[n0 + e] = sum;
    else reinterpret_cast<uint16_t*>(g.db)[n0 + e] = f32_elem<DT>(sum);
  }
}
template <int DT, int BN, int T, bool VEC>
__device__ __forceinline__ void col_sums(const LowWgrad& g, int64_t n0, int64_t rb, int64_t re, int64_t piece, float* red) {
  constexpr int C8 = BN / 8, R = T / C8;
  const int64_t c = n0 / 8 + threadIdx.x % C8;
  const int64_t cols = DT == NC_F32 ? g.N : (g.N + 7) / 8 * 8;  // 16-bit rows are padded to 64 columns
  float t[8] = {};
  int64_t r = rb + threadIdx.x / C8;
  for (; r + 3 * R < re; r += 4 * R) {
    float v[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) load8<DT, VEC>(g.dy, (r + u * R) * g.ldy, c, cols, v[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) clear8<VEC>(c, cols, v[u]);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] += (v[0][e] + v[1][e]) + (v[2][e] + v[3][e]);
  }
  for (; r < re; r += R) {
    float v[8];
    load8<DT, VEC>(g.dy, r * g.ldy, c, cols, v);
    clear8<VEC>(c, cols, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] += v[e];
  }
  put_col_sums<DT, BN, T>(g, n0, piece, t, red);
}

// The pipeline is k_low_gemm's: phases of 4 x FK blocks, the next phase's operands read from LDS while
// one multiplies; before a stage's last phase the barrier that frees its half.  dY goes into LDS by itself,
// codes through registers: loaded with dY a stage ahead, decoded and written before the stage's
// last phase but one.
// NP = 3: dY is float, split into its planes on the way like A in k_low_gemm_f, and its columns are added up
// in passing (the bias gradient).  Where dW is not asked for, the workgroups add up the columns alone.
// CODED = false: the codes' values lie in memory already, with zeros behind the last row, and go into LDS by
// themselves too.
template <int NP, int DT, bool RELU, bool CODED, int BN, int BK, int MS, int WN, int WK, bool VEC>
__global__ void __launch_bounds__(64 * WN * WK) __attribute__((amdgpu_waves_per_eu(2))) k_low_wgrad(const LowWgrad g) {
  constexpr int W = WN * WK, T = 64 * W;
  constexpr int FN = BN / WN / 16, FK = BK / WK / 16;
  constexpr int YROW = 2 * BN, XROW = 2 * BK;               // bytes of a staged row
  constexpr int YSTAGE = MS * YROW, XSTAGE = MS * XROW, STAGE = NP * YSTAGE + XSTAGE;
  constexpr bool F16 = DT == NC_F16;
  constexpr int YL = NP == 3 ? 0 : YSTAGE / 1024 / W;       // 1-KB loads a wave
  constexpr int YF = NP == 3 ? MS * BN / 8 / T : 0;         // 8-column chunks a thread
  constexpr int XL = CODED ? MS * BK / 16 / T : 0;          // 16-code loads a thread
  constexpr int XD = CODED ? 0 : XSTAGE / 1024 / W;         // 1-KB loads of values a wave
  constexpr int NG = FN / 4, NH = MS / 32, PH = NH * NP * NG;
  static_assert(YSTAGE % (1024 * W) == 0 && MS * BK % (16 * T) == 0 && XSTAGE % (1024 * W) == 0 && YL + YF > 0, "whole loads");
  static_assert(NP == 1 || MS * BN % (8 * T) == 0, "whole chunks");
  static_assert(BN >= 128 && BK >= 128, "rows of at least 8 units of 32 bytes");
  static_assert((NG == 1 || (NG == 2 && FN == 8)) && YROW % 256 == 0 && XROW % 256 == 0, "the second group is 128 bytes away");
  static_assert(FN % 4 == 0 && PH >= 2 && (NH == 1 || NH == 2), "phases");
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q = lane >> 4, j16 = lane & 15;
  const int64_t n0 = (int64_t)blockIdx.x * BN, k0 = (int64_t)blockIdx.y * BK;
  int64_t rb = (int64_t)blockIdx.z * g.rows_per;
  int64_t re = rb + g.rows_per < g.M ? rb + g.rows_per : g.M;
  const int64_t ychunks = (g.N + 7) / 8, xchunks = g.code_stride / 16, steps_row = g.code_stride / CODE_GROUP;
  const int total = (int)((re - rb + MS - 1) / MS);
  const uint32_t lds0 = lds_address(lds);
  const int kt = (int)gridDim.y;
  if (!g.want_dw) {
    const int piece = blockIdx.y;
    rb += piece * (int64_t)SUM_ROWS;
    re = rb + SUM_ROWS < re ? rb + SUM_ROWS : re;
    col_sums<DT, BN, T, VEC>(g, n0, rb, re, (int64_t)blockIdx.z * g.pieces + piece, reinterpret_cast<float*>(lds));
    return;
  }

  float yf[YF > 0 ? YF : 1][8], ysum[8] = {};  // float dY: its columns' sums in passing (T is a multiple of BN / 8)
  const bool summing = YF > 0 && g.want_db && blockIdx.y == 0;
  const bool ragged = g.N % 8 != 0 && n0 + BN > g.N;  // the last columns: moved to their places
  uint32_t yo[YL > 0 ? YL : 1];  // 16-bit dY: byte offsets from the stage's first row
  int yrow[YL > 0 ? YL : 1];
#pragma unroll
  for (int l = 0; l < YL; ++l) {
    const int at = (wave * YL + l) * 64 + lane;  // 16-byte position in the tile
    yrow[l] = at / (YROW / 16);
    int64_t c = n0 / 8 + ((at % (YROW / 16)) ^ ((yrow[l] & 7) << 1));
    c = c < ychunks ? c : ychunks - 1;  // columns behind the last: not stored
    yo[l] = (uint32_t)(yrow[l] * 2 * g.ldy + 16 * c);
  }
  uint32_t xd[XD > 0 ? XD : 1];
#pragma unroll
  for (int l = 0; l < XD; ++l) {
    const int at = (wave * XD + l) * 64 + lane, row = at / (XROW / 16);
    int64_t c = k0 / 8 + ((at % (XROW / 16)) ^ ((row & 7) << 1));
    c = c < 2 * xchunks ? c : 2 * xchunks - 1;  // columns behind the last: not stored
    xd[l] = (uint32_t)(row * 2 * g.code_stride + 16 * c);
  }
  uint32_t xo[XL > 0 ? XL : 1], so[XL > 0 ? XL : 1];  // codes and steps
#pragma unroll
  for (int l = 0; l < XL; ++l) {
    const int at = l * T + threadIdx.x, row = at / (BK / 16);
    int64_t c = k0 / 16 + at % (BK / 16);
    c = c < xchunks ? c : xchunks - 1;
    xo[l] = (uint32_t)(row * g.code_stride + 16 * c);
    so[l] = (uint32_t)(row * steps_row + (c >> 1));
  }
  auto stage_y = [&](int t) {
#pragma unroll
    for (int l = 0; l < YF; ++l) {
      const int at = l * T + threadIdx.x, row = at / (BN / 8);
      const int64_t m = rb + (int64_t)t * MS + row, mm = m < re ? m : re - 1;
      load8<NC_F32, VEC>(g.dy, mm * g.ldy, n0 / 8 + at % (BN / 8), g.N, yf[l]);
    }
    if (YL > 0) {
      const uint8_t* base = reinterpret_cast<const uint8_t*>(g.dy) + 2 * (rb + (int64_t)t * MS) * g.ldy;
      const int last = (int)(re - rb - (int64_t)t * MS) - 1;  // rows behind the last: its copies, cleared later
#pragma unroll
      for (int l = 0; l < YL; ++l) {
        const uint32_t o = last >= MS - 1 || yrow[l] <= last ? yo[l] : yo[l] - (uint32_t)(yrow[l] - last) * (uint32_t)(2 * g.ldy);
        load_lds16(base, o, lds0 + (t & 1) * STAGE + (wave * YL + l) * 1024);
      }
    }
    if (XD > 0) {
      const uint8_t* base = reinterpret_cast<const uint8_t*>(g.x) + 2 * (rb + (int64_t)t * MS) * g.code_stride;
#pragma unroll
      for (int l = 0; l < XD; ++l) load_lds16(base, xd[l], lds0 + (t & 1) * STAGE + NP * YSTAGE + (wave * XD + l) * 1024);
    }
  };
  uint4 xc[XL > 0 ? XL : 1];
  uint32_t xs[XL > 0 ? XL : 1];
  auto load_x = [&](int t) {
    const uint8_t* codes = g.codes + (rb + (int64_t)t * MS) * g.code_stride;
    const uint8_t* steps = g.steps + (rb + (int64_t)t * MS) * steps_row;
    const int last = (int)(re - rb - (int64_t)t * MS) - 1;
#pragma unroll
    for (int l = 0; l < XL; ++l) {
      const int row = (l * T + (int)threadIdx.x) / (BK / 16);
      const uint32_t back = row <= last ? 0u : (uint32_t)(row - last);
      xc[l] = *reinterpret_cast<const uint4*>(codes + (xo[l] - back * (uint32_t)g.code_stride));
      xs[l] = steps[so[l] - back * (uint32_t)steps_row];
    }
  };
  auto store_xy = [&](int t) {
    unsigned char* s = lds + (t & 1) * STAGE + NP * YSTAGE;
#pragma unroll
    for (int l = 0; l < XL; ++l) {
      const int at = l * T + threadIdx.x, row = at / (BK / 16), u = at % (BK / 16);
      __builtin_amdgcn_sched_barrier(0);  // one chunk's temporaries at a time
      const bool in = rb + (int64_t)t * MS + row < re;
      const float step = xs[l] == 255u ? __builtin_nanf("") : __builtin_bit_cast(float, xs[l] << 23);
      uint4 lo, hi;
      decode16<F16, RELU>(xc[l], step, lo, hi);
      if (!in) lo = hi = uint4{0u, 0u, 0u, 0u};
      uint4* d = reinterpret_cast<uint4*>(s + row * XROW + 32 * (u ^ (row & 7)));
      d[0] = lo;
      d[1] = hi;
    }
#pragma unroll
    for (int l = 0; l < YF; ++l) {
      const int at = l * T + threadIdx.x, row = at / (BN / 8), c = at % (BN / 8);
      if (ragged) clear8<VEC>(n0 / 8 + c, g.N, yf[l]);  // (columns behind the last are not stored)
      const bool in = rb + (int64_t)t * MS + row < re;
      if (!in)
#pragma unroll
        for (int e = 0; e < 8; ++e) yf[l][e] = 0.f;
      if (summing)
#pragma unroll
        for (int e = 0; e < 8; ++e) ysum[e] += yf[l][e];
      uint4 p[3];
      split3(yf[l], p);
      unsigned char* y = lds + (t & 1) * STAGE + row * YROW + 16 * (c ^ ((row & 7) << 1));
#pragma unroll
      for (int k = 0; k < NP; ++k) *reinterpret_cast<uint4*>(y + k * YSTAGE) = p[k];
    }
  };

  floatx4 acc[FN][FK];
#pragma unroll
  for (int u = 0; u < FN; ++u)
#pragma unroll
    for (int v = 0; v < FK; ++v) acc[u][v] = zero4();
  const int wn = (wave / WK) * (BN / WN), wk = (wave % WK) * (BK / WK);
  // 16-bit dY: the bias gradient as products with ones, every kt-th stage by each tile column and every
  // WK-th block of n by each wave (65536 x 1024 x 1024: workgroups that read dY again for it took 115 us more)
  constexpr int FB = NP == 1 ? FN / WK : 1;
  floatx4 bias[FB];
#pragma unroll
  for (int u = 0; u < FB; ++u) bias[u] = zero4();
  int next_bias = NP == 1 && g.want_db ? (int)blockIdx.y : total;
  // a lane's transposed reads: row tr of a step, 8 bytes tc of a 32-byte unit; the addresses are kept for the
  // first group of units and recomputed from them at each read, so that they take few registers
  const int tr = 4 * q + (j16 >> 2), tc = 8 * (j16 & 3);
  uint32_t ya[4], xa[FK];
#pragma unroll
  for (int u = 0; u < 4; ++u) ya[u] = lds0 + tr * YROW + 32 * ((wn / 16 + u) ^ (tr & 7)) + tc;
#pragma unroll
  for (int v = 0; v < FK; ++v) xa[v] = lds0 + NP * YSTAGE + tr * XROW + 32 * ((wk / 16 + v) ^ (tr & 7)) + tc;
  uint4 a[2][4], b[2][FK];
  auto pair = [](uint32_t at, int next) {
    asm volatile("" : "+v"(at));
    const uint2 x0 = tr_read(at), x1 = tr_read(at + next);
    return uint4{x0.x, x0.y, x1.x, x1.y};
  };
  // phase p = (half h, plane, group of 4 n blocks); the smallest plane first
  auto read = [&](int t, int p, int to_a, int to_b) {
    const int h = p / (NP * NG), pl = NP - 1 - (p / NG) % NP, gr = p % NG;
    const uint32_t s = (t & 1) * STAGE;
#pragma unroll
    for (int u = 0; u < 4; ++u)  // the second group's units: 4 more, of 32 bytes, in a row cut into 8
      a[to_a][u] = pair((ya[u] ^ (128u * gr)) + (s + pl * YSTAGE + 32 * h * YROW), 16 * YROW);
    if (p % (NP * NG) == 0) {
#pragma unroll
      for (int v = 0; v < FK; ++v) b[to_b][v] = pair(xa[v] + (s + 32 * h * XROW), 16 * XROW);
    }
  };
  auto multiply = [&](int p) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int v = 0; v < FK; ++v) {
        auto& c = acc[(p % NG) * 4 + u][v];
        c = Mac<F16 ? LOW_F16 : LOW_BF16>::mac(b[p / (NP * NG)][v], a[p & 1][u], c);
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto add_bias = [&](int t, int p) {
    if (NP != 1 || t != next_bias) return;
    constexpr uint32_t ONES = F16 ? 0x3c003c00u : 0x3f803f80u;
    const uint4 w = {ONES, ONES, ONES, ONES};
#pragma unroll
    for (int u0 = 0; u0 < 4; u0 += WK) {  // this wave's block of the WK, selected without a branch
      uint4 y = a[p & 1][u0];
#pragma unroll
      for (int u = 1; u < WK; ++u) {
        const bool mine = wave % WK == u;
        const uint4 o = a[p & 1][u0 + u];
        y = uint4{mine ? o.x : y.x, mine ? o.y : y.y, mine ? o.z : y.z, mine ? o.w : y.w};
      }
      constexpr int PER = 4 / WK > 0 ? 4 / WK : 1;  // blocks a group and wave
      auto& c = bias[((p % NG) * PER + u0 / WK) % FB];
      c = Mac<F16 ? LOW_F16 : LOW_BF16>::mac(w, y, c);
    }
    if (p == PH - 1) next_bias += kt;
  };
  // 16-bit dY: zeros for the copies behind the last row (whose infinities would be products 0 x inf)
  auto clear_tail = [&](int t) {
    const int in = (int)(re - rb - (int64_t)t * MS);
    if (NP != 1 || in >= MS) return;  // (the whole workgroup)
    for (int e = threadIdx.x; e < (MS - in) * (YROW / 16); e += T)
      *reinterpret_cast<uint4*>(lds + (t & 1) * STAGE + in * YROW + 16 * e) = uint4{0u, 0u, 0u, 0u};
    __syncthreads();
  };
  if (total > 0) {
    stage_y(0);
    load_x(0);
    store_xy(0);
    if (total > 1) {
      load_x(1);
      stage_y(1);
    }
    staged_barrier();
    clear_tail(0);
    read(0, 0, 0, 0);
    for (int t = 0; t + 1 < total; ++t) {
#pragma unroll
      for (int p = 0; p < PH; ++p) {
        if (p + 1 < PH) {
          if (p == PH - 2) store_xy(t + 1);
          read(t, p + 1, (p + 1) & 1, (p + 1) / (NP * NG));
        } else {
          staged_barrier();
          clear_tail(t + 1);
          if (t + 2 < total) {
            load_x(t + 2);
            stage_y(t + 2);
          }
          read(t + 1, 0, PH & 1, NH == 1 ? 1 : 0);
        }
        multiply(p);
        add_bias(t, p);
      }
      if (PH & 1)
#pragma unroll
        for (int u = 0; u < 4; ++u) a[0][u] = a[1][u];
      if (NH == 1)
#pragma unroll
        for (int v = 0; v < FK; ++v) b[0][v] = b[1][v];
    }
    read(total - 1, 0, 0, 0);  // again: kept across the loop's end, the operands would not fit the registers
#pragma unroll
    for (int p = 0; p < PH; ++p) {
      if (p + 1 < PH) read(total - 1, p + 1, (p + 1) & 1, (p + 1) / (NP * NG));
      multiply(p);
      add_bias(total - 1, p);
    }
  }
  matrix_drain();
  const int i = j16;
  float* part = g.part + (int64_t)blockIdx.z * g.N * g.K;
#pragma unroll
  for (int u = 0; u < FN; ++u) {
    const int64_t n = n0 + wn + 16 * u + i;
#pragma unroll
    for (int v = 0; v < FK; ++v) {
      const int64_t k = k0 + wk + 16 * v + 4 * q, at = n * g.K + k;
      if (n >= g.N || k >= g.K) continue;
      const floatx4 c = acc[u][v];
      if (!g.dw || DT == NC_F32) {
        float* p = (g.dw ? reinterpret_cast<float*>(g.dw) : part) + at;
        if (k + 4 <= g.K) {
          store_any(p, c);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k + e < g.K) p[e] = c[e];
        }
      } else {
        uint16_t* p = reinterpret_cast<uint16_t*>(g.dw) + at;
        uint16_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = f32_elem<DT>(c[e]);
        if (k + 4 <= g.K) {
          store_any(p, uint2{o[0] | (uint32_t)o[1] << 16, o[2] | (uint32_t)o[3] << 16});
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k + e < g.K) p[e] = o[e];
        }
      }
    }
  }
  if (summing) put_col_sums<DT, BN, T>(g, n0, blockIdx.z, ysum, reinterpret_cast<float*>(lds));
  if (NP == 1 && g.want_db && q == 0) {  // all rows of the product with ones are alike
#pragma unroll
    for (int u = 0; u < FN; ++u) {
      const int64_t n = n0 + wn + 16 * u + i;
      if (u % WK != wave % WK || n >= g.N) continue;
      const float sum = bias[u / WK < FB ? u / WK : 0][0];
      if (!g.db) g.sums[((int64_t)blockIdx.z * kt + blockIdx.y) * g.N + n] = sum;
      else reinterpret_cast<uint16_t*>(g.db)[n] = f32_elem<DT>(sum);
    }
  }
}

// Tiles: 256 x 256 (float: 128 of dY, whose three planes take the room, x 256) are 4/3 as fast in full, 128 x
// 128 leave fewer partial sums when an output of few tiles has to be cut along the rows.  Large tiles of
// 16-bit elements take the codes' values written out (4 bytes moved for a code, 0.6-1 ps): decoding them in
// each tile column costs 0.3-0.4 ps a code and column.  M x K x N, us with the values' decoding, bfloat16, small and
// large tiles: 1237 x 517 x 1031 53, 72; 4096 x 1024 x 1024 52, 59; 4096 x 512 x 4096 61, 65; 8192 x 2048 x 2048 150, 127;
// 1000 x 4096 x 4096 93, 77; 65536 x 1024 x 1024 313, 262; float 4096 x 1024 x 1024 48, 43; 220000 x 256 x 256 120, 107.
static bool wgrad_wide(int dtype, int64_t M, int64_t N, int64_t K) {
  if (dtype == NC_F32) return K > 128;
  const int64_t tiles = tiles_of(N, K, 256, 256);
  return N >= 1024 && (tiles >= 64 || (tiles >= 16 && M >= 65536));
}
bool low_wgrad_decodes(int dtype, int64_t M, int64_t N, int64_t K) { return dtype != NC_F32 && wgrad_wide(dtype, M, N, K); }

// Cuts of the rows.  Large tiles: one workgroup a compute unit.  Small ones: what a row costs a workgroup and
// a cut costs for an element of dW is balanced by sqrt(8000 M / (N K)) cuts (of 1 to 192, within 6 % of the best
// from 500 x 256 x 256 to 220000 x 256 x 256).  Up to 128 rows stay whole: 64 x 256 x 256 takes as long as in two
// parts, with a launch less.
void low_wgrad_splits(int dtype, int64_t M, int64_t N, int64_t K, bool want_dw, int32_t& splits, int32_t& pieces,
                      int64_t& rows_per) {
  const bool wide = wgrad_wide(dtype, M, N, K);
  const int64_t tn = wide && dtype != NC_F32 ? 256 : 128, tk = wide ? 256 : 128;
  const int64_t tiles = tiles_of(N, K, (int)tn, (int)tk);
  int64_t want = (wide ? 256 : 512) / tiles, most = wide ? (M + 127) / 128 : (M + 63) / 64;
  if (!wide) {
    const int64_t balanced = (int64_t)(sqrt(8000. * (double)M / ((double)N * (double)K)) + 0.5);
    if (want > balanced) want = balanced;
  }
  if (want > most) want = most;
  if (want < 1 || M <= 128) want = 1;
  rows_per = round_up((M + want - 1) / want, 64);
  if (rows_per < 64) rows_per = 64;
  splits = (int32_t)((M + rows_per - 1) / rows_per);
  if (splits < 1) splits = 1;
  pieces = (int32_t)(!want_dw ? (rows_per + SUM_ROWS - 1) / SUM_ROWS : dtype == NC_F32 ? 1 : (K + tk - 1) / tk);
}

template <int NP, int DT, bool RELU, bool CODED, int TN, int TK, int MS, int WN, int WK, bool VEC>
static int run_low_wgrad(const LowWgrad& g, hipStream_t s) {
  constexpr int lds = 2 * (NP * MS * 2 * TN + MS * 2 * TK);
  auto kernel = k_low_wgrad<NP, DT, RELU, CODED, TN, TK, MS, WN, WK, VEC>;
  static std::atomic<uint64_t> done{0};
  if (const int e = allow_lds(kernel, lds, done)) return e;
  const dim3 grid((unsigned)((g.N + TN - 1) / TN), (unsigned)(g.want_dw ? (g.K + TK - 1) / TK : g.pieces), (unsigned)g.splits);
  hipLaunchKernelGGL(kernel, grid, dim3(64 * WN * WK), lds, s, g);
  return (int)hipGetLastError();
}

template <int DT>
static int pick_low_wgrad(const LowWgrad& g, hipStream_t s) {
  if (wgrad_wide(DT, g.M, g.N, g.K)) {
    if (g.want_dw && !g.x) return (int)hipErrorInvalidValue;
    return run_low_wgrad<1, DT, false, false, 256, 256, 64, 2, 4, true>(g, s);
  }
  if (g.relu) return run_low_wgrad<1, DT, true, true, 128, 128, 64, 2, 2, true>(g, s);
  return run_low_wgrad<1, DT, false, true, 128, 128, 64, 2, 2, true>(g, s);
}

template <bool RELU, bool VEC>
static int pick_low_wgrad_f(const LowWgrad& g, hipStream_t s) {
  if (wgrad_wide(NC_F32, g.M, g.N, g.K)) return run_low_wgrad<3, NC_F32, RELU, true, 128, 256, 64, 2, 4, VEC>(g, s);
  return run_low_wgrad<3, NC_F32, RELU, true, 128, 128, 32, 2, 2, VEC>(g, s);
}

int launch_low_wgrad(const LowWgrad& g, hipStream_t s) {
  if (g.N <= 0 || g.K <= 0 || (!g.want_dw && !g.want_db)) return 0;
  switch (g.dtype) {
    case NC_F16: return pick_low_wgrad<NC_F16>(g, s);
    case NC_BF16: return pick_low_wgrad<NC_BF16>(g, s);
    case NC_F32: {
      const bool vec = wide8(g.N);
      if (vec) return g.relu ? pick_low_wgrad_f<true, true>(g, s) : pick_low_wgrad_f<false, true>(g, s);
      return g.relu ? pick_low_wgrad_f<true, false>(g, s) : pick_low_wgrad_f<false, false>(g, s);
    }
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace nc
