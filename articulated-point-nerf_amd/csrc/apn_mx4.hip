// 4-bit microscaled rows (apn_lowbit.h: the mx4 format) and the Linear layers evaluated on them:
//   quantize / dequantize   rows of a float matrix <-> codes and scales
//   linear                  Y = act(A B^T + b), A [M,K] and B [N,K] both mx4, on the block-scaled
//                           matrix instruction (exact products of the 4-bit values, f32 sums)
#include "apn_lowbit.h"

#include <algorithm>
#include <type_traits>

namespace apn {
namespace mx4 {
using namespace lb;

// 8 values to 8 nibbles; the hardware conversion divides by the (power of two) scale, rounds half
// to even and saturates at 6. byte 255: the codes are zeros (the block reads back as NaN).
__device__ __forceinline__ uint32_t quant8(const float (&v)[8], int byte) {
  const float sc = pow2_of(byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], sc, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], sc, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], sc, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], sc, 3);
  return byte == 255 ? 0u : w;
}
// one nibble's value: magnitudes 0, .5, 1, 1.5 as m / 2; 2, 3, 4, 6 as (2 + m) 2^(e - 2) -- the
// nibble's exponent and mantissa bits put into an f32 (subnormal codes 0 / 1 by the multiply)
__device__ __forceinline__ float value4(uint32_t n, float scale) {
  const uint32_t mag = n & 7u;
  const float f = mag < 2u ? 0.5f * (float)mag : __uint_as_float(((mag >> 1) + 126u) << 23 | (mag & 1u) << 22);
  return (n & 8u ? -f : f) * scale;
}

// One thread per 8 columns, 4 threads per block, as the q8 pack.
template <int T>
__global__ __launch_bounds__(256) void k_quant(const typename Elem<T>::type* __restrict__ x, uint32_t units, int K,
                                               int64_t ldx, FastDiv upr, uint8_t* __restrict__ codes,
                                               uint8_t* __restrict__ scales, int ss) {
  const uint32_t u = blockIdx.x * 256u + threadIdx.x;
  const bool live = u < units;
  const uint32_t m = div_by(min(u, units - 1), upr), cu = min(u, units - 1) - m * upr.d;
  const int c = (int)cu * 8, n = min(8, K - c);
  float v[8];
  load8<T>(x + (int64_t)m * ldx + c, n, v);
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) a = max(a, abs_bits(v[j]));
  a = max(a, (uint32_t)__shfl_xor((int)a, 1));
  a = max(a, (uint32_t)__shfl_xor((int)a, 2));
  const int byte = mx4_byte(a);
  const uint32_t w = quant8(v, byte);
  if (!live) return;
  *(uint32_t*)(codes + (int64_t)m * (4 * upr.d) + 4 * cu) = w;
  if ((cu & 3) == 0) {
    uint8_t* s = scales + (int64_t)m * ss;
    s[cu >> 2] = (uint8_t)byte;
    if (cu + 4 == upr.d)
      for (int i = (int)(cu >> 2) + 1; i < ss; ++i) s[i] = 0;
  }
}

template <int T>
__global__ __launch_bounds__(256) void k_dequant(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                 uint32_t units, int K, FastDiv upr, int ss,
                                                 typename Elem<T>::type* __restrict__ out, int64_t ldo) {
  const uint32_t u = blockIdx.x * 256u + threadIdx.x;
  if (u >= units) return;
  const uint32_t m = div_by(u, upr), cu = u - m * upr.d;
  const int c = (int)cu * 8, n = min(8, K - c);
  if (n <= 0) return;
  const uint32_t w = *(const uint32_t*)(codes + (int64_t)m * (4 * upr.d) + 4 * cu);
  const float sc = pow2_of(scales[(int64_t)m * ss + (cu >> 2)]);
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = value4((w >> (4 * j)) & 15u, sc);
  store8<T>(out + (int64_t)m * ldo + c, n, v);
}

// Y[m][n] = act(sum_k A[m][k] B[n][k] + bias[n]) on v_mfma_scale_f32_16x16x128: a lane holds the 32
// values (16 B) of k block lane / 16 of row lane % 16 and that block's scale byte. The operands are
// swapped -- the instruction's A is B's rows n -- so a lane's four results are consecutive columns of
// ONE row of Y.
struct Args {
  const uint8_t* ac;
  const uint8_t* as;
  const uint8_t* bc;
  const uint8_t* bs;
  const float* bias;
  void* out;
  int64_t M, ld_out;
  int N, nb, ss, act;   // nb: blocks of K; ss: bytes per scale row
  float slope;
};

template <int I>   // the scales are byte I of sa and sb
__device__ __forceinline__ f32x4 mma(u32x4 a, int sa, u32x4 b, int sb, f32x4 c) {
  const i32x8 A = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 B = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, I, sa, I, sb);
}

// This workgroup's tile. XCD x (workgroup b: b % 8) takes a run of tiles of its own, in groups of 8
// row tiles by all column tiles, so that its L2 sees the same operands again.
template <int RM, int RN>
__device__ __forceinline__ void tile_of(const Args& p, int64_t& m0, int& n0) {
  const int64_t tm = (p.M + RM - 1) / RM;
  const int tn = (p.N + RN - 1) / RN;
  const int64_t total = tm * tn, b = blockIdx.x, per = total / 8, rest = total % 8, x = b % 8;
  const int64_t lin = x * per + min(x, rest) + b / 8;
  const int64_t group = lin / (8 * tn), in_group = lin % (8 * tn), gm = min((int64_t)8, tm - group * 8);
  m0 = (group * 8 + in_group % gm) * RM;
  n0 = (int)(in_group / gm) * RN;
}
// The activation, by kind: none, ReLU, LeakyReLU with a slope below 1 and with any other. (A maximum
// that keeps NaN is one instruction where comparing and selecting are up to six.)
enum { NONE, RELU, LEAKY, SLOPE };
inline int act_kind(int act, float slope) {
  return !act || slope == 1.f ? NONE : slope == 0.f ? RELU : slope < 1.f ? LEAKY : SLOPE;
}
template <int ACT>
__device__ __forceinline__ float activate(float v, float slope) {
  if (ACT == RELU) return __builtin_elementwise_maximum(v, 0.f);
  if (ACT == LEAKY) return __builtin_elementwise_maximum(v, v * slope);
  if (ACT == SLOPE) return v > 0.f ? v : v * slope;
  return v;
}
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {   // act: uniform
  if (act == LEAKY) f(std::integral_constant<int, LEAKY>());
  else if (act == RELU) f(std::integral_constant<int, RELU>());
  else if (act == NONE) f(std::integral_constant<int, NONE>());
  else f(std::integral_constant<int, SLOPE>());
}
__device__ __forceinline__ f32x4 bias4(const Args& p, int n) {
  f32x4 b = {0.f, 0.f, 0.f, 0.f};
  if (p.bias) {
#pragma unroll
    for (int r = 0; r < 4; ++r) b[r] = p.bias[min(n + r, p.N - 1)];
  }
  return b;
}
template <int ACT>
__device__ __forceinline__ void finish4(const Args& p, const f32x4& v, const f32x4& bias, float (&y)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = activate<ACT>(v[r] + bias[r], p.slope);
}
// The results of TN column tiles of one row tile, four tiles at a time: 16-bit types are transposed
// over the four lanes of a row, so that lane q stores the 32 B of tile q and a row's 128 B go out
// together; floats go out as they are (64 B of a row together). All biases come before any store:
// a load waited for behind a store waits for the store too. values(t, y): the four of tile t.
template <int T, int TN, typename F>
__device__ __forceinline__ void store_row(void* out, int64_t ld_out, int64_t m, bool live, int left, int q, F values) {
  typedef typename Elem<T>::type E;
  E* o = (E*)out + m * ld_out;
#pragma unroll
  for (int g = 0; g < TN; g += 4) {
    bool whole = false;
    if constexpr (T != APN_F32) {
      whole = g + 4 <= TN && left >= 16 * g + 64;   // uniform
      if (whole) {
        typedef E e2 __attribute__((ext_vector_type(2)));
        typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
        uint32_t a[4], b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float y[4];
          values((g + j) % TN, y);
          a[j] = __builtin_bit_cast(uint32_t, e2{(E)y[0], (E)y[1]});
          b[j] = __builtin_bit_cast(uint32_t, e2{(E)y[2], (E)y[3]});
        }
        transpose4(a);
        transpose4(b);
        if (live) {
          E* d = o + 16 * (g + q);
          *(u32x4u*)d = u32x4{a[0], b[0], a[1], b[1]};
          *(u32x4u*)(d + 8) = u32x4{a[2], b[2], a[3], b[3]};
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int j = g; j < g + 4 && j < TN; ++j) {
        float y[4];
        values(j, y);
        if (live) store4<T>(o + 16 * j + 4 * q, left - 16 * j - 4 * q, y);
      }
    }
  }
}

// A row's scale bytes of steps s .. s + 3 (word i: step s + i, byte c: block c): zero behind the last
// block, whatever the padding holds ...
__device__ __forceinline__ u32x4 trim_scales(const Args& p, int s, u32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = p.nb - 4 * (s + i);
    v[i] = n >= 4 ? v[i] : n <= 0 ? 0u : v[i] & ((1u << (8 * n)) - 1u);
  }
  return v;
}
// ... and transposed: word c, byte i
__device__ __forceinline__ u32x4 by_block(u32x4 v) {
  const uint32_t a = __builtin_amdgcn_perm(v[1], v[0], 0x05010400u);
  const uint32_t b = __builtin_amdgcn_perm(v[3], v[2], 0x05010400u);
  const uint32_t d = __builtin_amdgcn_perm(v[1], v[0], 0x07030602u);
  const uint32_t e = __builtin_amdgcn_perm(v[3], v[2], 0x07030602u);
  return u32x4{__builtin_amdgcn_perm(b, a, 0x05040100u), __builtin_amdgcn_perm(b, a, 0x07060302u),
               __builtin_amdgcn_perm(e, d, 0x05040100u), __builtin_amdgcn_perm(e, d, 0x07060302u)};
}

// Tile kernel: WM x WN waves of TM x TN 16 x 16 tiles. Both operands go through LDS in fragment
// order, one step of 4 blocks (64 B of a row) at a time, double-buffered, the two steps after the
// next on their way in registers: 16-B piece (row tile, block, row), the row xor-ed with twice the block so that
// the lanes that write (4 blocks of 2 rows) and those that read (8 rows of a block) meet all bank
// groups. Scale bytes go by four steps: a thread reads 16 of one row and writes them transposed, so
// that a lane's word holds its own block's scales of the four steps and the instruction picks the
// byte. Blocks behind the last one count as zero codes of scale 2^-127; rows behind the ends are the
// last row again and are not stored.
template <int WM, int WN, int TM, int TN, int T>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_tile(Args p) {
  constexpr int THREADS = 64 * WM * WN, RM = 16 * WM * TM, RN = 16 * WN * TN, ROWS = RM + RN;
  constexpr int PIECES = ROWS * 4 / THREADS, BUF = ROWS * 4;
  static_assert(RM * 4 % THREADS == 0 && RN * 4 % THREADS == 0 && (ROWS < THREADS || ROWS % THREADS == 0) && TN <= TM,
                "whole passes");
  __shared__ u32x4 sh[2 * BUF];
  __shared__ u32x4 sc[2 * ROWS];
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
  int64_t m0;
  int n0;
  tile_of<RM, RN>(p, m0, n0);
  const int steps = (p.nb + 3) / 4;
  // Everything in the loop is read without a branch around it: from a step behind the last one the
  // last one's again, from a block behind the last one the step's first (and zeroed when stored), so
  // that no load is waited for before its own store.
  const int last = steps - 1, c = tid & 3, blocks = p.nb - 4 * last;   // a thread's block; blocks of the last step
  const uint8_t* const xrow = p.ac + m0 * (p.nb * 16);
  const uint8_t* const wrow = p.bc + (int64_t)n0 * (p.nb * 16);
  const uint32_t back = c < blocks ? 0u : 16u * c;
  uint32_t src[PIECES];
  int dst[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int row = (tid + THREADS * i) >> 2;   // (whole passes: X's rows or B's)
    const int r = row < RM ? (int)min((int64_t)row, p.M - 1 - m0) : min(row - RM, p.N - 1 - n0);
    src[i] = (uint32_t)r * (uint32_t)(p.nb * 16) + 16u * c;
    dst[i] = (row >> 4) * 64 + c * 16 + ((row & 15) ^ (2 * c));
  }
  u32x4 piece[PIECES];
  auto load_piece = [&](int s, int i) __attribute__((always_inline)) {
    const int at = min(s, last);
    piece[i] = *(const u32x4*)((THREADS * i < RM * 4 ? xrow : wrow) + (int64_t)at * 64 +
                               (src[i] - (at == last ? back : 0u)));
  };
  auto store_piece = [&](int s, int buf, int i) __attribute__((always_inline)) {
    if (s == last && blocks < 4) {
      if (c >= blocks) piece[i] = u32x4{0u, 0u, 0u, 0u};
    }
    sh[buf + dst[i]] = piece[i];
  };
  auto load = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) load_piece(s, i);
  };
  auto store = [&](int s, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) store_piece(s, buf, i);
  };
  constexpr int SR = (ROWS + THREADS - 1) / THREADS;   // scale rows of a thread
  const uint8_t* scales[SR];
#pragma unroll
  for (int r = 0; r < SR; ++r) {
    const int row = min(tid + THREADS * r, ROWS - 1);
    scales[r] = row < RM ? p.as + min(m0 + row, p.M - 1) * p.ss
                         : p.bs + (int64_t)min(n0 + row - RM, p.N - 1) * p.ss;
  }
  u32x4 sv[SR];
  auto load_scales = [&](int s) __attribute__((always_inline)) {   // of steps s .. s + 3
#pragma unroll
    for (int r = 0; r < SR; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) sv[r][i] = *(const uint32_t*)(scales[r] + min(4 * (s + i), p.ss - 4));
  };
  auto store_scales = [&](int s, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < SR; ++r) {   // bytes (step i, block c) to (block c, step i)
      u32x4 v = sv[r];
      if (4 * s + 16 > p.nb) v = trim_scales(p, s, v);
      if (ROWS >= THREADS || tid < ROWS) sc[buf + tid + THREADS * r] = by_block(v);
    }
  };
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  int sm[TM], sn[TN];
  u32x4 xf[2][TM], wf[2][TN];   // this step's fragments and the next one's
  const int frag = q * 16 + (l ^ (2 * q));
  auto fetch_part = [&](int buf, int m, u32x4 (&x)[TM], u32x4 (&w)[TN]) __attribute__((always_inline)) {
    x[m] = sh[buf + (wm * TM + m) * 64 + frag];
    if (m < TN) w[m] = sh[buf + RM * 4 + (wn * TN + m) * 64 + frag];
  };
  auto fetch_scales = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < TM; ++j) sm[j] = ((const int*)(sc + buf + (wm * TM + j) * 16 + l))[q];
#pragma unroll
    for (int j = 0; j < TN; ++j) sn[j] = ((const int*)(sc + buf + RM + (wn * TN + j) * 16 + l))[q];
  };
  load_scales(0);
  load(0);
  store_scales(0, 0);
  store(0, 0);
  load(1);
  __syncthreads();
#pragma unroll
  for (int m = 0; m < TM; ++m) fetch_part(0, m, xf[0], wf[0]);
  fetch_scales(0);
  store(1, BUF);
  load(2);
  int sbuf = 0;
  // Step s multiplies the fragments in registers; meanwhile the fragments of s + 1 come from the
  // buffer that the barrier has just closed, the pieces of s + 2 go into the other one (whose
  // fragments every wave took before the barrier) and those of s + 3 set out.
  for (int s = 0; s < steps; s += 4) {
    auto turn = [&](auto I) __attribute__((always_inline)) {
      constexpr int i = decltype(I)::value;
      if (i && s + i >= steps) return;
      __syncthreads();
      if (i == 0) load_scales(s + 4);
      if (i == 2) store_scales(s + 4, sbuf ^ ROWS);
      // in TM parts, each with its products first in line: a wave issues in order, so a wait for a
      // piece must not stand before them
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        fetch_part((i & 1) ? 0 : BUF, m, xf[(i & 1) ^ 1], wf[(i & 1) ^ 1]);
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = mma<i>(wf[i & 1][n], sn[n], xf[i & 1][m], sm[m], acc[m][n]);
        constexpr int PP = (PIECES + TM - 1) / TM;
#pragma unroll
        for (int f = m * PP; f < (m + 1) * PP && f < PIECES; ++f) {
          store_piece(s + i + 2, (i & 1) ? BUF : 0, f);
          load_piece(s + i + 3, f);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i == 3) fetch_scales(sbuf ^ ROWS);   // (behind the last step: not used)
    };
    turn(std::integral_constant<int, 0>());
    turn(std::integral_constant<int, 1>());
    turn(std::integral_constant<int, 2>());
    turn(std::integral_constant<int, 3>());
    sbuf ^= ROWS;
  }
  f32x4 bias[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) bias[j] = bias4(p, n0 + (wn * TN + j) * 16 + 4 * q);
  const int c0 = n0 + wn * TN * 16;
  with_act(p.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t m = m0 + (wm * TM + i) * 16 + l;
      store_row<T, TN>((typename Elem<T>::type*)p.out + c0, p.ld_out, m, m < p.M, p.N - c0, q,
                       [&](int t, float (&y)[4]) __attribute__((always_inline)) {
                         finish4<decltype(act)::value>(p, acc[i][t], bias[t], y);
                       });
    }
  });
}

// 256 x 256 tile for large products: 4 waves, one per SIMD, each 128 x 128 (256 accumulators), both
// operands straight from memory into LDS (no registers on the way), four buffers of one step (32 KB)
// so that three steps are on their way: a step is 0.5 us of matrix work and L2 answers in about 1 us
// (with one step on its way in registers the 8192 x 4096 x 4096 product took 150 us, with two 119; here
// 85, of which the products alone are 50, the results' stores 13 and their arithmetic 3). Bound by the
// matrix units' rate under load, the loads beside them, and an epilogue that nothing hides.
// The LDS side of such a load is lane by lane, so the lanes choose what they read: row lane / 4, and
// of its four blocks the one that lands conflict-free -- slot 4 r + (c ^ r / 4) of a 16-row tile. The
// next step's fragments come from LDS while this step's are multiplied.
__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}
// 64 lanes x W bytes from base + lane bytes to LDS byte address `to` + W lane; arrives under vmcnt
// (no register is written by the load, so nothing waits for it but the kernel's own s_waitcnt). m0
// is the compiler's, and a clobber of it is not honoured: it is put back behind the load, which reads
// it when it is issued. One wait state between m0 and its use.
template <int W>
__device__ __forceinline__ void to_lds(const uint8_t* base, uint32_t lane_bytes, uint32_t to) {
  uint32_t kept;
  if (W == 16)
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(kept)
                 : "s"(to), "v"(lane_bytes), "s"(base)
                 : "memory");
  else
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(kept)
                 : "s"(to), "v"(lane_bytes), "s"(base)
                 : "memory");
}
// at most N loads out, LDS reads done, all waves here
template <int N>
__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

constexpr int TILE256_LDS = 4 * 2 * 256 * 64 + 2 * 2 * 256 * 16;

// WIDE: rows of scales are whole 16-B pieces (K a multiple of 512) and lie on 16-B boundaries
template <int T, bool WIDE>
__global__ __launch_bounds__(256, 1) void k_tile256(Args p) {
  constexpr int R = 256, STAGE = 2 * R * 64, SCALES = 2 * R * 16;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // 4 STAGE of codes, SCALES as read, SCALES turned
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave & 1, wn = wave >> 1;
  int64_t m0;
  int n0;
  tile_of<R, R>(p, m0, n0);
  m0 = min(m0, p.M - R), n0 = min(n0, p.N - R);   // (M, N >= R) the last tiles reach back: same values twice
  const int steps = (p.nb + 3) / 4, last = steps - 1, blocks = p.nb - 4 * last;
  // a wave loads row tiles 8 wave .. 8 wave + 7 of the 32 (X's 16, then B's 16) of a step
  const int r = lane >> 2, c = (lane & 3) ^ (r >> 2);
  const uint32_t row_bytes = (uint32_t)p.nb * 16, back = c < blocks ? 0u : 16u * c;
  const bool xs_side = wave < 2;
  const int64_t row0 = (xs_side ? m0 : n0) + (wave & 1) * 128;   // the wave's first row
  const uint8_t* const base = (xs_side ? p.ac : p.bc) + row0 * row_bytes;
  const uint32_t src = (uint32_t)r * row_bytes + 16u * c;
  const uint32_t lds0 = lds_at(lds);
  auto load = [&](int s, int i) __attribute__((always_inline)) {   // (behind the last step: it again)
    const int at = min(s, last);
    to_lds<16>(base + (int64_t)at * 64 + (int64_t)i * 16 * row_bytes, src - (at == last ? back : 0u),
               lds0 + (s & 3) * STAGE + (wave * 8 + i) * 1024);
  };
  // Scales of steps s .. s + 3 as they lie in memory: 16 B of a row, 64 rows an instruction, or the
  // four words one by one (word j of all rows together)
  const uint8_t* const sbase = (xs_side ? p.as : p.bs) + row0 * p.ss;
  auto load_scales = [&](int s) __attribute__((always_inline)) {
    const uint32_t to = lds0 + 4 * STAGE;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* const b = sbase + (int64_t)i * 64 * p.ss;
      if (WIDE) {
        to_lds<16>(b + min(4 * s, p.ss - 16), (uint32_t)lane * (uint32_t)p.ss, to + (wave * 2 + i) * 1024);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          to_lds<4>(b + min(4 * (s + j), p.ss - 4), (uint32_t)lane * (uint32_t)p.ss,
                    to + j * 2048 + (wave * 2 + i) * 256);
      }
    }
  };
  // ... and as they are used: a row's words by block, byte i that of step s + i; a thread turns two rows.
  // (Every lane picking its bytes from the rows as they lie, 16 B read for 4 B used: 91 us against 85,
  // 8192 x 4096 x 4096.)
  u32x4* const turned = (u32x4*)(lds + 4 * STAGE + SCALES);
  auto raw_scales = [&](int r) __attribute__((always_inline)) {
    const uint8_t* const b = lds + 4 * STAGE;
    const int row = tid + 256 * r;
    u32x4 v;
    if (WIDE) {
      v = *(const u32x4*)(b + 16 * row);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *(const uint32_t*)(b + j * 2048 + 4 * row);
    }
    return v;
  };
  auto turn_scales = [&](int s, int r, u32x4 v) __attribute__((always_inline)) {
    v = trim_scales(p, s, v);   // (a branch here, and the step's products move behind it)
    turned[tid + 256 * r] = by_block(v);
  };
  f32x4 acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 xf[2][8], wf[2][8];
  int sm[8], sn[8];
  const int frag = (l * 4 + (q ^ (l >> 2))) * 16;
  auto fetch = [&](int s, int i, u32x4 (&x)[8], u32x4 (&w)[8]) __attribute__((always_inline)) {
    const uint8_t* b = lds + (s & 3) * STAGE + frag;
    x[i] = *(const u32x4*)(b + (wm * 8 + i) * 1024);
    w[i] = *(const u32x4*)(b + (16 + wn * 8 + i) * 1024);
  };
  auto scale_of = [&](int row) __attribute__((always_inline)) { return ((const int*)(turned + row + l))[q]; };
  // blocks of step s behind the last one: X's codes as zeros (in LDS: in registers, the compiler
  // copies the fragments around the branch in every step)
  auto clear = [&](int s) __attribute__((always_inline)) {
    const int have = p.nb - 4 * s;
    if (have < 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = tid + 256 * j, c = (at & 3) ^ ((at >> 4) & 3);   // slot 4 r + (c ^ r / 4) of a row tile
        if (c >= have) *(u32x4*)(lds + (s & 3) * STAGE + 16 * at) = u32x4{0u, 0u, 0u, 0u};
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
  };
  load_scales(0);
#pragma unroll
  for (int s = 0; s < 3; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) load(s, i);
  arrive<16>();
  turn_scales(0, 0, raw_scales(0));
  turn_scales(0, 1, raw_scales(1));
  clear(0);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    fetch(0, i, xf[0], wf[0]);
    sm[i] = scale_of((wm * 8 + i) * 16);
    sn[i] = scale_of(256 + (wn * 8 + i) * 16);
  }
  for (int s = 0; s < steps; s += 4) {
    auto turn = [&](auto I) __attribute__((always_inline)) {
      constexpr int i = decltype(I)::value;
      if (i && s + i >= steps) return;
      // Step s + i + 1 has arrived when no more are out than the last step sent: 8, and the scales
      // with step 0's. Every wave then has its fragments of the buffer that is written next.
      if (i != 1) arrive<8>();
      else arrive<WIDE ? 10 : 16>();
      if (i == 0) load_scales(s + 4);
      clear(s + i + 1);
      int next[8];
      u32x4 raw;   // (there since this turn's wait; turned, they are read behind the next one)
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        fetch(s + i + 1, m, xf[(i & 1) ^ 1], wf[(i & 1) ^ 1]);
        if (i == 2 && m % 4 == 1) raw = raw_scales(m / 4);
        if (i == 2 && m % 4 == 3) turn_scales(s + 4, m / 4, raw);
        int x_scale;
        if (i == 3) x_scale = scale_of((wm * 8 + m) * 16), next[m] = scale_of(256 + (wn * 8 + m) * 16);
#pragma unroll
        for (int n = 0; n < 8; ++n) acc[m][n] = mma<i>(wf[i & 1][n], sn[n], xf[i & 1][m], sm[m], acc[m][n]);
        load(s + i + 3, m);
        if (i == 3) sm[m] = x_scale;
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i == 3) {
#pragma unroll
        for (int m = 0; m < 8; ++m) sn[m] = next[m];
      }
    };
    turn(std::integral_constant<int, 0>());
    turn(std::integral_constant<int, 1>());
    turn(std::integral_constant<int, 2>());
    turn(std::integral_constant<int, 3>());
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing may land in LDS after the end
  f32x4 bias[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) bias[j] = bias4(p, n0 + (wn * 8 + j) * 16 + 4 * q);
  const int c0 = n0 + wn * 128;
  with_act(p.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      store_row<T, 8>((typename Elem<T>::type*)p.out + c0, p.ld_out, m0 + (wm * 8 + i) * 16 + l, true, p.N - c0, q,
                      [&](int t, float (&y)[4]) __attribute__((always_inline)) {
                        finish4<decltype(act)::value>(p, acc[i][t], bias[t], y);
                      });
  });
}

// Up to 16 rows: 16 columns a workgroup, K over its 8 waves -- two steps (128 B of a row of B, a
// line) at a time -- and the partial tiles joined in order. The rows come as mx4 codes (T = -1) or as
// floats, which every workgroup quantizes for itself, a panel of 64 steps at a time, into LDS. Bound
// by the latency of B's rows: all loads of a panel are in flight together.
struct FewArgs {
  Args a;            // a.ac, a.as: the rows' codes (T = -1)
  const void* x;     // the rows as floats
  int64_t ldx;
  int K;
};
constexpr int PANEL = 64;

template <int TX, int T>
__global__ __launch_bounds__(512) void k_few(FewArgs f) {
  const Args& p = f.a;
  __shared__ u32x4 rows[TX < 0 ? 1 : PANEL * 4 * 16];   // [step][block][row]
  __shared__ uint8_t rscale[TX < 0 ? 1 : PANEL * 4 * 16];
  __shared__ f32x4 red[8 * 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, M = (int)p.M;
  const int64_t n = min(n0 + l, p.N - 1);
  const uint8_t* bc = p.bc + n * p.nb * 16;
  const uint8_t* bs = p.bs + n * p.ss;
  const int64_t m = min(l, M - 1);
  const int steps = (p.nb + 3) / 4;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < steps; s0 += PANEL) {
    const int end = min(steps, s0 + PANEL);
    constexpr int U = PANEL / 8;   // a wave's steps of a panel: pairs wave, wave + 8, ..
    u32x4 w[U], x[U];
    int ws[U], xs[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int s = s0 + 2 * (wave + 8 * (i >> 1)) + (i & 1), b = min(4 * s + q, p.nb - 1);
      w[i] = *(const u32x4*)(bc + (int64_t)b * 16);
      ws[i] = bs[b];
      if (TX < 0) {
        x[i] = *(const u32x4*)(p.ac + (m * p.nb + b) * 16);
        xs[i] = p.as[m * p.ss + b];
      }
    }
    if constexpr (TX >= 0) {
      typedef typename Elem<TX>::type E;
      if (s0) __syncthreads();   // the last panel's rows are read
      const int units = (end - s0) * 16;   // 8 columns each, four a block, of each row
      for (int u = tid; u < M * units; u += 512) {   // (units is a multiple of 4: a block's threads stay together)
        const int r = u / units, c = u - r * units, k = s0 * 128 + c * 8;
        float v[8];
        load8<TX>((const E*)f.x + r * f.ldx + k, min(8, f.K - k), v);
        uint32_t a = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) a = max(a, abs_bits(v[j]));
        a = max(a, (uint32_t)__shfl_xor((int)a, 1));
        a = max(a, (uint32_t)__shfl_xor((int)a, 2));
        const int byte = mx4_byte(a);
        ((uint32_t*)rows)[((c >> 2) * 16 + r) * 4 + (c & 3)] = quant8(v, byte);
        if ((c & 3) == 0) rscale[(c >> 2) * 16 + r] = (uint8_t)byte;
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int s = s0 + 2 * (wave + 8 * (i >> 1)) + (i & 1);
      if (s >= end) continue;   // uniform in the wave
      if (TX >= 0) {
        const int at = ((s - s0) * 4 + q) * 16 + (int)m;
        x[i] = rows[at];
        xs[i] = rscale[at];
      }
      if (4 * s + q >= p.nb) w[i] = x[i] = u32x4{0u, 0u, 0u, 0u}, ws[i] = xs[i] = 0;
      acc = mma<0>(w[i], ws[i], x[i], xs[i], acc);
    }
  }
  red[wave * 64 + lane] = acc;
  __syncthreads();
  if (wave == 0 && l < M) {
    f32x4 t = red[lane];
#pragma unroll
    for (int j = 1; j < 8; ++j) t += red[64 * j + lane];
    float y[4];
    const int c = n0 + 4 * q;
    const f32x4 bias = bias4(p, c);
    with_act(p.act, [&](auto act) __attribute__((always_inline)) { finish4<decltype(act)::value>(p, t, bias, y); });
    typedef typename Elem<T>::type E;
    store4<T>((E*)p.out + l * p.ld_out + c, p.N - c, y);
  }
}

// A stack of layers on 16 rows a wave, everything between the input rows and the output in registers.
// All layers' weights (fragment order), scales and biases lie in LDS. A layer's results -- lane
// (row, q) holds columns 4 q .. 4 q + 3 of every 16 -- are quantized where they are: a 32-column block
// is 8 values of each of a row's four lanes, its codes 32 bits a lane, and four blocks transposed over
// the four lanes are the next product's operand: lane q the 16 B of block 4 s + q. The input's floats
// come in the same arrangement (four lanes on 64 B of a row), the next tile's while this one is
// computed. 262144 rows through 191-128-128-128-128 take 77 us (84 with f32 output), the input and output
// rows' 52 us (66) at a copy's rate; half of the cycles are vector instructions (1280 a tile; with
// compares and selects for the activations 95 us), the rest mostly waits for rows, of which the registers
// leave few on their way.
struct NetLayer {
  const uint8_t* codes;
  const uint8_t* scales;
  const float* bias;
  int N, nb, ss;
  float slope, floor;   // activation: risen()
  int at;   // byte offset of its LDS part: codes [column tile][step][lane] 16 B, scales [tile][lane], biases
};
constexpr int NET_DEPTH = 8, NET_COLS = 256;
struct NetArgs {
  NetLayer layer[NET_DEPTH];
  const void* x;
  void* out;
  int64_t M, ldx, ld_out;
  int depth, K, bytes;
};
// LDS bytes of a layer: column tiles of 16, padded to whole blocks of 32 columns
inline int net_bytes(int N, int nb) {
  const int tiles = (N + 31) / 32 * 2;
  return tiles * (((nb + 3) / 4) * 1024 + 256 + 64);
}

// Any activation of slope at most 1 without a branch: ReLU has slope 0 and floor 0 (which also takes
// the place of 0 x infinity), LeakyReLU and none (slope 1) floor -infinity.
__device__ __forceinline__ float risen(float v, const NetLayer& y) {
  return __builtin_elementwise_maximum(v, fmaxf(v * y.slope, y.floor));
}
// A lane has 8 values of each of four blocks (columns 4 q .. and 16 + 4 q ..): the largest magnitude of
// one block's (NaN if there is one) ...
__device__ __forceinline__ uint32_t max8(const float (&v)[8]) {
  float a = fabsf(v[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) a = __builtin_elementwise_maximum(a, fabsf(v[j]));
  return abs_bits(a);
}
// ... of block q over the row's four lanes, of all four at once ...
__device__ __forceinline__ uint32_t group_max(const uint32_t (&a)[4]) {
  const auto s = __builtin_amdgcn_permlane32_swap(a[0], a[2], false, false);
  const auto t = __builtin_amdgcn_permlane32_swap(a[1], a[3], false, false);
  const auto u = __builtin_amdgcn_permlane16_swap(max(s[0], s[1]), max(t[0], t[1]), false, false);
  return max(u[0], u[1]);
}
// ... the four scale bytes, block q's in lane q, in every lane ...
__device__ __forceinline__ uint32_t all_bytes(int byte, int q) {
  const uint32_t w = (uint32_t)byte << (8 * q);
  const auto s = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  const uint32_t v = s[0] | s[1];
  const auto t = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return t[0] | t[1];
}
// ... and block k's codes (of a block that is not finite any: its scale says so)
__device__ __forceinline__ uint32_t quant8_of(const float (&v)[8], uint32_t bytes, int k) {
  const float sc = __uint_as_float(max((bytes >> (8 * k) & 0xffu) << 23, 0x00400000u));
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], sc, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], sc, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], sc, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], sc, 3);
}
// four blocks' nibbles as the operand of a step: lane q's block, its columns in order
__device__ __forceinline__ u32x4 to_operand(uint32_t (&r)[4]) {
  transpose4(r);   // r[p]: columns 4 p .. (lower half) and 16 + 4 p .. (upper half) of the lane's block
  return u32x4{__builtin_amdgcn_perm(r[1], r[0], 0x05040100u), __builtin_amdgcn_perm(r[3], r[2], 0x05040100u),
               __builtin_amdgcn_perm(r[1], r[0], 0x07060302u), __builtin_amdgcn_perm(r[3], r[2], 0x07060302u)};
}

// KB: blocks of the input's columns at most; NT: column tiles of any layer at most; SW waves
template <int TX, int T, int KB, int NT, int SW>
__global__ __launch_bounds__(64 * SW, SW / 4) void k_network(NetArgs f) {
  extern __shared__ __attribute__((aligned(16))) uint8_t net_lds[];
  constexpr int STEPS = (KB > NT / 2 ? KB + 3 : NT / 2 + 3) / 4;
  typedef typename Elem<TX>::type E;
  typedef E quad __attribute__((ext_vector_type(4), aligned(sizeof(E))));
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t tiles = (f.M + 15) / 16, stride = (int64_t)gridDim.x * SW;
  quad x[KB][2];
  const int last = (f.K - 1) / 32, whole = f.K % 32 == 0;
  // (the tile's first row in scalar registers, the lane's row and quad as 32-bit offsets)
  uint32_t row = 0, quad_at = 4 * q;
  auto load = [&](int64_t tile, int b) __attribute__((always_inline)) {
    const E* in = (const E*)f.x + tile * 16 * f.ldx;
    if (b == 0) row = (uint32_t)min((int64_t)l, f.M - 1 - tile * 16) * (uint32_t)f.ldx;
    if (b < last || whole) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        x[b][i] = *(const quad*)((const char*)(in + 32 * b + 16 * i) + (row + quad_at) * (uint32_t)sizeof(E));
    } else {   // the last, short block: element by element, the row's last one behind its end
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t c = min(32 * b + 16 * i + quad_at + j, (uint32_t)f.K - 1);
          x[b][i][j] = *(const E*)((const char*)in + (row + c) * (uint32_t)sizeof(E));
        }
    }
  };
  int64_t tile = blockIdx.x + (int64_t)wave * gridDim.x;
  if (tile < tiles) {
#pragma unroll
    for (int b = 0; b < KB; ++b)
      if (b <= last) load(tile, b);
  }
  for (int d = 0; d < f.depth; ++d) {
    const NetLayer& y = f.layer[d];
    const int nt = (y.N + 31) / 32 * 2, steps = (y.nb + 3) / 4;
    u32x4* codes = (u32x4*)(net_lds + y.at);
    uint32_t* scales = (uint32_t*)(codes + nt * steps * 64);
    float* bias = (float*)(scales + nt * 64);
    for (int i = tid; i < nt * steps * 64; i += 64 * SW) {
      const int ln = i & 63, s = (i >> 6) % steps, n = (i >> 6) / steps * 16 + (ln & 15), b = 4 * s + (ln >> 4);
      const u32x4 w = *(const u32x4*)(y.codes + ((int64_t)min(n, y.N - 1) * y.nb + min(b, y.nb - 1)) * 16);
      codes[i] = n < y.N && b < y.nb ? w : u32x4{0u, 0u, 0u, 0u};
    }
    for (int i = tid; i < nt * 64; i += 64 * SW) {   // byte s: step s
      const int n = (i >> 6) * 16 + (i & 15), k = (i & 63) >> 4;
      uint32_t w = 0;
      for (int s = 0; s < steps; ++s)
        if (n < y.N && 4 * s + k < y.nb) w |= (uint32_t)y.scales[(int64_t)n * y.ss + 4 * s + k] << (8 * s);
      scales[i] = w;
    }
    for (int i = tid; i < nt * 16; i += 64 * SW) bias[i] = y.bias && i < y.N ? y.bias[i] : 0.f;
  }
  __syncthreads();
  for (; tile < tiles; tile += stride) {
    asm volatile("" : "+v"(quad_at));   // or every block's lane offsets are kept (and spilled)
    u32x4 op[STEPS];     // the product's row operand
    uint32_t os = 0;     // its scale bytes by step
    const bool more = tile + stride < tiles;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) op[s] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int s = 0; s < (KB + 3) / 4; ++s) {   // the input
      uint32_t r[4] = {0u, 0u, 0u, 0u}, top[4] = {0u, 0u, 0u, 0u};
      auto values = [&](int b, float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)x[b][j >> 2][j & 3];
        if (b == last && !whole) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = 32 * b + 16 * (j >> 2) + 4 * q + (j & 3) < f.K ? v[j] : 0.f;
        }
      };
#pragma unroll
      for (int k = 0; k < 4 && 4 * s + k < KB; ++k)
        if (4 * s + k <= last) {
          float v[8];
          values(4 * s + k, v);
          top[k] = max8(v);
        }
      const int byte = mx4_byte(group_max(top));
      const uint32_t bytes = all_bytes(byte, q);
#pragma unroll
      for (int k = 0; k < 4 && 4 * s + k < KB; ++k)
        if (4 * s + k <= last) {
          float v[8];
          values(4 * s + k, v);
          r[k] = quant8_of(v, bytes, k);
          if (more) load(tile + stride, 4 * s + k);
          __builtin_amdgcn_sched_barrier(0);
        }
      op[s] = to_operand(r);
      os |= (uint32_t)byte << (8 * s);
    }
    for (int d = 0; d < f.depth; ++d) {
      const NetLayer& y = f.layer[d];
      const int nt = (y.N + 31) / 32 * 2, steps = (y.nb + 3) / 4;
      const u32x4* codes = (const u32x4*)(net_lds + y.at) + lane;
      const int* scales = (const int*)(net_lds + y.at + nt * steps * 1024) + lane;
      const float* bias = (const float*)(net_lds + y.at + nt * (steps * 1024 + 256)) + 4 * q;
      f32x4 acc[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (t < nt) {
          const int ws = scales[64 * t];
          f32x4 a = *(const f32x4*)(bias + 16 * t);
          a = mma<0>(codes[t * steps * 64], ws, op[0], (int)os, a);
          if (STEPS > 1 && steps > 1) a = mma<1>(codes[(t * steps + 1) * 64], ws, op[STEPS > 1 ? 1 : 0], (int)os, a);
          acc[t] = a;
        }
      if (d + 1 == f.depth) {
        const int64_t m = tile * 16 + l;
        store_row<T, NT>(f.out, f.ld_out, m, m < f.M, y.N, q, [&](int t, float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = risen(acc[t][j], y);
        });
        break;
      }
      os = 0;
#pragma unroll
      for (int s = 0; s < NT / 8; ++s) {
        uint32_t r[4] = {0u, 0u, 0u, 0u}, sb = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t = 8 * s + 2 * k;
          if (t < nt) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = risen(acc[t + (j >> 2)][j & 3], y);
            const int byte = mx4_byte(row_max(max8(v)));   // (columns behind N are zeros: zero weights and bias)
            r[k] = quant8_of(v, (uint32_t)byte, 0);
            sb |= (uint32_t)byte << (8 * k);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        op[s] = to_operand(r);
        os |= ((sb >> (8 * q)) & 0xffu) << (8 * s);
      }
    }
  }
}

inline int64_t row_piece(int64_t upr) { return std::max<int64_t>(1, ((int64_t)1 << 30) / upr); }

template <int T>
int quantize(const void* x, int64_t M, int64_t K, int64_t ldx, uint8_t* codes, uint8_t* scales, hipStream_t s) {
  typedef typename Elem<T>::type E;
  const int64_t upr = blocks_of(K) * 4, ss = scale_stride(K), piece = row_piece(upr);
  for (int64_t m = 0; m < M; m += piece) {
    const int64_t rows = std::min(piece, M - m), units = rows * upr;
    const E* p = (const E*)x + m * ldx;
    hipLaunchKernelGGL((k_quant<T>), dim3((unsigned)ceil_div(units, 256)), dim3(256), 0, s, p, (uint32_t)units, (int)K,
                       ldx, fast_div((uint32_t)upr), codes + m * upr * 4, scales + m * ss,
                       (int)ss);
  }
  return launch_status();
}

template <int T>
int dequantize(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out, int64_t ldo,
               hipStream_t s) {
  typedef typename Elem<T>::type E;
  const int64_t upr = blocks_of(K) * 4, ss = scale_stride(K), piece = row_piece(upr);
  for (int64_t m = 0; m < M; m += piece) {
    const int64_t rows = std::min(piece, M - m), units = rows * upr;
    E* p = (E*)out + m * ldo;
    hipLaunchKernelGGL((k_dequant<T>), dim3((unsigned)ceil_div(units, 256)), dim3(256), 0, s, codes + m * upr * 4,
                       scales + m * ss, (uint32_t)units, (int)K, fast_div((uint32_t)upr), (int)ss, p, ldo);
  }
  return launch_status();
}

constexpr int64_t MAX_COLS = (int64_t)1 << 20, MAX_LD = (int64_t)1 << 24;

template <int WM, int WN, int TM, int TN, int T>
int64_t tiles_of(const Args& a) {
  return ((a.M + 16 * WM * TM - 1) / (16 * WM * TM)) * ((a.N + 16 * WN * TN - 1) / (16 * WN * TN));
}
template <int WM, int WN, int TM, int TN, int T>
void launch_tile(const Args& a, hipStream_t s) {
  hipLaunchKernelGGL((k_tile<WM, WN, TM, TN, T>), dim3((unsigned)tiles_of<WM, WN, TM, TN, T>(a)), dim3(64 * WM * WN), 0,
                     s, a);
}
template <int T>
void launch_tile256(const Args& a, hipStream_t s) {
  const bool wide = a.ss % 16 == 0 && ((uintptr_t)a.as | (uintptr_t)a.bs) % 16 == 0;
  const auto kernel = wide ? k_tile256<T, true> : k_tile256<T, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles_of<2, 2, 8, 8, T>(a)), dim3(256), TILE256_LDS, s, a);
}
// Few rows of codes and a long K: k_few (1 x 4096 x 4096 7.1 us, in tiles 10.1; 16 rows 10.0 and 10.4;
// but 4 x 2048 x 2048 7.6 and 6.7). Else the largest tile that still gives half of the CUs one: 169 tiles
// of 256 x 256 (M = N = 3328, K = 4096) 38 us, as 128 x 128 50, and 121 tiles (2816) 36 and 35; 144 tiles
// of 128 x 128 (1500 x 1000 x 1500) 9.6 us, as 64 x 64 9.4, and 64 tiles (1000 x 1000 x 1000) 8.6 and 6.4.
template <int T>
void launch_linear(const Args& a, hipStream_t s) {
  if (a.M <= 16 && a.nb > 64)
    hipLaunchKernelGGL((k_few<-1, T>), dim3((unsigned)ceil_div(a.N, 16)), dim3(512), 0, s, FewArgs{a, nullptr, 0, 0});
  else if (a.N >= 256 && a.M >= 256 && tiles_of<2, 2, 8, 8, T>(a) >= 128) launch_tile256<T>(a, s);
  else if (tiles_of<2, 2, 4, 4, T>(a) >= 128) launch_tile<2, 2, 4, 4, T>(a, s);
  else launch_tile<2, 2, 2, 2, T>(a, s);
}

template <int TX>
void launch_few(const FewArgs& a, int32_t type, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div(a.a.N, 16));
  if (type == APN_F32) hipLaunchKernelGGL((k_few<TX, APN_F32>), grid, dim3(512), 0, s, a);
  else if (type == APN_BF16) hipLaunchKernelGGL((k_few<TX, APN_BF16>), grid, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((k_few<TX, APN_F16>), grid, dim3(512), 0, s, a);
}

template <int TX, int T, int KB, int NT, int SW>
void launch_net_as(const NetArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((k_network<TX, T, KB, NT, SW>), dim3((unsigned)std::min<int64_t>((a.M + 15) / 16, 256)),
                     dim3(64 * SW), a.bytes, s, a);
}
template <int TX, int T>
void launch_net(const NetArgs& a, hipStream_t s) {
  int cols = 0;
  for (int d = 0; d < a.depth; ++d) cols = std::max(cols, a.layer[d].N);
  // (feat_net's 262144 rows: 76 us, in the wide form 115)
  if (a.K <= 192 && cols <= 128) launch_net_as<TX, T, 6, 8, 16>(a, s);
  else launch_net_as<TX, T, 8, 16, 8>(a, s);
}
template <int TX>
void launch_net_in(const NetArgs& a, int32_t type, hipStream_t s) {
  if (type == APN_F32) launch_net<TX, APN_F32>(a, s);
  else if (type == APN_BF16) launch_net<TX, APN_BF16>(a, s);
  else launch_net<TX, APN_F16>(a, s);
}

}  // namespace mx4
}  // namespace apn

using namespace apn;
using namespace apn::lb;

extern "C" int apn_mx4_quantize(const void* x, int32_t type, int64_t M, int64_t K, int64_t ldx, uint8_t* codes,
                                uint8_t* scales, void* stream) {
  if (M < 0 || K < 1 || K > mx4::MAX_COLS || ldx < K || !ok_type(type)) return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!x || !codes || !scales || (uintptr_t)codes % 16 || (uintptr_t)scales % 4) return APN_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (type == APN_F32) return mx4::quantize<APN_F32>(x, M, K, ldx, codes, scales, s);
  if (type == APN_BF16) return mx4::quantize<APN_BF16>(x, M, K, ldx, codes, scales, s);
  return mx4::quantize<APN_F16>(x, M, K, ldx, codes, scales, s);
}

extern "C" int apn_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out,
                                  int32_t type, int64_t ldo, void* stream) {
  if (M < 0 || K < 1 || K > mx4::MAX_COLS || ldo < K || !ok_type(type)) return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!out || !codes || !scales || (uintptr_t)codes % 16 || (uintptr_t)scales % 4) return APN_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (type == APN_F32) return mx4::dequantize<APN_F32>(codes, scales, M, K, out, ldo, s);
  if (type == APN_BF16) return mx4::dequantize<APN_BF16>(codes, scales, M, K, out, ldo, s);
  return mx4::dequantize<APN_F16>(codes, scales, M, K, out, ldo, s);
}

extern "C" int apn_mx4_linear(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes,
                              const uint8_t* b_scales, const float* bias, int64_t M, int64_t N, int64_t K, int32_t act,
                              float slope, void* out, int32_t type, int64_t ld_out, void* stream) {
  if (M < 0 || N < 1 || K < 1 || N > mx4::MAX_COLS || K > mx4::MAX_COLS || ld_out < N || !ok_type(type))
    return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!a_codes || !a_scales || !b_codes || !b_scales || !out) return APN_ERR_ARG;
  if ((uintptr_t)a_scales % 4 || (uintptr_t)b_scales % 4) return APN_ERR_ARG;
  if ((uintptr_t)a_codes % 16 || (uintptr_t)b_codes % 16) return APN_ERR_ARG;
  // rows per launch: fewer than 2^24 tiles of 64 x 64 (a launch has at most 2^32 threads)
  const int64_t piece = std::max<int64_t>(256, ((int64_t)1 << 35) / (N + 256) / 256 * 256);
  hipStream_t s = (hipStream_t)stream;
  const int64_t row = blocks_of(K) * 16, ss = scale_stride(K);
  for (int64_t m = 0; m < M; m += piece) {
    char* o = (char*)out + m * ld_out * (type == APN_F32 ? 4 : 2);
    mx4::Args a{a_codes + m * row, a_scales + m * ss, b_codes, b_scales, bias, o, std::min(piece, M - m), ld_out,
                (int)N, (int)blocks_of(K), (int)ss, mx4::act_kind(act, slope), slope};
    if (type == APN_F32) mx4::launch_linear<APN_F32>(a, s);
    else if (type == APN_BF16) mx4::launch_linear<APN_BF16>(a, s);
    else mx4::launch_linear<APN_F16>(a, s);
  }
  return launch_status();
}

extern "C" int apn_mx4_linear_few(const void* x, int32_t x_type, int64_t ldx, const uint8_t* b_codes,
                                  const uint8_t* b_scales, const float* bias, int64_t M, int64_t N, int64_t K,
                                  int32_t act, float slope, void* out, int32_t type, int64_t ld_out, void* stream) {
  if (M < 0 || M > 16 || N < 1 || K < 1 || N > mx4::MAX_COLS || K > mx4::MAX_COLS || ldx < K || ld_out < N ||
      !ok_type(x_type) || !ok_type(type))
    return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!x || !b_codes || !b_scales || !out || (uintptr_t)b_codes % 16 || (uintptr_t)b_scales % 4) return APN_ERR_ARG;
  const mx4::FewArgs a{{nullptr, nullptr, b_codes, b_scales, bias, out, M, ld_out, (int)N, (int)blocks_of(K),
                        (int)scale_stride(K), mx4::act_kind(act, slope), slope}, x, ldx, (int)K};
  hipStream_t s = (hipStream_t)stream;
  if (x_type == APN_F32) mx4::launch_few<APN_F32>(a, type, s);
  else if (x_type == APN_BF16) mx4::launch_few<APN_BF16>(a, type, s);
  else mx4::launch_few<APN_F16>(a, type, s);
  return launch_status();
}

extern "C" size_t apn_mx4_network_lds_bytes(int32_t depth, const apn_mx4_layer* layers) {
  if (depth < 1 || depth > mx4::NET_DEPTH || !layers) return 0;
  size_t bytes = 0;
  for (int d = 0; d < depth; ++d) {
    const apn_mx4_layer& y = layers[d];
    if (y.N < 1 || y.K < 1 || y.N > mx4::NET_COLS || y.K > mx4::NET_COLS || (d && y.K != layers[d - 1].N) ||
        (y.act && !(y.slope <= 1.f)))
      return 0;
    bytes += (size_t)mx4::net_bytes((int)y.N, (int)blocks_of(y.K));
  }
  return bytes <= 160 * 1024 ? bytes : 0;
}

extern "C" int apn_mx4_network(const void* x, int32_t x_type, int64_t ldx, int64_t M, int32_t depth,
                               const apn_mx4_layer* layers, void* out, int32_t type, int64_t ld_out, void* stream) {
  const size_t bytes = apn_mx4_network_lds_bytes(depth, layers);
  if (M < 0 || bytes == 0 || !ok_type(x_type) || !ok_type(type) || ldx < layers[0].K || ld_out < layers[depth - 1].N ||
      ldx >= mx4::MAX_LD || ld_out >= mx4::MAX_LD)
    return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!x || !out) return APN_ERR_ARG;
  mx4::NetArgs a{};
  a.x = x, a.out = out, a.M = M, a.ldx = ldx, a.ld_out = ld_out, a.depth = depth, a.K = (int)layers[0].K;
  for (int d = 0; d < depth; ++d) {
    const apn_mx4_layer& y = layers[d];
    if (!y.codes || !y.scales || (uintptr_t)y.codes % 16) return APN_ERR_ARG;
    a.layer[d] = {y.codes, y.scales, y.bias, (int)y.N, (int)blocks_of(y.K), (int)scale_stride(y.K),
                  y.act ? y.slope : 1.f, y.act && y.slope == 0.f ? 0.f : -INFINITY, a.bytes};
    a.bytes += mx4::net_bytes((int)y.N, (int)blocks_of(y.K));
  }
  hipStream_t s = (hipStream_t)stream;
  if (x_type == APN_F32) mx4::launch_net_in<APN_F32>(a, type, s);
  else if (x_type == APN_BF16) mx4::launch_net_in<APN_BF16>(a, type, s);
  else mx4::launch_net_in<APN_F16>(a, type, s);
  return launch_status();
}
