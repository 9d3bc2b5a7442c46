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

// Tile kernel: WM x WN waves of TM x TN 16 x 16 tiles. Both operands go through LDS in fragment
// order, one step of 4 blocks (64 B of a row) at a time, double-buffered, the step after the next on
// its way in registers: 16-B piece (row tile, block, row), the row xor-ed with twice the block so that
// the lanes that write (4 blocks of 2 rows) and those that read (8 rows of a block) meet all bank
// groups. Scale bytes go by four steps: a thread reads 16 of one row and writes them transposed, so
// that a lane's word holds its own block's scales of the four steps and the instruction picks the
// byte. Blocks behind the last one count as zero codes of scale 2^-127; rows behind the ends are the
// last row again and are not stored.
template <int WM, int WN, int TM, int TN, int T>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_tile(Args p) {
  constexpr int THREADS = 64 * WM * WN, RM = 16 * WM * TM, RN = 16 * WN * TN, ROWS = RM + RN;
  constexpr int PIECES = ROWS * 4 / THREADS, BUF = ROWS * 4;
  static_assert(ROWS * 4 % THREADS == 0 && ROWS <= THREADS && RM % 16 == 0, "piece per thread");
  __shared__ u32x4 sh[2 * BUF];
  __shared__ u32x4 sc[2 * ROWS];
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
  // XCD x (workgroup b: b % 8) takes a run of tiles of its own, in groups of 8 row tiles by all
  // column tiles, so that its L2 sees the same operands again
  const int64_t tm = (p.M + RM - 1) / RM;
  const int tn = (p.N + RN - 1) / RN;
  const int64_t total = tm * tn, b = blockIdx.x, per = total / 8, rest = total % 8, x = b % 8;
  const int64_t lin = x * per + min(x, rest) + b / 8;
  const int64_t group = lin / (8 * tn), in_group = lin % (8 * tn), gm = min((int64_t)8, tm - group * 8);
  const int64_t m0 = (group * 8 + in_group % gm) * RM;
  const int n0 = (int)(in_group / gm) * RN;
  const int steps = (p.nb + 3) / 4;
  const uint8_t* src[PIECES];
  int dst[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int f = tid + THREADS * i, row = f >> 2, c = f & 3;
    const uint8_t* base = row < RM ? p.ac + min(m0 + row, p.M - 1) * (p.nb * 16)
                                   : p.bc + (int64_t)min(n0 + row - RM, p.N - 1) * (p.nb * 16);
    src[i] = base + c * 16;
    dst[i] = (row >> 4) * 64 + c * 16 + ((row & 15) ^ (2 * c));
  }
  const uint8_t* scales = tid < RM ? p.as + min(m0 + tid, p.M - 1) * p.ss
                                   : p.bs + (int64_t)min(n0 + tid - RM, p.N - 1) * p.ss;
  u32x4 piece[PIECES];
  auto load = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {   // a block behind the last one: the row's first instead
      const int c = (tid + THREADS * i) & 3;
      piece[i] = *(const u32x4*)(src[i] + (4 * s + c < p.nb ? s * 64 : -c * 16));
    }
  };
  auto store = [&](int s, int buf) __attribute__((always_inline)) {
    if (4 * s + 4 > p.nb) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        if (4 * s + ((tid + THREADS * i) & 3) >= p.nb) piece[i] = u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) sh[buf + dst[i]] = piece[i];
  };
  u32x4 sv;
  auto load_scales = [&](int s) __attribute__((always_inline)) {   // of steps s .. s + 3
    if (ROWS < THREADS && tid >= ROWS) return;
    if (4 * s + 16 <= p.nb) {
      __builtin_memcpy(&sv, scales + 4 * s, 16);   // (4-B aligned)
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 4 * (s + i), n = p.nb - at;
        uint32_t w = *(const uint32_t*)(scales + min(at, p.ss - 4));
        sv[i] = n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1u);
      }
    }
  };
  auto store_scales = [&](int buf) __attribute__((always_inline)) {
    if (ROWS < THREADS && tid >= ROWS) return;
    // bytes (step i, block c) to (block c, step i)
    const uint32_t a = __builtin_amdgcn_perm(sv[1], sv[0], 0x05010400u), b = __builtin_amdgcn_perm(sv[3], sv[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(sv[1], sv[0], 0x07030602u), d = __builtin_amdgcn_perm(sv[3], sv[2], 0x07030602u);
    sc[buf + tid] = u32x4{__builtin_amdgcn_perm(b, a, 0x05040100u), __builtin_amdgcn_perm(b, a, 0x07060302u),
                          __builtin_amdgcn_perm(d, c, 0x05040100u), __builtin_amdgcn_perm(d, c, 0x07060302u)};
  };
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  int sm[TM], sn[TN];
  const int frag = q * 16 + (l ^ (2 * q));
  auto multiply = [&](int buf, auto I) __attribute__((always_inline)) {
    u32x4 w[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) w[j] = sh[buf + RM * 4 + (wn * TN + j) * 64 + frag];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const u32x4 x = sh[buf + (wm * TM + i) * 64 + frag];
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mma<decltype(I)::value>(w[j], sn[j], x, sm[i], acc[i][j]);
    }
  };
  load_scales(0);
  load(0);
  store_scales(0);
  store(0, 0);
  if (steps > 1) load(1);
  int sbuf = 0;
  for (int s = 0; s < steps; s += 4) {
    auto turn = [&](auto I) __attribute__((always_inline)) {
      constexpr int i = decltype(I)::value;
      if (i && s + i >= steps) return;
      __syncthreads();
      if (i == 0) {
#pragma unroll
        for (int j = 0; j < TM; ++j) sm[j] = ((const int*)(sc + sbuf + (wm * TM + j) * 16 + l))[q];
#pragma unroll
        for (int j = 0; j < TN; ++j) sn[j] = ((const int*)(sc + sbuf + RM + (wn * TN + j) * 16 + l))[q];
        if (s + 4 < steps) load_scales(s + 4);
      }
      if (s + i + 1 < steps) store(s + i + 1, (i & 1) ? 0 : BUF);
      if (s + i + 2 < steps) load(s + i + 2);
      multiply((i & 1) ? BUF : 0, I);
      if (i == 3 && s + 4 < steps) store_scales(sbuf ^ ROWS);
    };
    turn(std::integral_constant<int, 0>());
    turn(std::integral_constant<int, 1>());
    turn(std::integral_constant<int, 2>());
    turn(std::integral_constant<int, 3>());
    sbuf ^= ROWS;
  }
  typedef typename Elem<T>::type E;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t m = m0 + (wm * TM + i) * 16 + l;
    E* o = (E*)p.out + m * p.ld_out;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + (wn * TN + j) * 16 + 4 * q;
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        y[r] = acc[i][j][r];
        if (p.bias) y[r] += p.bias[min(n + r, p.N - 1)];
        if (p.act) y[r] = leaky(y[r], p.slope);
      }
      if (m < p.M) store4<T>(o + n, p.N - n, y);
    }
  }
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
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      y[r] = t[r];
      if (p.bias) y[r] += p.bias[min(c + r, p.N - 1)];
      if (p.act) y[r] = leaky(y[r], p.slope);
    }
    typedef typename Elem<T>::type E;
    store4<T>((E*)p.out + l * p.ld_out + c, p.N - c, y);
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

constexpr int64_t MAX_COLS = (int64_t)1 << 20;

template <int WM, int WN, int TM, int TN, int T>
int64_t tiles_of(const Args& a) {
  return ((a.M + 16 * WM * TM - 1) / (16 * WM * TM)) * ((a.N + 16 * WN * TN - 1) / (16 * WN * TN));
}
template <int WM, int WN, int TM, int TN, int T>
void launch_tile(const Args& a, hipStream_t s) {
  hipLaunchKernelGGL((k_tile<WM, WN, TM, TN, T>), dim3((unsigned)tiles_of<WM, WN, TM, TN, T>(a)), dim3(64 * WM * WN), 0,
                     s, a);
}
// The largest tile that still gives most CUs one
template <int T>
void launch_linear(const Args& a, hipStream_t s) {
  if (a.M <= 16) {
    hipLaunchKernelGGL((k_few<-1, T>), dim3((unsigned)ceil_div(a.N, 16)), dim3(512), 0, s, FewArgs{a, nullptr, 0, 0});
    return;
  }
  if (tiles_of<2, 4, 8, 4, T>(a) >= 192) launch_tile<2, 4, 8, 4, T>(a, s);
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

}  // namespace mx4
}  // namespace apn

using namespace apn;
using namespace apn::lb;

extern "C" int apn_mx4_quantize(const void* x, int32_t type, int64_t M, int64_t K, int64_t ldx, uint8_t* codes,
                                uint8_t* scales, void* stream) {
  if (M < 0 || K < 1 || K > mx4::MAX_COLS || ldx < K || !ok_type(type)) return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!x || !codes || !scales || (uintptr_t)codes % 16) return APN_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (type == APN_F32) return mx4::quantize<APN_F32>(x, M, K, ldx, codes, scales, s);
  if (type == APN_BF16) return mx4::quantize<APN_BF16>(x, M, K, ldx, codes, scales, s);
  return mx4::quantize<APN_F16>(x, M, K, ldx, codes, scales, s);
}

extern "C" int apn_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out,
                                  int32_t type, int64_t ldo, void* stream) {
  if (M < 0 || K < 1 || K > mx4::MAX_COLS || ldo < K || !ok_type(type)) return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!out || !codes || !scales || (uintptr_t)codes % 16) return APN_ERR_ARG;
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
  if ((uintptr_t)a_codes % 16 || (uintptr_t)b_codes % 16) return APN_ERR_ARG;
  // rows per launch: fewer than 2^24 tiles of 64 x 64 (a launch has at most 2^32 threads)
  const int64_t piece = std::max<int64_t>(256, ((int64_t)1 << 35) / (N + 256) / 256 * 256);
  hipStream_t s = (hipStream_t)stream;
  const int64_t row = blocks_of(K) * 16, ss = scale_stride(K);
  for (int64_t m = 0; m < M; m += piece) {
    char* o = (char*)out + m * ld_out * (type == APN_F32 ? 4 : 2);
    mx4::Args a{a_codes + m * row, a_scales + m * ss, b_codes, b_scales, bias, o, std::min(piece, M - m), ld_out, (int)N,
                (int)blocks_of(K), (int)ss, act, slope};
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
  if (!x || !b_codes || !b_scales || !out || (uintptr_t)b_codes % 16) return APN_ERR_ARG;
  const mx4::FewArgs a{{nullptr, nullptr, b_codes, b_scales, bias, out, M, ld_out, (int)N, (int)blocks_of(K),
                        (int)scale_stride(K), act, slope}, x, ldx, (int)K};
  hipStream_t s = (hipStream_t)stream;
  if (x_type == APN_F32) mx4::launch_few<APN_F32>(a, type, s);
  else if (x_type == APN_BF16) mx4::launch_few<APN_BF16>(a, type, s);
  else mx4::launch_few<APN_F16>(a, type, s);
  return launch_status();
}
