// 4-bit microscaled rows (apn_lowbit.h: the mx4 format) and the Linear layers evaluated on them:
//   quantize / dequantize   rows of a float matrix <-> codes and scales
//   linear                  Y = act(A B^T + b), A [M,K] and B [N,K] both mx4, on the block-scaled
//                           matrix instruction (exact products of the 4-bit values, f32 sums)
#include "apn_lowbit.h"

#include <algorithm>

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

// Y[m][n]: 32 x 32 tiles of v_mfma_scale_f32_32x32x64 (lane: row lane % 32, the 32 values -- 16 B
// -- of k block 2 s + lane / 32, and that block's scale), operands swapped as in the q8 products
// (A = B's rows n, B = the data rows m), so a lane's 16 results are 16 of 32 columns of one row.
// One wave per 32 rows x 64 columns, 4 waves on 128 rows, operands straight from memory.
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

__device__ __forceinline__ f32x16 mma(u32x4 a, int sa, u32x4 b, int sb, f32x16 c) {
  const i32x8 A = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 B = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, 0, sa, 0, sb);
}

template <int T>
__global__ __launch_bounds__(256) void k_linear(Args p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane & 31, h = lane >> 5;
  const int n0 = blockIdx.y * 64;
  for (int64_t mt = blockIdx.x; mt * 128 < p.M; mt += gridDim.x) {
    const int64_t m = mt * 128 + wave * 32 + l;
    f32x16 acc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    for (int b = h; b < p.nb + h; b += 2) {   // p.nb + h: both halves make the same number of steps
      const bool in = b < p.nb;
      u32x4 x = zero;
      int xs = 127;
      if (in && m < p.M) {
        x = *(const u32x4*)(p.ac + (m * p.nb + b) * 16);
        xs = p.as[m * p.ss + b];
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int64_t n = n0 + 32 * t + l;
        u32x4 w = zero;
        int ws = 127;
        if (in && n < p.N) {
          w = *(const u32x4*)(p.bc + (n * p.nb + b) * 16);
          ws = p.bs[n * p.ss + b];
        }
        acc[t] = mma(w, ws, x, xs, acc[t]);
      }
    }
    if (m >= p.M) continue;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int n = n0 + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3);
        float v = acc[t][i];
        if (p.bias && n < p.N) v += p.bias[n];
        y[i] = p.act ? leaky(v, p.slope) : v;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + 32 * t + 8 * j + 4 * h;
        store4<T>((typename Elem<T>::type*)p.out + m * p.ld_out + n, p.N - n, y + 4 * j);
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

constexpr int64_t MAX_COLS = (int64_t)1 << 20;

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
  mx4::Args a{a_codes, a_scales, b_codes, b_scales, bias, out, M, ld_out, (int)N, (int)blocks_of(K),
              (int)scale_stride(K), act, slope};
  const dim3 grid((unsigned)std::min<int64_t>((M + 127) / 128, 1 << 20), (unsigned)ceil_div(N, 64));
  hipStream_t s = (hipStream_t)stream;
  if (type == APN_F32) hipLaunchKernelGGL((mx4::k_linear<APN_F32>), grid, dim3(256), 0, s, a);
  else if (type == APN_BF16) hipLaunchKernelGGL((mx4::k_linear<APN_BF16>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((mx4::k_linear<APN_F16>), grid, dim3(256), 0, s, a);
  return launch_status();
}
