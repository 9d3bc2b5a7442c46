// Narrow block formats of the Linear layers (gfx950): the 8-bit activation checkpoint (q8) and the
// 4-bit microscaled format (mx4, E2M1 elements), both in blocks of 32 consecutive columns of a row
// with one power-of-two scale 2^(byte - 127) per block (byte 255: the block held an infinity or
// NaN and reads back as NaN).
//
//   q8   code = (x > 0 ? 0 : 0x80) | q, q = min(rint(|x| / 2^s), 127): the sign bit answers
//        "was the activation's output positive" exactly, also where q rounds to 0, so the backward
//        pass takes the LeakyReLU derivative from it (slopes of 0 and above). s is the smallest
//        exponent that holds the block's largest magnitude in 7 bits after rounding. Half a step of
//        rounding: at most 2^-7 of the block's largest magnitude (the power of two costs up to one
//        bit against a free scale; it makes scaling exact and q 2^s exact in bf16, the matrix operand).
//   mx4  nibble = sign << 3 | index into {0, .5, 1, 1.5, 2, 3, 4, 6}; s = floor(log2 max|x|) - 2
//        (the OCP microscaling conversion: the largest magnitude lands in [4, 8) and saturates
//        at 6), nearest, ties to even.
#pragma once
#include "apn_common.h"

namespace apn {
namespace lb {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int BLK = 32;
inline int64_t blocks_of(int64_t k) { return (k + BLK - 1) / BLK; }
inline int64_t scale_stride(int64_t k) { return (blocks_of(k) + 3) / 4 * 4; }   // bytes per scale row

// Bits of |x|: as unsigned integers they order like the magnitudes, with inf and NaN above all
// finite ones, so an integer maximum finds the block's largest magnitude and any non-finite value.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ int q8_byte(uint32_t amax) {
  const int e = (int)((amax + 0x10000u) >> 23) - 6;   // +0x10000: the 7-bit rounding carries
  return amax >= 0x7f800000u ? 255 : min(max(e, 0), 248);
}
__device__ __forceinline__ int mx4_byte(uint32_t amax) {
  return amax >= 0x7f800000u ? 255 : max((int)(amax >> 23) - 2, 0);
}
__device__ __forceinline__ float pow2_of(int byte) {   // 2^(byte - 127)
  const uint32_t b = byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : (uint32_t)byte << 23;
  return __uint_as_float(b);
}
__device__ __forceinline__ float inv_pow2_of(int byte) {   // 2^(127 - byte); byte 255 (no scale): 0
  return byte == 255 ? 0.f : __uint_as_float((uint32_t)(254 - byte) << 23);
}
// Four q8 codes; inv = inv_pow2_of(byte). |x| inv is exact (a power of two), + 2^23 rounds it half
// to even into the low mantissa byte. With byte 255 the product is 0 or NaN: fminf makes the NaN
// 127, and the block reads back as NaN whatever the code.
__device__ __forceinline__ uint32_t q8_codes4(const float* x, float inv) {
  uint32_t t[4], s = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    t[j] = __float_as_uint(fminf(fabsf(x[j]) * inv, 127.f) + 8388608.f);
    s |= x[j] > 0.f ? 0u : 0x80u << (8 * j);
  }
  const uint32_t lo = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(t[3], t[2], 0x04000c0cu);
  return lo | hi | s;
}
__device__ __forceinline__ float q8_value(uint32_t code, float scale) {
  const float m = (float)(code & 0x7fu) * scale;
  return code & 0x80u ? -m : m;
}

// element types of the C-ABI's row inputs and outputs (apn_hip.h: APN_F32 / APN_BF16 / APN_F16)
template <int T> struct Elem;
template <> struct Elem<APN_F32> { typedef float type; };
template <> struct Elem<APN_BF16> { typedef __bf16 type; };
template <> struct Elem<APN_F16> { typedef _Float16 type; };

// x / d for 0 <= x < 2^31 by a multiply and a shift (round-up reciprocal, d < 2^31)
struct FastDiv {
  uint32_t mul, shift, d;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return FastDiv{(uint32_t)(((1ull << (31 + s)) + d - 1) / d), s, d};
}
__device__ __forceinline__ uint32_t div_by(uint32_t x, FastDiv f) {
  return (uint32_t)(((uint64_t)x * f.mul) >> (31 + f.shift));
}

// 8 consecutive elements x[0..n-1] (n <= 8) of one row as floats, zeros behind. Whole octets move in
// 16-B pieces at any element alignment (global memory takes them; the aligned(...) below says so):
// a row of 191 bf16 starts at 2-B alignment, and element by element its read-back took 52 us
// against 19 us (203 k rows).
template <typename E> struct Octet {
  typedef E type __attribute__((ext_vector_type(8), aligned(sizeof(E))));
  typedef E half __attribute__((ext_vector_type(4), aligned(sizeof(E))));
};
template <int T>
__device__ __forceinline__ void load8(const typename Elem<T>::type* x, int n, float (&v)[8]) {
  typedef typename Elem<T>::type E;
  if (n >= 8) {
    const typename Octet<E>::type a = *(const typename Octet<E>::type*)x;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)x[j] : 0.f;
  }
}
template <int T>
__device__ __forceinline__ void store8(typename Elem<T>::type* x, int n, const float (&v)[8]) {
  typedef typename Elem<T>::type E;
  if (n >= 8) {
    typename Octet<E>::type a;
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = (E)v[j];
    *(typename Octet<E>::type*)x = a;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) x[j] = (E)v[j];
  }
}
template <int T>
__device__ __forceinline__ void store4(typename Elem<T>::type* x, int n, const float* v) {
  typedef typename Elem<T>::type E;
  if (n >= 4) {
    *(typename Octet<E>::half*)x = typename Octet<E>::half{(E)v[0], (E)v[1], (E)v[2], (E)v[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) x[i] = (E)v[i];
  }
}

// r[t] of lane (row, q) to r[q] of lane (row, t), q = lane / 16: two exchanges of register halves
__device__ __forceinline__ void transpose4(uint32_t (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto s = __builtin_amdgcn_permlane32_swap(r[i], r[i + 2], false, false);
    r[i] = s[0], r[i + 2] = s[1];
  }
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const auto s = __builtin_amdgcn_permlane16_swap(r[i], r[i + 1], false, false);
    r[i] = s[0], r[i + 1] = s[1];
  }
}
// the largest of the four lanes of a row (lanes l, l + 16, l + 32, l + 48), in all of them
__device__ __forceinline__ uint32_t row_max(uint32_t a) {
  const auto s = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  a = max(s[0], s[1]);
  const auto t = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  return max(t[0], t[1]);
}

// activation of the layers' epilogue: v > 0 ? v : slope v; slope 0 (ReLU) gives +0 for -inf and keeps NaN
__device__ __forceinline__ float leaky(float v, float slope) {
  return v > 0.f ? v : (slope == 0.f ? (v != v ? v : 0.f) : v * slope);
}

inline bool ok_type(int32_t t) { return t == APN_F32 || t == APN_BF16 || t == APN_F16; }

}  // namespace lb
}  // namespace apn
