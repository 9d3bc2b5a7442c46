// 8-bit activation checkpoints of the training step's Linear layers (apn_lowbit.h: the format) and
// the products that write and read them:
//   pack / unpack      rows of a float matrix <-> codes and scales
//   linear forward     Y = act(X W^T + b), and q8(Y) written by the epilogue
//   linear backward    G = dY * (code of Y positive ? 1 : slope);  dX = G W;
//                      dW = G^T X', db = sum_m G with X' the checkpoint of X
//   IDW-sum backward   d_out = w dh, d_w = <out', dh> with out' the checkpoint of the rows
//
// f32 products on the bf16 matrix units: every f32 factor is cut (not rounded) into three bf16
// numbers hi + mid + lo whose 3 x 8 mantissa bits are its 24 exactly, and
//   x w = hi hi + (hi mid + mid hi) + (hi lo + mid mid + lo hi) + (<= 2^-21 |x w|, left out)
// (mid < 2^-7 and lo < 2^-15 of the factor; what is left out has the product's own sign, so a sum of
// products of one sign loses it in one direction) with f32 accumulation: six bf16 products, 2.5 PFLOP/s
// / 6 = 416 TFLOP/s against 157 of the f32-input MFMA. A checkpoint factor q 2^s is one exact bf16
// number, so dW takes three. Values below 2^-110 lose mantissa bits to bf16's smallest subnormal
// (2^-133, absolute). An infinity makes its row's outputs NaN (inf - inf in the cut, inf * 0 in the
// products): non-finite stays non-finite.
#include "apn_lowbit.h"

#include <algorithm>

namespace apn {
namespace q8 {
using namespace lb;

// --- pack / unpack ---------------------------------------------------------------------------
// One thread per 8 consecutive columns, 4 threads per block: the block maximum is two lane
// exchanges; 32 B (f32) in and 8 B out per thread, consecutive threads on consecutive columns.
// Bound by memory.
template <int T>
__global__ __launch_bounds__(256) void k_pack(const typename Elem<T>::type* __restrict__ x, uint32_t units, int K,
                                              int64_t ldx, FastDiv upr, uint8_t* __restrict__ codes,
                                              uint8_t* __restrict__ scales, int ss) {
  const uint32_t u = blockIdx.x * 256u + threadIdx.x;
  const bool live = u < units;
  const uint32_t m = div_by(min(u, units - 1), upr), cu = min(u, units - 1) - m * upr.d;
  const int c = (int)cu * 8;
  const int n = min(8, K - c);   // <= 0 in the padding of the last block
  float v[8];
  load8<T>(x + (int64_t)m * ldx + c, n, v);
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) a = max(a, abs_bits(v[j]));
  a = max(a, (uint32_t)__shfl_xor((int)a, 1));
  a = max(a, (uint32_t)__shfl_xor((int)a, 2));
  const int byte = q8_byte(a);
  const float inv = inv_pow2_of(byte);
  const u32x2 w = {q8_codes4(v, inv), q8_codes4(v + 4, inv)};
  if (!live) return;
  *(u32x2*)(codes + (int64_t)m * (8 * upr.d) + c) = w;
  if ((cu & 3) == 0) {
    uint8_t* s = scales + (int64_t)m * ss;
    s[cu >> 2] = (uint8_t)byte;
    if (cu + 4 == upr.d)
      for (int i = (int)(cu >> 2) + 1; i < ss; ++i) s[i] = 0;
  }
}

template <int T>
__global__ __launch_bounds__(256) void k_unpack(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                uint32_t units, int K, FastDiv upr, int ss,
                                                typename Elem<T>::type* __restrict__ out, int64_t ldo) {
  const uint32_t u = blockIdx.x * 256u + threadIdx.x;
  if (u >= units) return;
  const uint32_t m = div_by(u, upr), cu = u - m * upr.d;
  const int c = (int)cu * 8, n = min(8, K - c);
  if (n <= 0) return;
  const u32x2 w = *(const u32x2*)(codes + (int64_t)m * (8 * upr.d) + c);
  const float sc = pow2_of(scales[(int64_t)m * ss + (cu >> 2)]);
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = q8_value((w[j >> 2] >> (8 * (j & 3))) & 0xffu, sc);
  store8<T>(out + (int64_t)m * ldo + c, n, v);
}

// --- f32 products on bf16 matrix units -------------------------------------------------------

// 8 floats as three bf16 octets, cut after 8 mantissa bits each
__device__ __forceinline__ void cut3(const float (&v)[8], u32x4& hi, u32x4& mid, u32x4& lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = v[2 * j], b = v[2 * j + 1];
    const float ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u);
    const float rb = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    const float sa = ra - __uint_as_float(__float_as_uint(ra) & 0xffff0000u);
    const float sb = rb - __uint_as_float(__float_as_uint(rb) & 0xffff0000u);
    hi[j] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    mid[j] = __builtin_amdgcn_perm(__float_as_uint(rb), __float_as_uint(ra), 0x07060302u);
    lo[j] = __builtin_amdgcn_perm(__float_as_uint(sb), __float_as_uint(sa), 0x07060302u);
  }
}
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

// Rows kernel: out[m][c] = sum_r in[m][r] Wop[c][r], the forward (r = input column, c = output
// column) and dX (r = output column, c = input column, Wop = W^T, `in` masked by Y's signs). The
// matrix operands are swapped -- A = W's rows, B = the data rows -- so that a lane's results are
// columns of ONE data row (of a 32 x 32 tile 16 of its 32 columns, 8 j + 4 h + i, the other half in
// lane ^ 32; of a 16 x 16 tile 4), which makes a q8 block's maximum mostly in-lane.

struct RowArgs {
  const float* in;
  const uint8_t* mask;   // codes of Y beside `in`, or null
  const float* w;
  const float* bias;
  float* out;
  uint8_t* codes;
  uint8_t* scales;
  int64_t M, ld_in, ld_mask, ldw, ld_out, ld_codes;
  int R, C, ss, act;
  float slope;
};

// The gradient through the activation; slope 0 gives 0 whatever g holds. The output's sign is the
// input's only for slopes of 0 and above (the entry points refuse others).
__device__ __forceinline__ float masked(float g, uint32_t code, float slope) {
  return code & 0x80u ? (slope == 0.f ? 0.f : g * slope) : g;
}

template <bool Q8, int NT>
__device__ __forceinline__ void finish_rows(const RowArgs& p, int64_t m0, int c0, int l, int h,
                                            const f32x16 (&acc)[NT], const float* bias) {
  if (c0 >= p.C) return;   // uniform in the wave; bias: the 32 columns', or null
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t m = m0 + 32 * t + l;
    float y[16];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int c = c0 + 8 * (i >> 2) + 4 * h + (i & 3);
      float v = acc[t][i];
      if (bias) v += bias[8 * (i >> 2) + 4 * h + (i & 3)];
      if (p.act) v = leaky(v, p.slope);
      if (Q8) {
        v = c < p.C ? v : 0.f;
        amax = max(amax, abs_bits(v));
      }
      y[i] = v;
    }
    if (m < p.M) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = c0 + 8 * j + 4 * h;
        store4<APN_F32>(p.out + m * p.ld_out + c, p.C - c, y + 4 * j);
      }
    }
    if (Q8) {
      amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
      const int byte = q8_byte(amax);
      const float inv = inv_pow2_of(byte);
      if (m < p.M) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          *(uint32_t*)(p.codes + m * p.ld_codes + c0 + 8 * j + 4 * h) = q8_codes4(y + 4 * j, inv);
        }
        if (h == 0) {
          uint8_t* s = p.scales + m * p.ss;
          s[c0 >> 5] = (uint8_t)byte;
          if (c0 + 32 >= p.C)
            for (int i = (c0 >> 5) + 1; i < p.ss; ++i) s[i] = 0;
        }
      }
    }
  }
}

// R <= 32 KS, 16 CT columns a workgroup: the columns' weights lie cut in LDS in fragment order, and
// each of 12 waves streams its own 16 rows at a time from memory straight into fragments of the
// 16 x 16 x 32 product -- no barrier, every row cut once, and a wave's whole next tile
// (16 x 32 KS floats) on its way while this one is multiplied. The order of the reduction is free:
// lane (row, q) takes columns 4 q .. 4 q + 3 and 16 + 4 q .. of a step, so that four lanes read 64
// consecutive bytes of a row with each load, and the weights are laid out to match. (With 32-row
// tiles and each lane on 64 B of its own, every load touched 64 lines: 77 / 90 us for dX / forward
// of 203 k x 128 x 128.) A lane's results are 4 of 16 columns of one row.
// A quad of columns that reaches behind R is read as the row's last four (so R >= 4), and its
// weights move with it; weights of columns read twice or behind R are zero.
constexpr int SW = 12;   // waves of a workgroup
__device__ __forceinline__ int quad_start(int r0, int R) { return min(r0, R - 4); }
__device__ __forceinline__ bool quad_has(int r0, int j, int R) {   // whether element j is this quad's own
  const int c = quad_start(r0, R) + j;
  return c >= r0 && c < R;
}
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

// Where a tile's results go: addresses of its first row in scalar registers (out, codes, scales), the
// lane's row and quad as 32-bit byte offsets.
struct Dest {
  char* out;
  uint8_t* codes;
  uint8_t* scales;
  uint32_t out_at, codes_at, scales_at;
  bool live;   // the lane's row exists
};

// One 32-column block of 16 rows from c0 on: lane (row, q) holds columns 4 q .. and 16 + 4 q .. . The
// floats are stored; codes and scale byte are returned.
template <bool Q8>
__device__ __forceinline__ void finish_block(const RowArgs& p, const Dest& d, int c0, int q, const f32x4& v0,
                                             const f32x4& v1, const float* bias, uint32_t& k0, uint32_t& k1,
                                             int& byte) {
  const bool whole = c0 + 32 <= p.C;
  float y[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = v0[i], y[4 + i] = v1[i];
  if (Q8) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x4 b = *(const f32x4*)(bias + 16 * j + 4 * q);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[4 * j + i] += b[i];
    }
    if (p.act) {   // two loops: the ReLU's select costs one more operation
      if (p.slope == 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] <= 0.f ? 0.f : y[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] > 0.f ? y[i] : y[i] * p.slope;
      }
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = c0 + 16 * (i >> 2) + 4 * q + (i & 3) < p.C ? y[i] : 0.f;
    }
  }
  if (d.live) {
    float* o = (float*)(d.out + d.out_at) + c0;
    if (whole) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        *(typename Octet<float>::half*)(o + 16 * j) = f32x4{y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]};
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) store4<APN_F32>(o + 16 * j, p.C - c0 - 16 * j - 4 * q, y + 4 * j);
    }
  }
  if (Q8) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, abs_bits(y[i]));
    byte = q8_byte(row_max(amax));
    const float inv = inv_pow2_of(byte);
    k0 = q8_codes4(y, inv), k1 = q8_codes4(y + 4, inv);
  }
}
// Four blocks (NB of them computed) from block b0 on: transposed over the four lanes of a row, lane q
// stores block q's 32 codes, so that a row's 128 go out as one line (lane by lane as they are
// computed, 16 B of a row at a time, the stores of 203 k rows took 20 us more), and one lane the
// scale bytes, with the padding behind the last block.
template <int NB>
__device__ __forceinline__ void store_codes(const RowArgs& p, const Dest& d, int b0, int q, uint32_t (&k0)[4],
                                            uint32_t (&k1)[4], const int (&byte)[4]) {
  transpose4(k0);
  transpose4(k1);
  const int nb = (p.C + 31) / 32;
  if (!d.live) return;
  if (q < NB && b0 + q < nb) {
    uint8_t* c = d.codes + d.codes_at + (b0 + q) * 32;
    *(u32x4*)c = u32x4{k0[0], k0[1], k0[2], k0[3]};
    *(u32x4*)(c + 16) = u32x4{k1[0], k1[1], k1[2], k1[3]};
  }
  if (q == 0) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < NB; ++i) w |= b0 + i < nb ? (uint32_t)byte[i] << (8 * i) : 0u;
    uint8_t* s = d.scales + d.scales_at + b0;
    if (b0 % 4 == 0 && (NB == 4 || b0 + NB >= nb)) *(uint32_t*)s = w;   // scale rows are whole words
    else *(uint16_t*)s = (uint16_t)w;
  }
}

template <bool WT, bool MASK, bool Q8, int KS, int CT>
__global__ __launch_bounds__(64 * SW, SW / 4) void k_rows_stream(RowArgs p) {
  extern __shared__ u32x4 ws[];   // [plane][step][column tile][lane], then 16 CT biases
  constexpr int PLANE = KS * CT * 64, MG = (KS + 3) / 4;
  float* bias = (float*)(ws + 3 * PLANE);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);   // the tile's address stays in scalar registers
  const int l = lane & 15, q = lane >> 4;
  const int c0 = blockIdx.y * 16 * CT;
  const int64_t tiles = (p.M + 15) / 16, stride = (int64_t)gridDim.x * SW;
  f32x4 x[KS][2];   // [step][half of the step]
  u32x4 s[MASK ? MG : 1][2];
  // a quad is at (the tile's rows less 32 columns, in scalar registers) + lane bytes + a constant; in
  // the last step the lane part moves back by `back` where the quad reaches behind R, and stays
  // positive by the 32 columns
  const int last = (p.R - 1) / 32;
  int back[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 32 * last + 16 * i + 4 * q;
    back[i] = quad_start(r, p.R) - r;
  }
  const uint32_t out_at = (uint32_t)l * (uint32_t)p.ld_out * 4u + 16u * q;
  const uint32_t codes_at = (uint32_t)l * (uint32_t)p.ld_codes, scales_at = (uint32_t)(l * p.ss);
  uint32_t row;
  auto load = [&](int64_t tile, int ks) __attribute__((always_inline)) {
    const char* in = (const char*)(p.in + tile * 16 * p.ld_in) - 128;
    if (ks == 0) {
      row = (uint32_t)min((int64_t)l, p.M - 1 - tile * 16);
      if (MASK) {   // lane q: the 32 codes of step 4 g + q
        const uint8_t* c = p.mask + tile * 16 * p.ld_mask + row * (uint32_t)p.ld_mask;
#pragma unroll
        for (int g = 0; g < MG; ++g) {
          const u32x4* at = (const u32x4*)(c + 32 * min(4 * g + q, last));
          s[g][0] = at[0], s[g][1] = at[1];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = (ks == last ? back[i] : 0) + 4 * q + 32;   // back + 4 q >= R - 4 - 32 last - 16 > -20
      x[ks][i] =
          *(const Octet<float>::half*)(in + (uint32_t)(row * (uint32_t)p.ld_in + at) * 4u + (32 * ks + 16 * i) * 4);
    }
  };
  int64_t tile = blockIdx.x + (int64_t)wave * gridDim.x;
  if (tile < tiles) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      if (32 * ks < p.R) load(tile, ks);
  }
#pragma unroll 2
  for (int f = tid; f < PLANE; f += 64 * SW) {
    const int ln = f & 63, ct = (f >> 6) % CT, ks = (f >> 6) / CT;
    const int c = c0 + 16 * ct + (ln & 15), r = 32 * ks + 4 * (ln >> 4), cc = min(c, p.C - 1);
    float v[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = quad_start(r + 16 * i, p.R);
      if (WT) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = p.w[(int64_t)(at + j) * p.ldw + cc];
      } else {
        const f32x4 a = *(const Octet<float>::half*)(p.w + (int64_t)cc * p.ldw + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = a[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c < p.C && quad_has(r + 16 * (j >> 2), j & 3, p.R) ? v[j] : 0.f;
    u32x4 a, b, d;
    cut3(v, a, b, d);
    ws[f] = a, ws[PLANE + f] = b, ws[2 * PLANE + f] = d;
  }
  if (Q8 && tid < 16 * CT) bias[tid] = p.bias && c0 + tid < p.C ? p.bias[c0 + tid] : 0.f;
  __syncthreads();
  for (; tile < tiles; tile += stride) {
    asm volatile("" : "+v"(back[0]), "+v"(back[1]));   // or every step's lane address is kept (and spilled)
    f32x4 acc[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t code[MASK ? 4 * MG : 1][2];   // [step][half]: the quads' codes, brought to their lanes
    if (MASK) {
#pragma unroll
      for (int g = 0; g < MG; ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t r[4] = {s[g][i][0], s[g][i][1], s[g][i][2], s[g][i][3]};
          transpose4(r);
#pragma unroll
          for (int k = 0; k < 4; ++k) code[4 * g + k][i] = r[k];
        }
    }
    const bool more = tile + stride < tiles;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (32 * ks >= p.R) break;
      u32x4 xh, xm, xl;
      float v[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t k = 0;
        if (MASK) {   // a quad that moved back has its own columns' codes that many bytes up, and the
          k = code[ks][i];   // columns before them, whose weights are 0, masked (they may hold NaN)
          if (ks == last) {
            const int up = 8 * min(-back[i], 3);
            k = k << up | (0x80808080u & ((1u << up) - 1u));
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[4 * i + j] = MASK ? masked(x[ks][i][j], k >> (8 * j), p.slope) : x[ks][i][j];
      }
      cut3(v, xh, xm, xl);
      if (more) load(tile + stride, ks);
      // the next weights are read while these are multiplied; the scheduler stays within a step
      // (left alone it hoists all of them and spills)
      const u32x4* w = ws + ks * CT * 64 + lane;
#pragma unroll
      for (int t = 0; t < CT; t += 2) {
        const u32x4 wh = w[64 * t], wm = w[PLANE + 64 * t], wl = w[2 * PLANE + 64 * t];
        const u32x4 vh = w[64 * t + 64], vm = w[PLANE + 64 * t + 64], vl = w[2 * PLANE + 64 * t + 64];
        f32x4 a = acc[t], b = acc[t + 1];
        a = mma16(wl, xh, a), b = mma16(vl, xh, b), a = mma16(wh, xl, a), b = mma16(vh, xl, b);
        a = mma16(wm, xm, a), b = mma16(vm, xm, b), a = mma16(wm, xh, a), b = mma16(vm, xh, b);
        a = mma16(wh, xm, a), b = mma16(vh, xm, b), a = mma16(wh, xh, a), b = mma16(vh, xh, b);
        acc[t] = a, acc[t + 1] = b;
        if (t % 4 == 2) __builtin_amdgcn_sched_barrier(0);
      }
    }
    const int64_t m = tile * 16;
    const Dest d{(char*)(p.out + m * p.ld_out), p.codes + m * p.ld_codes, p.scales + m * p.ss, out_at, codes_at,
                 scales_at, l < p.M - m};
#pragma unroll
    for (int g = 0; g < CT / 2; g += 4) {
      constexpr int LAST = CT / 2 % 4 ? CT / 2 % 4 : 4;   // blocks of the last group
      uint32_t k0[4] = {0, 0, 0, 0}, k1[4] = {0, 0, 0, 0};
      int byte[4] = {0, 0, 0, 0};
#pragma unroll
      for (int t = g; t < g + 4 && t < CT / 2; ++t) {
        if (c0 + 32 * t < p.C)
          finish_block<Q8>(p, d, c0 + 32 * t, q, acc[2 * t], acc[2 * t + 1], bias + 32 * t, k0[t - g], k1[t - g],
                           byte[t - g]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (Q8) {
        if (g + 4 <= CT / 2) store_codes<4>(p, d, c0 / 32 + g, q, k0, k1, byte);
        else store_codes<LAST>(p, d, c0 / 32 + g, q, k0, k1, byte);
      }
    }
  }
}

// Any R: 128 rows x 128 columns a workgroup of 8 waves (64 x 32 each), rows and weights in chunks of
// 32 columns of the reduction cut once per workgroup into LDS (fragment order), the next chunk's on
// their way to registers. A thread cuts one octet of each; rows and columns behind the ends are read
// at the last one and zeroed, so that no lane branches around a load. One buffer, so that a CU holds
// two workgroups and one multiplies while the other cuts: 77 us for 20000 x 400 x 400 and 250 for dX
// of 60000 x 512 x 512; with two buffers and one workgroup a CU 85 and 290 (and 27 against 31 where
// the workgroups are few, 1000 x 512 x 512). Bound by the matrix and vector units in turn.
template <bool WT, bool MASK, bool Q8>
__global__ __launch_bounds__(512, 4) void k_rows(RowArgs p) {
  __shared__ u32x4 rsh[2 * 1536];   // (rows, weights) x [plane][step][tile of 32][half, slot]
  constexpr int PLANE = 512, SIDE = 3 * PLANE;
  __shared__ float bias[128];
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave & 1, wc = wave >> 1;
  const int64_t m0 = (int64_t)blockIdx.x * 128;
  const int c0 = blockIdx.y * 128;
  if (Q8 && tid < 128) bias[tid] = p.bias && c0 + tid < p.C ? p.bias[c0 + tid] : 0.f;   // (read behind a barrier)
  // the thread's octets: row xr, columns 8 xu .. of a chunk; weight column wcol, reduction 8 wu ..
  const int xr = tid >> 2, xu = tid & 3, wcol = WT ? tid & 127 : tid >> 2, wu = WT ? tid >> 7 : tid & 3;
  const int64_t xm = min(m0 + xr, p.M - 1);
  const float* const in = p.in + xm * p.ld_in;
  const uint8_t* const mask = MASK ? p.mask + xm * p.ld_mask : nullptr;
  const int cw = min(c0 + wcol, p.C - 1);
  const float* const w = WT ? p.w + cw : p.w + (int64_t)cw * p.ldw;
  float xv[8], wv[8];
  u32x2 xs = {0u, 0u};
  auto load = [&](int r0) __attribute__((always_inline)) {
    const int r = r0 + 8 * xu, s = r0 + 8 * wu;
    if (r0 + 32 <= p.R) {
      load8<APN_F32>(in + r, 8, xv);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {   // (the weights' zeros alone would leave inf x 0)
        const float x = in[min(r + j, p.R - 1)];
        xv[j] = r + j < p.R ? x : 0.f;
      }
    }
    if (MASK) xs = *(const u32x2*)(mask + min(r, (int)p.ld_mask - 8));
    if (!WT && r0 + 32 <= p.R) {
      load8<APN_F32>(w + s, 8, wv);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = min(s + j, p.R - 1);
        const float x = WT ? w[(int64_t)i * p.ldw] : w[i];
        wv[j] = s + j < p.R ? x : 0.f;
      }
    }
  };
  auto stage = [&](u32x4* sh) __attribute__((always_inline)) {
    // (registers of their own: in an earlier form of this loop the compiled code let the cut parts overwrite
    // an octet's elements before their use)
#pragma unroll
    for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(xv[j]), "+v"(wv[j]));
    if (MASK) {
#pragma unroll
      for (int j = 0; j < 8; ++j) xv[j] = masked(xv[j], xs[j >> 2] >> (8 * (j & 3)), p.slope);
    }
    u32x4 a, b, c;
    cut3(xv, a, b, c);
    const int x = ((xu >> 1) * 4 + (xr >> 5)) * 64 + (xu & 1) * 32 + ((xr & 31) ^ (2 * xu));
    sh[x] = a, sh[PLANE + x] = b, sh[2 * PLANE + x] = c;
    cut3(wv, a, b, c);
    const int y = SIDE + ((wu >> 1) * 4 + (wcol >> 5)) * 64 + (wu & 1) * 32 + ((wcol & 31) ^ (2 * wu));
    sh[y] = a, sh[PLANE + y] = b, sh[2 * PLANE + y] = c;
  };
  f32x16 acc[2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
  load(0);
  for (int r0 = 0; r0 < p.R; r0 += 32) {
    stage(rsh);
    __syncthreads();
    load(min(r0 + 32, (p.R - 1) / 32 * 32));
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int at = ks * 256 + h * 32 + (l ^ (2 * (2 * ks + h)));
      const u32x4* y = rsh + SIDE + at + wc * 64;
      const u32x4 wh = y[0], wm = y[PLANE], wl = y[2 * PLANE];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4* x = rsh + at + (wr * 2 + t) * 64;
        const u32x4 xh = x[0], xm = x[PLANE], xl = x[2 * PLANE];
        f32x16 a = acc[t];
        a = mma(wl, xh, a), a = mma(wh, xl, a), a = mma(wm, xm, a);   // small products first
        a = mma(wm, xh, a), a = mma(wh, xm, a), a = mma(wh, xh, a);
        acc[t] = a;
      }
    }
    __syncthreads();
  }
  finish_rows<Q8, 2>(p, m0 + 64 * wr, c0 + 32 * wc, l, h, acc, Q8 ? bias + 32 * wc : nullptr);
}

// A few rows: f32 products, bound by the latency of W. Forward: 32 columns a workgroup, 16 lanes
// each, four rows at a time (blockIdx.y).
__global__ __launch_bounds__(512) void k_few_fwd(RowArgs p) {
  __shared__ float ys[4][32];
  const int tid = threadIdx.x, c0 = blockIdx.x * 32, c = min(c0 + (tid >> 4), p.C - 1), part = tid & 15;
  const int64_t m0 = (int64_t)blockIdx.y * 4;
  const float* w = p.w + (int64_t)c * p.ldw;
  const float* x[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) x[r] = p.in + min(m0 + r, p.M - 1) * p.ld_in;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int k = 4 * part; k < p.R; k += 64) {
    if (k + 4 <= p.R) {
      const f32x4 a = *(const Octet<float>::half*)(w + k);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 b = *(const Octet<float>::half*)(x[r] + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[r] = fmaf(a[j], b[j], s[r]);
      }
    } else {
      for (int j = k; j < p.R; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = fmaf(w[j], x[r][j], s[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int d = 1; d < 16; d *= 2) s[r] += __shfl_xor(s[r], d);
    if (part == 0) ys[r][tid >> 4] = s[r];
  }
  __syncthreads();
  if (tid >= 128) return;
  const int r = tid >> 5, o = tid & 31;
  const int64_t m = m0 + r;
  float y = ys[r][o];
  if (c0 + o < p.C) {
    if (p.bias) y += p.bias[c0 + o];
    if (p.act) y = leaky(y, p.slope);
  } else {
    y = 0.f;
  }
  uint32_t a = abs_bits(y);
#pragma unroll
  for (int d = 1; d < 32; d *= 2) a = max(a, (uint32_t)__shfl_xor((int)a, d));
  const int byte = q8_byte(a);
  if (m >= p.M) return;
  if (c0 + o < p.C) p.out[m * p.ld_out + c0 + o] = y;
  const float v[4] = {y, 0.f, 0.f, 0.f};
  p.codes[m * p.ld_codes + c0 + o] = (uint8_t)q8_codes4(v, inv_pow2_of(byte));
  uint8_t* q = p.scales + m * p.ss + (c0 >> 5);
  if (o == 0) *q = (uint8_t)byte;
  else if (c0 + 32 >= p.C && (c0 >> 5) + o < p.ss) q[o] = 0;
}
// dX: 64 columns a workgroup, the reduction over its 8 waves, four rows at a time.
template <bool MASK>
__global__ __launch_bounds__(512) void k_few_dx(RowArgs p) {
  __shared__ float red[8][4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = blockIdx.x * 64 + lane, cc = min(c, p.C - 1);
  const int64_t m0 = (int64_t)blockIdx.y * 4;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int r = wave; r < p.R; r += 8) {
    const float w = p.w[(int64_t)r * p.ldw + cc];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = min(m0 + i, p.M - 1);
      const float g = p.in[m * p.ld_in + r];
      s[i] = fmaf(MASK ? masked(g, p.mask[m * p.ld_mask + r], p.slope) : g, w, s[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[wave][i][lane] = s[i];
  __syncthreads();
  if (wave < 4 && c < p.C && m0 + wave < p.M) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) t += red[j][wave][lane];
    p.out[(m0 + wave) * p.ld_out + c] = t;
  }
}

// Weight gradient: dW[n][k] = sum_m G[m][n] X'[m][k], db[n] = sum_m G[m][n], 128 x 64 KT outputs per
// workgroup of 8 waves, wave (i, j) 32 x 32 KT of them, the rows in chunks of 64 over the splits
// (blockIdx.z takes every splits-th chunk), partial sums to the workspace and added in a fixed
// order. Both operands need 8 consecutive rows m per lane: a thread reads 4 columns of 8 rows of G
// (threads 0..255) or X' (256..511) and writes the four 8-row pieces in fragment order, column
// slots xor-ed with bits 3..4 of the column so that the writing lanes (4 columns apart) meet all
// bank groups. While a chunk is multiplied the next one is cut into the other LDS buffer, a column
// per step, and the two after it are on their way.
struct DwArgs {
  const float* dy;
  const uint8_t* mask;
  const uint8_t* xc;
  const uint8_t* xs;
  float* dw;        // partial z at dw + z stride
  float* db;        // partial z at db + z stride, or null
  int64_t M, stride;
  uint32_t ld_dy, ld_mask, ld_xc;   // below 2^24: 64 rows stay within 32 bits of bytes
  int N, K, ss, splits;
  float slope;
};

__device__ __forceinline__ int slot32(int c) { return (c & 31) ^ ((c >> 3) & 3); }

// 16-B pieces of a buffer: three planes of G, one of X'
constexpr int DW_G = 3 * 1024;   // G's three planes, then X'
template <int KT> constexpr int DW_BUF = DW_G + 512 * KT;

// One thread's part of a chunk: 8 rows of 4 columns of dY and Y's codes, or of X's codes and scales
// (v[j][0]; with KT = 3 two more columns' in the upper halves: codes t[j], scale v[j][1])
struct DwRows {
  f32x4 v[8];
  uint32_t s[8], t[8];
};
struct DwAt {   // where a thread works
  int wave, l, h, cq, mo;
  uint32_t gc, mc, xc, xd;   // its first column of dY, of Y's codes, of X's codes (and of the two more)
};

// Loads of chunk ch (one behind the last: the last one's again). Columns behind the ends are read
// somewhere in the row: their results are not stored. G: this wave's side.
template <bool G, bool QUADS, bool MASK, int KT>
__device__ __forceinline__ void dw_load(const DwArgs& p, const DwAt& w, int64_t ch, int64_t chunks, DwRows& x) {
  const int64_t m0 = min(ch, chunks - 1) * 64;
  const uint32_t lim = (uint32_t)min((int64_t)63, p.M - 1 - m0);
  if (G) {
    const char* q = (const char*)p.dy + m0 * p.ld_dy * 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t row = __umul24(min((uint32_t)(8 * w.mo + j), lim), p.ld_dy);
      if (QUADS) {
        x.v[j] = *(const Octet<float>::half*)(q + (row + w.gc) * 4u);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) x.v[j][c] = *(const float*)(q + (row + min(w.gc + c, (uint32_t)p.N - 1)) * 4u);
      }
    }
    if (MASK) {
      const uint8_t* c = p.mask + m0 * p.ld_mask;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x.s[j] = *(const uint32_t*)(c + (__umul24(min((uint32_t)(8 * w.mo + j), lim), p.ld_mask) + w.mc));
    }
  } else {
    const uint8_t* c = p.xc + m0 * p.ld_xc;
    const uint8_t* s = p.xs + m0 * p.ss;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t row = min((uint32_t)(8 * w.mo + j), lim);
      x.s[j] = *(const uint32_t*)(c + (__umul24(row, p.ld_xc) + w.xc));
      x.v[j][0] = __uint_as_float((uint32_t)s[__umul24(row, (uint32_t)p.ss) + (w.xc >> 5)]);
      if (KT == 3) {
        x.t[j] = *(const uint16_t*)(c + (__umul24(row, p.ld_xc) + w.xd));
        x.v[j][1] = __uint_as_float((uint32_t)s[__umul24(row, (uint32_t)p.ss) + (w.xd >> 5)]);
      }
    }
  }
}
// byte c of 8 rows' codes with their scales as bf16 values: q 2^s is exact in the upper 16 bits; the
// signs go in pairs
__device__ __forceinline__ u32x4 dw_values(const uint32_t (&s)[8], const f32x4 (&v)[8], int c, int k) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float e = (float)((s[2 * j] >> (8 * c)) & 0x7fu) * v[2 * j][k];
    const float o = (float)((s[2 * j + 1] >> (8 * c)) & 0x7fu) * v[2 * j + 1][k];
    const uint32_t sign = __builtin_amdgcn_perm(s[2 * j + 1], s[2 * j], 0x040c000cu + 0x01000100u * c);
    r[j] = __builtin_amdgcn_perm(__float_as_uint(o), __float_as_uint(e), 0x07060302u) | (sign & 0x80008000u);
  }
  return r;
}
// Column c of the thread's four, cut, as one 8-row piece per plane (and, c < 2, of the two more)
template <bool G, int KT>
__device__ __forceinline__ void dw_stage(const DwAt& w, const DwRows& x, int c, u32x4* sh) {
  const int row = (w.mo & 1) * 32, ks = w.mo >> 1, col = (w.cq >> 3) * 64 + row + slot32(4 * w.cq + c);
  if (G) {
    float g[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = x.v[j][c];
    u32x4 a, b, d;
    cut3(g, a, b, d);
    const int s = ks * 256 + col;
    sh[s] = a, sh[1024 + s] = b, sh[2048 + s] = d;
  } else {
    u32x4* xs = sh + DW_G + ks * (128 * KT);
    xs[col] = dw_values(x.s, x.v, c, 0);
    if (KT == 3 && c < 2) xs[256 + (w.cq >> 4) * 64 + row + slot32(2 * w.cq + c)] = dw_values(x.t, x.v, c, 1);
  }
}
// One side's waves: both sides' meet the same barriers.
template <bool G, bool QUADS, bool MASK, int KT>
__device__ __forceinline__ void dw_side(const DwArgs& p, const DwAt& w, u32x4* sh, f32x16 (&acc)[KT], float (&bs)[4]) {
  const int64_t chunks = (p.M + 63) / 64, step = p.splits;
  int64_t ch = blockIdx.z;
  // rows behind the last one as zeros (X's side: as scale 2^-127, times G's zero); G masked, its
  // column sums taken; X's scale bytes as scales
  auto ready = [&](int64_t c, DwRows& x) __attribute__((always_inline)) {
    if (c >= chunks - 1) {
      const int rows = c < chunks ? (int)(p.M - c * 64) - 8 * w.mo : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j >= rows) x.v[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (G) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (MASK) x.v[j][i] = masked(x.v[j][i], x.s[j] >> (8 * i), p.slope);
          bs[i] += x.v[j][i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < KT - 1; ++i) x.v[j][i] = pow2_of((int)__float_as_uint(x.v[j][i]));
      }
    }
  };
  auto multiply = [&](const u32x4* b, int ks) __attribute__((always_inline)) {
    const int o = w.h * 32 + slot32(w.l);
    const int s = ks * 256 + (w.wave >> 1) * 64 + o;
    const u32x4* x = b + DW_G + (ks * 2 + (w.wave & 1)) * (64 * KT) + o;
    const u32x4 g[3] = {b[2048 + s], b[1024 + s], b[s]};   // small products first
    u32x4 xf[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) xf[t] = x[64 * t];
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (int t = 0; t < KT; ++t) acc[t] = mma(g[i], xf[t], acc[t]);
  };
  DwRows xa, xb;
  dw_load<G, QUADS, MASK, KT>(p, w, ch, chunks, xa);
  dw_load<G, QUADS, MASK, KT>(p, w, ch + step, chunks, xb);
  ready(ch, xa);
#pragma unroll
  for (int c = 0; c < 4; ++c) dw_stage<G, KT>(w, xa, c, sh);
  // one chunk: multiply buffer `at`, stage the next chunk (held in x) into the other buffer (behind
  // the last chunk: zeros nobody reads), with the one after it on its way
  auto turn = [&](int at, DwRows& x, DwRows& other) __attribute__((always_inline)) {
    __syncthreads();
    dw_load<G, QUADS, MASK, KT>(p, w, ch + 2 * step, chunks, other);
    ready(ch + step, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      multiply(sh + at, i);
      dw_stage<G, KT>(w, x, i, sh + (DW_BUF<KT> - at));
    }
    ch += step;
  };
  while (ch < chunks) {
    turn(0, xb, xa);
    if (ch >= chunks) break;
    turn(DW_BUF<KT>, xa, xb);
  }
}

// QUADS: N a multiple of 4, dY's columns are read in fours
template <bool QUADS, bool MASK, int KT>
__global__ __launch_bounds__(512, 2) void k_dw(DwArgs p) {
  extern __shared__ u32x4 dw_sh[];   // 2 DW_BUF
  const int tid = threadIdx.x, lane = tid & 63, n0 = blockIdx.x * 128, k0 = blockIdx.y * (64 * KT);
  DwAt w{__builtin_amdgcn_readfirstlane(tid >> 6), lane & 31, lane >> 5, tid & 31, (tid & 255) >> 5};
  const int n = n0 + 4 * w.cq, wave = w.wave, l = w.l, h = w.h, cq = w.cq, mo = w.mo;
  const bool g_side = wave < 4;
  w.gc = (uint32_t)(QUADS ? min(n, p.N - 4) : n);
  w.mc = (uint32_t)min(n, (int)p.ld_mask - 4);
  w.xc = (uint32_t)min(k0 + 4 * w.cq, (int)p.ld_xc - 4);
  w.xd = (uint32_t)min(k0 + 128 + 2 * w.cq, (int)p.ld_xc - 2);
  f32x16 acc[KT];
#pragma unroll
  for (int b = 0; b < KT; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[b][i] = 0.f;
  float bs[4] = {0.f, 0.f, 0.f, 0.f};
  if (g_side) dw_side<true, QUADS, MASK, KT>(p, w, dw_sh, acc, bs);
  else dw_side<false, QUADS, MASK, KT>(p, w, dw_sh, acc, bs);
  float* dw = p.dw + (int64_t)blockIdx.z * p.stride;
#pragma unroll
  for (int b = 0; b < KT; ++b) {
    const int k = k0 + (wave & 1) * (32 * KT) + b * 32 + l;
    if (k >= p.K) continue;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int n = n0 + (wave >> 1) * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
      if (n < p.N) dw[(int64_t)n * p.K + k] = acc[b][i];
    }
  }
  if (p.db && blockIdx.y == 0) {   // 8 row octets per column, added in a fixed order
    __syncthreads();
    float* red = (float*)dw_sh;
    if (g_side) {
#pragma unroll
      for (int c = 0; c < 4; ++c) red[mo * 128 + 4 * cq + c] = bs[c];
    }
    __syncthreads();
    if (tid < 128 && n0 + tid < p.N) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += red[j * 128 + tid];
      p.db[(int64_t)blockIdx.z * p.stride + n0 + tid] = s;
    }
  }
}

// db alone (a frozen weight under a trained bias): 64 columns a workgroup, the sums in k_dw's order
__global__ __launch_bounds__(512) void k_db(DwArgs p) {
  __shared__ float red[512];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), mo = threadIdx.x >> 6;
  float s = 0.f;
  if (c < p.N)
    for (int64_t m0 = (int64_t)blockIdx.z * 64 + 8 * mo; m0 < p.M; m0 += 64 * (int64_t)p.splits) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t m = min(m0 + j, p.M - 1);
        const float g = p.dy[m * p.ld_dy + c];
        const float v = p.mask ? masked(g, p.mask[m * p.ld_mask + c], p.slope) : g;
        s += m0 + j < p.M ? v : 0.f;
      }
    }
  red[threadIdx.x] = s;
  __syncthreads();
  if (mo == 0 && c < p.N) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) t += red[64 * j + threadIdx.x];
    p.db[(int64_t)blockIdx.z * p.stride + c] = t;
  }
}

// dw and db from their partial sums: output o (the first `split_at` of them dw's) is the sum over z
// of part[z * n + o]. 64 outputs a workgroup (256-B reads), 16 waves each every 16th split, all its
// loads in flight together, joined in order.
__global__ __launch_bounds__(1024) void k_add_splits(const float* __restrict__ part, int splits, int64_t n,
                                                     int64_t split_at, float* __restrict__ dw,
                                                     float* __restrict__ db) {
  __shared__ float red[1024];
  const int64_t o = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  float s = 0.f;
  if (o < n) {
#pragma unroll 8
    for (int z = threadIdx.x >> 6; z < splits; z += 16) s += part[(int64_t)z * n + o];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x < 64 && o < n) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) t += red[64 * j + threadIdx.x];
    if (o < split_at) dw[o] = t;
    else db[o - split_at] = t;
  }
}

// Backward of h[s] = sum_k w[s,k] out[8s+k]: one wave per sample; lane = (row k, column eighth):
// each lane walks its row's columns 4 at a time in steps of 32, so 8 lanes cover a block.
__global__ __launch_bounds__(256) void k_idw_bwd(int64_t S, int C, const float* __restrict__ w,
                                                 const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                 int64_t ldc, int ss, const float* __restrict__ dh,
                                                 float* __restrict__ d_out, float* __restrict__ d_w) {
  const int lane = threadIdx.x & 63, k = lane >> 3, q = lane & 7;
  for (int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); s < S; s += (int64_t)gridDim.x * 4) {
    const int64_t row = 8 * s + k;
    const float wk = w[row];
    float dot = 0.f;
    for (int c = 4 * q; c < C; c += 32) {
      float g[4];
      if (c + 4 <= C) {
        const f32x4 a = *(const Octet<float>::half*)(dh + s * C + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = a[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = c + j < C ? dh[s * C + c + j] : 0.f;
      }
      if (d_w) {
        const uint32_t x = *(const uint32_t*)(codes + row * ldc + c);
        const float sc = pow2_of(scales[row * ss + (c >> 5)]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < C) dot = fmaf(q8_value((x >> (8 * j)) & 0xffu, sc), g[j], dot);
      }
      if (d_out) {
        const float o[4] = {wk * g[0], wk * g[1], wk * g[2], wk * g[3]};
        store4<APN_F32>(d_out + row * C + c, C - c, o);
      }
    }
    dot += __shfl_xor(dot, 1);
    dot += __shfl_xor(dot, 2);
    dot += __shfl_xor(dot, 4);
    if (d_w && q == 0) d_w[row] = dot;
  }
}

// rows per launch of the unit kernels, so that units (and their thread indices) stay below 2^31
inline int64_t row_piece(int64_t upr) { return std::max<int64_t>(1, ((int64_t)1 << 30) / upr); }

template <int T>
int pack(const void* x, int64_t M, int64_t K, int64_t ldx, uint8_t* codes, uint8_t* scales, hipStream_t s) {
  typedef typename Elem<T>::type E;
  const int64_t upr = blocks_of(K) * 4, ss = scale_stride(K), piece = row_piece(upr);
  for (int64_t m = 0; m < M; m += piece) {
    const int64_t rows = std::min(piece, M - m), units = rows * upr;
    const E* p = (const E*)x + m * ldx;
    hipLaunchKernelGGL((k_pack<T>), dim3((unsigned)ceil_div(units, 256)), dim3(256), 0, s, p, (uint32_t)units, (int)K,
                       ldx, fast_div((uint32_t)upr), codes + m * upr * 8, scales + m * ss,
                       (int)ss);
  }
  return launch_status();
}

template <int T>
int unpack(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out, int64_t ldo, hipStream_t s) {
  typedef typename Elem<T>::type E;
  const int64_t upr = blocks_of(K) * 4, ss = scale_stride(K), piece = row_piece(upr);
  for (int64_t m = 0; m < M; m += piece) {
    const int64_t rows = std::min(piece, M - m), units = rows * upr;
    E* p = (E*)out + m * ldo;
    hipLaunchKernelGGL((k_unpack<T>), dim3((unsigned)ceil_div(units, 256)), dim3(256), 0, s, codes + m * upr * 8,
                       scales + m * ss, (uint32_t)units, (int)K, fast_div((uint32_t)upr), (int)ss, p, ldo);
  }
  return launch_status();
}

constexpr int64_t MAX_COLS = (int64_t)1 << 20;   // row widths: 32-bit column arithmetic in the kernels
constexpr int64_t MAX_LD = (int64_t)1 << 24;     // row strides: 64 rows within 32 bits of bytes

// The weight gradient's tiles are 192 columns wide where one such tile takes the place of two of 128
// (dY is read once instead of twice: 203008 x 191 x 128 53 us, with 128 72).
inline int dw_width(int64_t K) { return K > 128 && K <= 192 ? 192 : 128; }
inline int64_t dw_tiles(int64_t N, int64_t K) {
  const int64_t kw = dw_width(K);
  return ((N + 127) / 128) * ((K + kw - 1) / kw);
}
// Splits of the weight gradient: each takes c chunks of 64 rows, about 2.5 us each, one workgroup a
// CU at most; a split's partial sums are written and read once, at about 4 TB/s together. The c with
// the smallest sum of both.
inline int dw_splits(int64_t M, int64_t N, int64_t K) {
  const int64_t chunks = (M + 63) / 64, tiles = dw_tiles(N, K), most = std::max<int64_t>(1, 256 / tiles);
  const int64_t first = std::max<int64_t>(1, (chunks + most - 1) / most);
  const double per_split = 8e-6 / 4.0 * (double)(N * (K + 1));   // us
  int64_t best = first;
  double cost = 1e30;
  for (int64_t c = first; c < 4 * first + 8 && c <= chunks; ++c) {
    const double t = 2.5 * (double)c + per_split * (double)((chunks + c - 1) / c);
    if (t < cost) cost = t, best = c;
  }
  return (int)std::max<int64_t>(1, (chunks + best - 1) / best);
}

template <int KT>
void launch_dw(const DwArgs& a, dim3 grid, hipStream_t s) {
  const auto kernel = a.N % 4 ? (a.mask ? k_dw<false, true, KT> : k_dw<false, false, KT>)
                              : (a.mask ? k_dw<true, true, KT> : k_dw<true, false, KT>);
  hipLaunchKernelGGL(kernel, grid, dim3(512), 2 * DW_BUF<KT> * 16, s, a);
}

template <bool WT, bool MASK, bool Q8, int KS, int CT>
void launch_stream(const RowArgs& a, hipStream_t s) {
  const int cols = ceil_div(a.C, 16 * CT);
  const int64_t tiles = (a.M + 15) / 16;   // one workgroup a CU, at first one tile each
  hipLaunchKernelGGL((k_rows_stream<WT, MASK, Q8, KS, CT>),
                     dim3((unsigned)std::min<int64_t>(tiles, std::max(1, 256 / cols)), (unsigned)cols), dim3(64 * SW),
                     3 * KS * CT * 64 * 16 + 16 * CT * 4, s, a);
}

// Few tiles: at most one for each wave of a full launch; the columns are then split finer (64 instead
// of 128 a workgroup: 8192 x 128 x 128 8.8 us against 11.2, but 203008 rows 69 against 65 and 191 columns
// of dX 104 against 84). Few rows: 16 x 256 x 256 forward 4.9 us and dX 7.3, 15 in k_rows; 16 x 128 x 128
// 4.2 and 4.8, 6.2 and 5.5 in k_rows_stream.
constexpr int64_t FEW_TILES = SW * 256, FEW_ROWS = 16;

template <bool WT, bool MASK, bool Q8>
int launch_rows(const RowArgs& a, hipStream_t s) {
  if (a.M <= FEW_ROWS) {
    const unsigned rows = (unsigned)((a.M + 3) / 4);
    if constexpr (Q8) hipLaunchKernelGGL(k_few_fwd, dim3((unsigned)ceil_div(a.C, 32), rows), dim3(512), 0, s, a);
    else hipLaunchKernelGGL((k_few_dx<MASK>), dim3((unsigned)ceil_div(a.C, 64), rows), dim3(512), 0, s, a);
    return launch_status();
  }
  // R < 4, or rows so far apart that a tile of them passes 32 bits of bytes: the general kernel
  const bool stream = a.R >= 4 && a.R <= 192 && a.ld_in < MAX_LD && a.ld_out < MAX_LD;
  const bool few = (a.M + 15) / 16 <= FEW_TILES;
  if (stream && few && a.R <= 128) launch_stream<WT, MASK, Q8, 4, 4>(a, s);
  else if (stream && few) launch_stream<WT, MASK, Q8, 6, 4>(a, s);
  else if (stream && a.R <= 128 && a.C > 128 && a.C <= 192)
    launch_stream<WT, MASK, Q8, 4, 12>(a, s);   // rows read once, not twice (dX of 191 columns: 84 us, not 88)
  else if (stream && a.R <= 128) launch_stream<WT, MASK, Q8, 4, 8>(a, s);
  else if (stream) launch_stream<WT, MASK, Q8, 6, 8>(a, s);
  else {
    const unsigned cols = (unsigned)ceil_div(a.C, 128);
    const int64_t most = (int64_t)1 << 21;   // workgroups a launch (2^32 threads at most)
    const int64_t tiles = std::max<int64_t>(1, most / cols);
    for (int64_t m = 0; m < a.M; m += tiles * 128) {
      RowArgs b = a;
      b.M = std::min(a.M - m, tiles * 128);
      b.in += m * a.ld_in, b.out += m * a.ld_out;
      if (MASK) b.mask += m * a.ld_mask;
      if (Q8) b.codes += m * a.ld_codes, b.scales += m * a.ss;
      hipLaunchKernelGGL((k_rows<WT, MASK, Q8>), dim3((unsigned)((b.M + 127) / 128), cols), dim3(512), 0, s, b);
    }
  }
  return launch_status();
}

}  // namespace q8
}  // namespace apn

using namespace apn;
using namespace apn::lb;

extern "C" int apn_q8_pack(const void* x, int32_t type, int64_t M, int64_t K, int64_t ldx, uint8_t* codes,
                           uint8_t* scales, void* stream) {
  if (M < 0 || K < 1 || K > q8::MAX_COLS || ldx < K || !ok_type(type)) return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!x || !codes || !scales || (uintptr_t)codes % 16 || (uintptr_t)scales % 4) return APN_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (type == APN_F32) return q8::pack<APN_F32>(x, M, K, ldx, codes, scales, s);
  if (type == APN_BF16) return q8::pack<APN_BF16>(x, M, K, ldx, codes, scales, s);
  return q8::pack<APN_F16>(x, M, K, ldx, codes, scales, s);
}

extern "C" int apn_q8_unpack(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out,
                             int32_t type, int64_t ldo, void* stream) {
  if (M < 0 || K < 1 || K > q8::MAX_COLS || ldo < K || !ok_type(type)) return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!out || !codes || !scales || (uintptr_t)codes % 16 || (uintptr_t)scales % 4) return APN_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (type == APN_F32) return q8::unpack<APN_F32>(codes, scales, M, K, out, ldo, s);
  if (type == APN_BF16) return q8::unpack<APN_BF16>(codes, scales, M, K, out, ldo, s);
  return q8::unpack<APN_F16>(codes, scales, M, K, out, ldo, s);
}

extern "C" int apn_q8_linear_fwd(const float* x, int64_t ldx, const float* w, int64_t ldw, const float* bias,
                                 int64_t M, int64_t N, int64_t K, int32_t act, float slope, float* y, int64_t ldy,
                                 uint8_t* codes, uint8_t* scales, void* stream) {
  if (M < 0 || N < 1 || K < 1 || N > q8::MAX_COLS || K > q8::MAX_COLS || ldx < K || ldw < K || ldy < N)
    return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!x || !w || !y || !codes || !scales || (uintptr_t)codes % 16 || (uintptr_t)scales % 4) return APN_ERR_ARG;
  q8::RowArgs a{x,   nullptr, w, bias, y, codes, scales, M, ldx, 0, ldw, ldy, blocks_of(N) * BLK, (int)K, (int)N,
                (int)scale_stride(N), act, slope};
  return q8::launch_rows<false, false, true>(a, (hipStream_t)stream);
}

extern "C" int apn_q8_linear_bwd_dx(const float* dy, int64_t ld_dy, const uint8_t* y_codes, float slope,
                                    const float* w, int64_t ldw, int64_t M, int64_t N, int64_t K, float* dx,
                                    int64_t ld_dx, void* stream) {
  if (M < 0 || N < 1 || K < 1 || N > q8::MAX_COLS || K > q8::MAX_COLS || ld_dy < N || ldw < K || ld_dx < K)
    return APN_ERR_ARG;
  if (M == 0) return APN_OK;
  if (!dy || !w || !dx || (uintptr_t)y_codes % 16 || (y_codes && !(slope >= 0.f))) return APN_ERR_ARG;
  q8::RowArgs a{dy, y_codes, w, nullptr, dx, nullptr, nullptr, M, ld_dy, blocks_of(N) * BLK, ldw, ld_dx, 0, (int)N,
                (int)K, 0, 0, slope};
  hipStream_t s = (hipStream_t)stream;
  return y_codes ? q8::launch_rows<true, true, false>(a, s) : q8::launch_rows<true, false, false>(a, s);
}

extern "C" size_t apn_q8_linear_bwd_dw_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 1 || K < 1) return 0;
  return (size_t)q8::dw_splits(M, N, K) * (size_t)N * (size_t)(K + 1) * sizeof(float);
}

extern "C" int apn_q8_linear_bwd_dw(const float* dy, int64_t ld_dy, const uint8_t* y_codes, float slope,
                                    const uint8_t* x_codes, const uint8_t* x_scales, int64_t M, int64_t N, int64_t K,
                                    float* dw, float* db, void* workspace, void* stream) {
  if (M < 0 || N < 1 || K < 1 || N > q8::MAX_COLS || K > q8::MAX_COLS || ld_dy < N) return APN_ERR_ARG;
  if (!dw && !db) return APN_OK;
  if (M > 0 && (!dy || !workspace || (dw && (!x_codes || !x_scales)))) return APN_ERR_ARG;
  if ((uintptr_t)y_codes % 16 || (uintptr_t)x_codes % 16 || ld_dy >= q8::MAX_LD || (y_codes && !(slope >= 0.f)))
    return APN_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (M == 0) {   // no rows: zero gradients
    if (dw) APN_TRY(fill_i32((int*)dw, 0, N * K, s));
    return db ? fill_i32((int*)db, 0, N, s) : APN_OK;
  }
  const int sp = q8::dw_splits(M, N, K);
  if (!dw) K = 0;   // column sums alone: no product columns
  const int64_t n = N * K + (db ? N : 0);
  float* part = sp > 1 ? (float*)workspace : dw;   // (null with db alone and one split: not used)
  float* bpart = !db ? nullptr : sp > 1 ? part + N * K : db;
  q8::DwArgs a{dy, y_codes, x_codes, x_scales, part, bpart, M, n, (uint32_t)ld_dy, (uint32_t)(blocks_of(N) * BLK),
               (uint32_t)(blocks_of(K) * BLK), (int)N, (int)K, (int)scale_stride(K), sp, slope};
  if (!dw) {
    hipLaunchKernelGGL(q8::k_db, dim3((unsigned)ceil_div(N, 64), 1, (unsigned)sp), dim3(512), 0, s, a);
    if (sp > 1)
      hipLaunchKernelGGL(q8::k_add_splits, dim3((unsigned)ceil_div(n, 64)), dim3(1024), 0, s, part, sp, n,
                         (int64_t)0, dw, db);
    return launch_status();
  }
  const int width = q8::dw_width(K);
  const dim3 grid((unsigned)ceil_div(N, 128), (unsigned)ceil_div(K, width), (unsigned)sp);
  if (width == 192) q8::launch_dw<3>(a, grid, s);
  else q8::launch_dw<2>(a, grid, s);
  if (sp > 1)
    hipLaunchKernelGGL(q8::k_add_splits, dim3((unsigned)ceil_div(n, 64)), dim3(1024), 0, s, part, sp, n, N * K, dw,
                       db);
  return launch_status();
}

extern "C" int apn_q8_idw_sum_bwd(int64_t S, int32_t C, const float* w, const uint8_t* codes, const uint8_t* scales,
                                  const float* dh, float* d_out, float* d_w, void* stream) {
  if (S < 0 || C < 1 || C > q8::MAX_COLS) return APN_ERR_ARG;
  if (S == 0) return APN_OK;
  if (!w || !dh || (d_w && (!codes || !scales)) || (uintptr_t)codes % 16) return APN_ERR_ARG;
  hipLaunchKernelGGL(q8::k_idw_bwd, dim3((unsigned)std::min<int64_t>((S + 3) / 4, 1 << 20)), dim3(256), 0,
                     (hipStream_t)stream, S, C, w, codes,
                     scales, blocks_of(C) * BLK, (int)scale_stride(C), dh, d_out, d_w);
  return launch_status();
}
