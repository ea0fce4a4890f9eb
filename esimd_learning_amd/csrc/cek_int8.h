// cek_int8.h -- arithmetic of the int8 path shared by its kernels: the codes of
// a row, the scaling of a product's sums, the gated block's activations.
#pragma once

#include "cek_common.h"

namespace cek {

// ---- codes -----------------------------------------------------------------
// s = max(amax / 127, 2^-126) in fp32; code = the integer nearest to x / s, ties
// to even, of the exact quotient: what a 64-bit host computes.  |x| <= amax and s
// within 2^-24 of amax / 127 put it within -127 .. 127 without a clamp.  The floor
// keeps s and 1 / s normal (a row of zeros: codes 0).  A row with a value that is
// not finite has s = NaN and codes 0, so that every product with it is NaN.
constexpr float kInt8MinScale = 0x1p-126f;

struct Int8Row {
  float s, r;  // scale, 1 / s
  bool bad;
};
// amax_bits: the largest |x| as fp32 bits (NaN above infinity above finite).
__device__ inline Int8Row int8_row(uint32_t amax_bits) {
  const bool bad = amax_bits >= 0x7F800000u;
  const float s = bad ? __uint_as_float(0x7FC00000u) : fmaxf(__uint_as_float(amax_bits) / 127.0f, kInt8MinScale);
  return Int8Row{s, 1.0f / s, bad};
}

// Codes of four values, packed.  m = x r + 1.5 2^23 in one fma holds the nearest
// integer to x r in its low bits; x r is within 2^-16 of x / s (|x / s| <= 127, r
// within 2^-24 of 1 / s), so only where x r lies within 2^-15 of a half can the
// exact quotient's nearest integer be another, and there the remainder x - c s, which
// one fma gives exactly (c 7 bits, s 24, x at most 24, and the difference is at most
// s / 2 + s 2^-16 and a multiple of the smaller last place), is doubled and compared with s.
// Three operations a value and a branch that one wave in some hundreds takes,
// where the divide takes about twelve.
__device__ inline uint32_t int8_codes4(const float (&x)[4], const Int8Row& row) {
  constexpr float kMagic = 0x1.8p23f;
  uint32_t b[4];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float m = fmaf(x[i], row.r, kMagic);
    b[i] = __float_as_uint(m);
    far = fmaxf(far, fabsf(fmaf(x[i], row.r, kMagic - m)));
  }
  if (far > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = __uint_as_float(b[i]) - kMagic;
      const float d = fmaf(-c, row.s, x[i]), d2 = 2.f * fabsf(d);
      const bool next = d2 > row.s || (d2 == row.s && (b[i] & 1));
      b[i] += next ? (d > 0.f ? 1u : 0xFFFFFFFFu) : 0u;
    }
  }
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
  return row.bad ? 0u : lo | hi;
}

// ---- products --------------------------------------------------------------
// Sums are exact in int32: |code| <= 128, so K <= 131071 keeps them below 2^31.
// They are what every kernel, tile and split of K agrees in, so outputs do not
// depend on which served a call.
constexpr int64_t kInt8MaxK = 131071;

// The sum's value: converted (rounded once above 2^24), times the channel's scale,
// times the token's.  In this order, so that a token's scale at either end of
// bf16's range meets a number of ordinary size and not the bare sum.
__device__ inline float int8_scaled(int acc, float sa, float sb) { return f32_round(f32_round((float)acc * sb) * sa); }

// C += A B^T on one 16 x 16 x 64 block, 16 codes per lane: lane l holds row l & 15
// and the same 16 K positions of A and of B; D[4 (l >> 4) + v][l & 15] is element v.
__device__ inline i4 mfma_i8(u4 a, u4 b, i4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4, a), __builtin_bit_cast(i4, b), c, 0, 0, 0);
}

// ---- the gated block's activations -----------------------------------------
// g sigmoid(z): silu has z = g, and gelu_tanh(g) = 0.5 g (1 + tanh(y)) is g
// sigmoid(2 y), y = sqrt(2 / pi) (g + 0.044715 g^3), which unlike 1 + tanh does not
// cancel for negative g.  exp(-z) by the hardware's exp2 (1 ulp), log2(e) in the
// constants: its argument's rounding is |z| 2^-24 of the result, below an output's
// step while sigmoid(z) matters.  The hardware's reciprocal (1 ulp) and a product in
// the place of the divide, which takes ten operations more (a 256 x 256 tile's
// epilogue is these operations: 4096 x 14336 x 4096 386 -> 370 us).  exp = inf far below
// zero gives -0, or NaN for g = -inf.
template <int ACT>
__device__ inline float int8_act(float g) {
  const float z = ACT == CEK_SILU ? -1.44269504089f * g : g * fmaf(g * g, -0.10294323958f, -2.302208198144f);
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z));
}
template <int ACT>
__device__ inline float int8_glu(int ag, int au, float sa, float sg, float su) {
  return f32_round(int8_act<ACT>(int8_scaled(ag, sa, sg)) * int8_scaled(au, sa, su));
}

// Two values to 16 bits, each rounded once (the compiler's packed conversion where the
// type has one).
template <typename T>
__device__ inline uint32_t int8_pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, typename T::pair));
}

template <typename T>
__device__ inline float unit_f32(u4 v, int e) { return T::to_f32((uint16_t)((e & 1) ? v[e >> 1] >> 16 : v[e >> 1] & 0xFFFF)); }

}  // namespace cek
