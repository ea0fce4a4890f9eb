// cek_kv4.h -- layout and number format of the 4-bit key/value cache, shared by
// the kernels that write, read and attend over it.
//
// The bytes of one (block, kv head), bs tokens of hd values:
//   K codes   [bs][hd / 2]          value d of a token: nibble d % 2 of byte d / 2
//   V codes   [bs / 4][hd / 4][4]   16-bit words: values 4u .. 4u + 3 of token 4t + i
//                                   are nibbles 0 .. 3 of word [t][u][i]
//   K params  [bs]                  bf16 step s (low half), bf16 centre m (high half)
//   V params  [bs]
// and a value is m + s (c - 7.5), c = 0 .. 15.  K rows are contiguous because
// the score product contracts over a row; V words hold four tokens side by side
// because the output product contracts over tokens: either way a 32-bit load
// unpacks by masks alone into the pairs an MFMA operand wants.
#pragma once

#include "cek_common.h"

namespace cek {

struct Kv4Dims {
  int64_t block_stride;  // bytes from a block to the next
  int num_blocks, n_kv, bs_log2;
};

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Inclusive sum over the lanes, by DPP: rows of 16 by shifts, then the rows' last
// lanes broadcast into the rows behind them.
#define CEK_DPP_ADD(x, ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xF, true)
__device__ inline int wave_scan_incl(int x) {
  CEK_DPP_ADD(x, 0x111, 0xF);  // row_shr 1, 2, 4, 8
  CEK_DPP_ADD(x, 0x112, 0xF);
  CEK_DPP_ADD(x, 0x114, 0xF);
  CEK_DPP_ADD(x, 0x118, 0xF);
  CEK_DPP_ADD(x, 0x142, 0xA);  // row_bcast 15 into rows 1 and 3
  CEK_DPP_ADD(x, 0x143, 0xC);  // row_bcast 31 into rows 2 and 3
  return x;
}

// Byte offsets inside one (block, head); hd / 2 bytes a token and part.
__host__ __device__ inline int kv4_v_codes(int bs, int hd) { return bs * (hd / 2); }
__host__ __device__ inline int kv4_k_params(int bs, int hd) { return bs * hd; }
__host__ __device__ inline int kv4_v_params(int bs, int hd) { return bs * hd + 4 * bs; }
__host__ __device__ inline int kv4_head_bytes(int bs, int hd) { return bs * (hd + 8); }

__device__ inline float kv4_step(uint32_t p) { return __uint_as_float(p << 16); }
__device__ inline float kv4_centre(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

// A row's parameters from its extremes.  m = bf16(lo / 2 + hi / 2), s = bf16 of
// the larger distance from m / 7.5, so that the codes reach both ends whatever
// m's rounding did; steps below 2^-100 (whose reciprocal would leave the fp32
// range) are kept as 0: such a row is its centre.  A row with a value that is
// not finite has m = NaN, s = 0: it reads as NaN throughout.
constexpr float kKv4MinStep = 0x1p-100f;
__device__ inline uint32_t kv4_params(float lo, float hi, bool finite) {
  if (!finite) return 0x7FC00000u;
  const float m = BF16::to_f32(BF16::from_f32(f32_round(0.5f * lo) + f32_round(0.5f * hi)));
  // a / 7.5 by the rounded reciprocal and one correction: the correctly rounded quotient
  const float a = fmaxf(hi - m, m - lo), q0 = a * (1.0f / 7.5f);
  uint32_t s = BF16::from_f32(fmaf(fmaf(-q0, 7.5f, a), 1.0f / 7.5f, q0));
  if (__uint_as_float(s << 16) < kKv4MinStep) s = 0;
  return s | (__float_as_uint(m) & 0xFFFF0000u);
}

// The nearest step to x, ties to even codes, all operations in fp32 and rounded
// one by one: rint((x - m) / s + 7.5), d = quant_div of the row's step.  0 .. 15
// without a clamp: |x - m| <= 7.5 s (1 + 2^-8), s being a / 7.5 to within 2^-9.  A row
// of step 0 has code 8 throughout (the caller's part).
__device__ inline float kv4_code(float x, float m, QuantDiv d) {
  const float v = x - m, q0 = v * d.r;
  return rintf(fmaf(fmaf(-q0, d.s, v), d.r, q0) + 7.5f);
}

__device__ inline float kv4_value(uint32_t code, uint32_t p) {
  return fmaf(kv4_step(p), (float)code - 7.5f, kv4_centre(p));  // the product is exact
}

// The arguments that the cache's operators share.
inline int kv4_dims(int64_t n_kv, int64_t hd, int64_t bs, int64_t num_blocks, int64_t block_stride, Kv4Dims& dm) {
  if (n_kv <= 0 || n_kv > 4096 || num_blocks <= 0 || num_blocks > INT32_MAX) return CEK_ERR_INVALID;
  if (hd != 64 && hd != 128 && hd != 256) return CEK_ERR_UNSUPPORTED;
  if (bs < 16 || bs > 256 || (bs & (bs - 1))) return CEK_ERR_UNSUPPORTED;
  if (block_stride > UINT32_MAX) return CEK_ERR_UNSUPPORTED;
  if (block_stride % 16 || block_stride < n_kv * kv4_head_bytes((int)bs, (int)hd)) return CEK_ERR_INVALID;
  dm = Kv4Dims{block_stride, (int)num_blocks, (int)n_kv, __builtin_ctzll((unsigned long long)bs)};
  return CEK_OK;
}

// CALL(64), CALL(128) or CALL(256) for the head size hd.
#define CEK_KV4_HD(CALL)             \
  do {                               \
    if (hd == 64) CALL(64);          \
    else if (hd == 128) CALL(128);   \
    else CALL(256);                  \
  } while (0)

}  // namespace cek
