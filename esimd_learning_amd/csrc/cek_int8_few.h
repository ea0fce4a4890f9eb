// cek_int8_few.h -- what the int8 kernels for a few rows of a share.
#pragma once

#include "cek_int8.h"

namespace cek {

struct Int8Few {
  const uint8_t* a;
  const float* sa;
  const uint8_t* b;
  const float* sb;
  uint16_t* y;
  int M, N, K;    // N: output columns
  int bf16, act;  // act < 0: the plain product
};

__device__ inline void int8_store(const Int8Few& p, int m, int n, int g, int u, float sa, float sg, float su) {
  const float o = p.act < 0 ? int8_scaled(g, sa, sg)
                            : (p.act == CEK_SILU ? int8_glu<CEK_SILU>(g, u, sa, sg, su) : int8_glu<CEK_GELU_TANH>(g, u, sa, sg, su));
  p.y[(size_t)m * p.N + n] = p.bf16 ? BF16::from_f32(o) : F16::from_f32(o);
}

// Sum over the 64 lanes (in lane 63's and every lane's value alike).
__device__ inline int wave_isum(int v) {
#define CEK_IDPP(c) v += __builtin_amdgcn_update_dpp(0, v, c, 0xF, 0xF, true)
  CEK_IDPP(0xB1);   // quad_perm [1,0,3,2]
  CEK_IDPP(0x4E);   // quad_perm [2,3,0,1]
  CEK_IDPP(0x141);  // row_half_mirror
  CEK_IDPP(0x140);  // row_mirror
#undef CEK_IDPP
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
         __builtin_amdgcn_readlane(v, 48);
}

// Up to 64 rows: whether these kernels serve the product rather than tiles that would take
// tile_us (NB: rows of b), and their launch.
bool int8_few_takes(int64_t M, int64_t NB, int64_t K, bool glu, double tile_us);
// Which of them serves N outputs (the codes of cek_gemm_int8_few_plan).
int int8_few_form(int64_t M, int64_t N, int64_t K, bool glu);
int launch_int8_few(const Int8Few& p, hipStream_t st);

}  // namespace cek
