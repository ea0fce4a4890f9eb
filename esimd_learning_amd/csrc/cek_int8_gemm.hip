// cek_int8_gemm.hip -- products of int8 codes with a scale per token and one per
// output channel, and the gated block over a merged gate/up matrix, gfx950:
//   y[m, n] = Out((f32(sum_k a[m, k] b[n, k]) sb[n]) sa[m])
//   y[m, i] = Out(act(g) u), g and u such values of b's rows i and d + i, unrounded
#include "cek_int8.h"

namespace cek {

// One 16 x 16 block of outputs per wave, operands straight from memory: 64 rows of
// a and 16 of b per workgroup.  Rows past the end repeat the last one, K values
// past the row are zeros.
template <typename T, int ACT>  // ACT < 0: the plain product
__global__ __launch_bounds__(256) void int8_simple_kernel(const uint8_t* __restrict__ a, const float* __restrict__ sa,
                                                          const uint8_t* __restrict__ b, const float* __restrict__ sb,
                                                          uint16_t* __restrict__ y, int M, int N, int K) {
  constexpr bool GLU = ACT >= 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
  const int n = blockIdx.x * 16 + r16, m0 = blockIdx.y * 64 + wave * 16;
  const uint8_t* pa = a + (size_t)min(m0 + r16, M - 1) * K;
  const uint8_t* pb = b + (size_t)min(n, N - 1) * K;
  const uint8_t* pu = pb + (size_t)(GLU ? N : 0) * K;
  i4 acc{0, 0, 0, 0}, acu{0, 0, 0, 0};
  for (int k = 16 * g; k < ((K + 63) & ~63); k += 64) {
    const bool in = k < K;
    const u4 z{0, 0, 0, 0};
    const u4 av = in ? load_u4(pa + k) : z, bv = in ? load_u4(pb + k) : z;
    acc = mfma_i8(av, bv, acc);
    if constexpr (GLU) acu = mfma_i8(av, in ? load_u4(pu + k) : z, acu);
  }
  if (n >= N) return;
  const float s0 = sb[n], s1 = GLU ? sb[N + n] : 0.f;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int m = m0 + 4 * g + v;
    if (m >= M) continue;
    float o;
    if constexpr (GLU) o = int8_glu<ACT>(acc[v], acu[v], sa[m], s0, s1);
    else o = int8_scaled(acc[v], sa[m], s0);
    y[(size_t)m * N + n] = T::from_f32(o);
  }
}

static int int8_args(const void* a, const void* sa, const void* b, const void* sb, const void* y, int64_t M, int64_t N,
                     int64_t K, int64_t rows_b, int out_dtype, const void* ws, int64_t ws_bytes) {
  if (M < 0 || N < 0 || K <= 0 || K % 16 != 0 || K > kInt8MaxK || M > (1 << 24) || rows_b > INT32_MAX) return CEK_ERR_INVALID;
  if (ws_bytes < 0 || (ws && !aligned(ws, 16))) return CEK_ERR_INVALID;
  if (out_dtype != CEK_F16 && out_dtype != CEK_BF16) return CEK_ERR_INVALID;
  if (M == 0 || N == 0) return CEK_OK;
  if (!a || !sa || !b || !sb || !y || !aligned(a, 16) || !aligned(b, 16) || !aligned(sa, 4) || !aligned(sb, 4) ||
      !aligned(y, 2))
    return CEK_ERR_INVALID;
  return CEK_OK;
}

template <int ACT>
static int launch_int8(const int8_t* a, const float* sa, const int8_t* b, const float* sb, void* y, int64_t M, int64_t N,
                       int64_t K, int out_dtype, void* ws, int64_t ws_bytes, hipStream_t st) {
  const uint8_t* ap = reinterpret_cast<const uint8_t*>(a);
  const uint8_t* bp = reinterpret_cast<const uint8_t*>(b);
  uint16_t* yp = static_cast<uint16_t*>(y);
  for (int64_t m = 0; m < M; m += 65535 * 64) {
    const int rows = (int)(M - m < 65535 * 64 ? M - m : 65535 * 64);
    const dim3 grid((unsigned)((N + 15) / 16), (unsigned)((rows + 63) / 64));
    if (out_dtype == CEK_F16)
      int8_simple_kernel<F16, ACT><<<grid, 256, 0, st>>>(ap + m * K, sa + m, bp, sb, yp + m * N, rows, (int)N, (int)K);
    else
      int8_simple_kernel<BF16, ACT><<<grid, 256, 0, st>>>(ap + m * K, sa + m, bp, sb, yp + m * N, rows, (int)N, (int)K);
  }
  return check_launch();
}

}  // namespace cek

using namespace cek;

extern "C" int64_t cek_gemm_int8_a8w8_workspace_size(int64_t M, int64_t N, int64_t K) { return 0; }
extern "C" int64_t cek_gemm_int8_a8w8_glu_workspace_size(int64_t M, int64_t d, int64_t K) { return 0; }

extern "C" int cek_gemm_int8_a8w8(const int8_t* a, const float* sa, const int8_t* b, const float* sb, void* y, int64_t M,
                                  int64_t N, int64_t K, int out_dtype, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  const int rc = int8_args(a, sa, b, sb, y, M, N, K, N, out_dtype, workspace, workspace_bytes);
  if (rc != CEK_OK || M == 0 || N == 0) return rc;
  return launch_int8<-1>(a, sa, b, sb, y, M, N, K, out_dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int cek_gemm_int8_a8w8_glu(const int8_t* a, const float* sa, const int8_t* b, const float* sb, void* y,
                                      int64_t M, int64_t d, int64_t K, int activation, int out_dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  if (activation != CEK_GELU_TANH && activation != CEK_SILU) return CEK_ERR_INVALID;
  if (d > INT32_MAX / 2) return CEK_ERR_INVALID;
  const int rc = int8_args(a, sa, b, sb, y, M, d, K, 2 * d, out_dtype, workspace, workspace_bytes);
  if (rc != CEK_OK || M == 0 || d == 0) return rc;
  return activation == CEK_SILU ? launch_int8<CEK_SILU>(a, sa, b, sb, y, M, d, K, out_dtype, workspace, workspace_bytes,
                                                        (hipStream_t)stream)
                                : launch_int8<CEK_GELU_TANH>(a, sa, b, sb, y, M, d, K, out_dtype, workspace,
                                                             workspace_bytes, (hipStream_t)stream);
}
