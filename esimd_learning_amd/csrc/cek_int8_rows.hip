// cek_int8_rows.hip -- int8 codes and scales of rows, alone or behind the residual
// add + RMS norm, gfx950 (the arithmetic: cek_int8.h).
#include "cek_int8.h"
#include "cek_rowops.h"

namespace cek {

constexpr int kRowThreads = 256;

// Largest of a value over the workgroup (bits of non-negative floats, as integers).
__device__ inline uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, 64));
  return v;
}
template <int NT>
__device__ inline uint32_t block_umax(uint32_t v, uint32_t* sh) {
  v = wave_umax(v);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) v = max(v, sh[w]);
  return v;
}

// Any length and alignment: one workgroup per row, element by element.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void int8_quant_any_kernel(const uint16_t* __restrict__ x, int H,
                                                                     int8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ uint32_t sh[kRowThreads / 64];
  const size_t at = (size_t)blockIdx.x * H;
  uint32_t amax = 0;
  for (int i = threadIdx.x; i < H; i += kRowThreads) amax = max(amax, __float_as_uint(fabsf(T::to_f32(x[at + i]))));
  const Int8Row row = int8_row(block_umax<kRowThreads>(amax, sh));
  if (threadIdx.x == 0) scale[blockIdx.x] = row.s;
  for (int i = threadIdx.x; i < H; i += kRowThreads) {
    const float v[4] = {T::to_f32(x[at + i]), 0.f, 0.f, 0.f};
    q[at + i] = (int8_t)(int8_codes4(v, row) & 0xFF);
  }
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void int8_norm_any_kernel(const uint16_t* __restrict__ hidden,
                                                                    uint16_t* residual,
                                                                    const uint16_t* __restrict__ weight, int H, float eps,
                                                                    int8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ float shf[4];
  __shared__ uint32_t sh[kRowThreads / 64];
  const size_t at = (size_t)blockIdx.x * H;
  float ss = 0.f;
  for (int i = threadIdx.x; i < H; i += kRowThreads) {
    const float t = T::to_f32(hidden[at + i]) + T::to_f32(residual[at + i]);
    ss = fmaf(t, t, ss);
    residual[at + i] = T::from_f32(t);  // read again below by this same thread only
  }
  const float inv = rsqrtf(wg4_sum(ss, shf) / (float)H + eps);
  uint32_t amax = 0;
  for (int i = threadIdx.x; i < H; i += kRowThreads)
    amax = max(amax, __float_as_uint(fabsf(f32_round(T::to_f32(residual[at + i]) * inv * T::to_f32(weight[i])))));
  const Int8Row row = int8_row(block_umax<kRowThreads>(amax, sh));
  if (threadIdx.x == 0) scale[blockIdx.x] = row.s;
  for (int i = threadIdx.x; i < H; i += kRowThreads) {
    const float v[4] = {f32_round(T::to_f32(residual[at + i]) * inv * T::to_f32(weight[i])), 0.f, 0.f, 0.f};
    q[at + i] = (int8_t)(int8_codes4(v, row) & 0xFF);
  }
}

}  // namespace cek

using namespace cek;

extern "C" int cek_per_token_quant_int8(const void* x, int64_t rows, int64_t H, int io_dtype, int8_t* q, float* scale,
                                        void* stream) {
  if (rows < 0 || H <= 0 || rows > INT32_MAX || H > INT32_MAX / 2) return CEK_ERR_INVALID;
  if (io_dtype != CEK_F16 && io_dtype != CEK_BF16) return CEK_ERR_INVALID;
  if (rows == 0) return CEK_OK;
  if (!x || !q || !scale) return CEK_ERR_INVALID;
  hipStream_t st = (hipStream_t)stream;
  const uint16_t* xp = static_cast<const uint16_t*>(x);
  if (io_dtype == CEK_F16) int8_quant_any_kernel<F16><<<(unsigned)rows, kRowThreads, 0, st>>>(xp, (int)H, q, scale);
  else int8_quant_any_kernel<BF16><<<(unsigned)rows, kRowThreads, 0, st>>>(xp, (int)H, q, scale);
  return check_launch();
}

extern "C" int cek_fused_add_rms_norm_quant_int8(const void* hidden, void* residual, const void* weight, int64_t rows,
                                                 int64_t H, float eps, int io_dtype, int8_t* q, float* scale,
                                                 void* stream) {
  if (rows < 0 || H <= 0 || rows > INT32_MAX || H > INT32_MAX / 2) return CEK_ERR_INVALID;
  if (io_dtype != CEK_F16 && io_dtype != CEK_BF16) return CEK_ERR_INVALID;
  if (rows == 0) return CEK_OK;
  if (!hidden || !residual || !weight || !q || !scale) return CEK_ERR_INVALID;
  hipStream_t st = (hipStream_t)stream;
  const uint16_t* h = static_cast<const uint16_t*>(hidden);
  const uint16_t* w = static_cast<const uint16_t*>(weight);
  uint16_t* r = static_cast<uint16_t*>(residual);
  if (io_dtype == CEK_F16)
    int8_norm_any_kernel<F16><<<(unsigned)rows, kRowThreads, 0, st>>>(h, r, w, (int)H, eps, q, scale);
  else
    int8_norm_any_kernel<BF16><<<(unsigned)rows, kRowThreads, 0, st>>>(h, r, w, (int)H, eps, q, scale);
  return check_launch();
}
