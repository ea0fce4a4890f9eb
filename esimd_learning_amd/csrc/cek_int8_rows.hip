// cek_int8_rows.hip -- int8 codes and scales of rows, alone or behind the residual
// add + RMS norm, gfx950 (the arithmetic: cek_int8.h).
//
// A row is read once and stays in registers between its maximum (or its sum of
// squares and its maximum) and its codes.  What bounds the kernels: for many rows HBM,
// for few the chain load, reduction, store (28672 x 4096 59 us, 6.0 TB/s; norm of 2048 x
// 4096 from HBM 13.9 us, 4.2 TB/s; one row of 14336 2.4 us).  The maximum is taken of the
// values' bits without their sign, which order as the values do and NaN above infinity, so
// that one reduction also tells whether the row is finite.
#include <type_traits>

#include "cek_int8.h"
#include "cek_rowops.h"

namespace cek {

constexpr int kRowThreads = 256;

// Largest of the lanes' values, in every lane.
__device__ inline uint32_t wave_umax(uint32_t v) {
#define CEK_UMAX_DPP(c) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, c, 0xF, 0xF, true))
  CEK_UMAX_DPP(0xB1);   // quad_perm [1,0,3,2]
  CEK_UMAX_DPP(0x4E);   // quad_perm [2,3,0,1]
  CEK_UMAX_DPP(0x141);  // row_half_mirror
  CEK_UMAX_DPP(0x140);  // row_mirror
#undef CEK_UMAX_DPP
  return max(max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16)),
             max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}

// The same and the sum over NW waves (sh: NW words, written once per call site).
template <int NW>
__device__ inline uint32_t block_umax(uint32_t v, uint32_t* sh) {
  v = wave_umax(v);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) v = max(v, sh[w]);
  }
  return v;
}
template <int NW>
__device__ inline float block_fsum(float v, float* sh) {
  v = wave_sum_dpp(v);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += sh[w];
  }
  return v;
}

// The largest 16-bit magnitude in a unit so far, two at a time.
typedef uint16_t us2 __attribute__((ext_vector_type(2)));
__device__ inline uint32_t pair_umax(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, b)));
}
template <typename T>
__device__ inline uint32_t amax_bits(uint32_t pair) {  // of a pair of 16-bit magnitudes, as fp32 bits
  const uint32_t m = max(pair & 0xFFFF, pair >> 16);
  return __float_as_uint(T::to_f32((uint16_t)m));
}

template <typename T>
__device__ inline uint2 unit_codes(u4 v, const Int8Row& row) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = unit_f32<T>(v, e);
  const float lo[4] = {x[0], x[1], x[2], x[3]}, hi[4] = {x[4], x[5], x[6], x[7]};
  return make_uint2(int8_codes4(lo, row), int8_codes4(hi, row));
}

// Where a row's unit u begins: eight values on from the last, but the last one at the
// row's end, where it may repeat values of the one before (ODD: H no multiple of 8, or rows
// that start anywhere, read and written without regard to alignment).
template <bool ODD>
__device__ inline int unit_at(int u, int H) { return ODD ? min(8 * u, H - 8) : 8 * u; }
template <bool ODD>
__device__ inline u4 load_unit(const uint16_t* p) {
  if constexpr (!ODD) return load_u4(p);
  u4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
template <bool ODD, typename V>
__device__ inline void store_unit(void* p, V v) {
  if constexpr (ODD) __builtin_memcpy(p, &v, sizeof(V));
  else *reinterpret_cast<V*>(p) = v;
}

// WPR waves per row (1: 256 / 64 rows per workgroup), UPT units of eight values per
// thread: 8 <= H <= 512 WPR UPT; without ODD H % 8 == 0, 16-byte aligned x and 8-byte
// aligned q.
template <typename T, int WPR, int UPT, bool ODD>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void int8_quant_kernel(const uint16_t* __restrict__ x, int rows,
                                                                               int H, int8_t* __restrict__ q,
                                                                               float* __restrict__ scale) {
  constexpr int TPR = 64 * WPR;
  __shared__ uint32_t sh[WPR];
  const int row = WPR == 1 ? (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6) : (int)blockIdx.x;
  if (WPR == 1 && row >= rows) return;
  const int tid = WPR == 1 ? threadIdx.x & 63 : threadIdx.x, units = (H + 7) >> 3;
  const uint16_t* xr = x + (size_t)row * H;
  u4 v[UPT];
#pragma unroll
  for (int j = 0; j < UPT; ++j) v[j] = load_unit<ODD>(xr + unit_at<ODD>(min(tid + j * TPR, units - 1), H));
  uint32_t pair = 0;  // (units past the row repeat its last one)
#pragma unroll
  for (int j = 0; j < UPT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) pair = pair_umax(pair, v[j][e] & 0x7FFF7FFF);
  const Int8Row r = int8_row(block_umax<WPR>(amax_bits<T>(pair), sh));
  if (tid == 0) scale[row] = r.s;
  int8_t* qr = q + (size_t)row * H;
#pragma unroll
  for (int j = 0; j < UPT; ++j) {
    const int u = tid + j * TPR;
    if (u < units) store_unit<ODD>(qr + unit_at<ODD>(u, H), unit_codes<T>(v[j], r));
  }
}

// A bf16 row's sum of squares passes fp32 where its root is 2^64 or more, far below the type's
// largest values (fp16 rows never get there).  Such a sum is taken again of the values times
// 2^-80, whose squares are at most 2^96 and the largest at least 2^-62, and 1 / rms is 2^-80
// times the scaled row's.  Ordinary rows pay a comparison (12 shapes: 6% faster to 1.4% slower).
constexpr float kFar = 0x1p-80f;
template <typename T>
__device__ inline bool sum_passes(float sum) { return std::is_same<T, BF16>::value && __float_as_uint(sum) == 0x7F800000u; }
__device__ inline float far_inv(float scaled, int H, float eps) { return kFar * rsqrtf(scaled / (float)H + eps * kFar * kFar); }

// Residual add + RMS norm + codes, likewise.  A value that two units hold counts once in the
// sum of squares, and the new residual is stored behind the sum's barrier, when every
// thread has read the old one.
template <typename T, int WPR, int UPT, bool ODD>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void int8_norm_kernel(const uint16_t* __restrict__ hidden,
                                                                              uint16_t* residual,
                                                                              const uint16_t* __restrict__ weight, int rows,
                                                                              int H, float eps, int8_t* __restrict__ q,
                                                                              float* __restrict__ scale) {
  constexpr int TPR = 64 * WPR;
  __shared__ uint32_t sh[WPR];
  __shared__ float shf[WPR], shg[WPR];
  const int row = WPR == 1 ? (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6) : (int)blockIdx.x;
  if (WPR == 1 && row >= rows) return;
  const int tid = WPR == 1 ? threadIdx.x & 63 : threadIdx.x, units = (H + 7) >> 3;
  const uint16_t* hr = hidden + (size_t)row * H;
  uint16_t* rr = residual + (size_t)row * H;
  u4 hv[UPT], rv[UPT], wv[UPT];
#pragma unroll
  for (int j = 0; j < UPT; ++j) {
    const int at = unit_at<ODD>(min(tid + j * TPR, units - 1), H);
    hv[j] = load_unit<ODD>(hr + at);
    rv[j] = load_unit<ODD>(rr + at);
  }
#pragma unroll
  for (int j = 0; j < UPT; ++j) wv[j] = load_unit<ODD>(weight + unit_at<ODD>(min(tid + j * TPR, units - 1), H));
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < UPT; ++j) {
    const int u = tid + j * TPR;
    if (u < units) {
      if constexpr (ODD) {
        const int twice = 8 * u - unit_at<true>(u, H);
        float a[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[e] = unit_f32<T>(hv[j], e) + unit_f32<T>(rv[j], e);
          ss = e < twice ? ss : fmaf(a[e], a[e], ss);
        }
        rv[j] = u4{int8_pack2<T>(a[0], a[1]), int8_pack2<T>(a[2], a[3]), int8_pack2<T>(a[4], a[5]), int8_pack2<T>(a[6], a[7])};
      } else {
        rv[j] = addnorm_pass1<T>(hv[j], rv[j], ss);
      }
    }
  }
  const float sum = block_fsum<WPR>(ss, shf);
  float inv = rsqrtf(sum / (float)H + eps);
  if (sum_passes<T>(sum)) {  // (the same in all of the row's threads; its values are read again)
    float far = 0.f;
    for (int u = tid; u < units; u += TPR) {
      const int at = unit_at<ODD>(u, H), twice = 8 * u - at;
      const u4 h = load_unit<ODD>(hr + at), r = load_unit<ODD>(rr + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = (unit_f32<T>(h, e) + unit_f32<T>(r, e)) * kFar;
        far = e < twice ? far : fmaf(a, a, far);
      }
    }
    inv = far_inv(block_fsum<WPR>(far, shg), H, eps);
  }
#pragma unroll
  for (int j = 0; j < UPT; ++j) {
    const int u = tid + j * TPR;
    if (u < units) store_unit<ODD>(rr + unit_at<ODD>(u, H), rv[j]);
  }
  // the normed values are computed twice, for the maximum and for the codes: cheaper than
  // the registers that would hold them (eight a unit)
  auto normed = [&](int j, int e) { return unit_f32<T>(rv[j], e) * inv * unit_f32<T>(wv[j], e); };
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < UPT; ++j) {
    if (tid + j * TPR < units) {
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(normed(j, e)) & 0x7FFFFFFF);
    }
  }
  const Int8Row r = int8_row(block_umax<WPR>(amax, sh));
  if (tid == 0) scale[row] = r.s;
  int8_t* qr = q + (size_t)row * H;
#pragma unroll
  for (int j = 0; j < UPT; ++j) {
    const int u = tid + j * TPR;
    if (u < units) {
      const float lo[4] = {normed(j, 0), normed(j, 1), normed(j, 2), normed(j, 3)};
      const float hi[4] = {normed(j, 4), normed(j, 5), normed(j, 6), normed(j, 7)};
      store_unit<ODD>(qr + unit_at<ODD>(u, H), make_uint2(int8_codes4(lo, r), int8_codes4(hi, r)));
    }
  }
}

// Any length and alignment: one workgroup per row, element by element, the row read again
// for each pass.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void int8_quant_any_kernel(const uint16_t* __restrict__ x, int H,
                                                                     int8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ uint32_t sh[kRowThreads / 64];
  const size_t at = (size_t)blockIdx.x * H;
  uint32_t amax = 0;
  for (int i = threadIdx.x; i < H; i += kRowThreads) amax = max(amax, __float_as_uint(T::to_f32(x[at + i])) & 0x7FFFFFFF);
  const Int8Row row = int8_row(block_umax<kRowThreads / 64>(amax, sh));
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
  __shared__ float shf[kRowThreads / 64], shg[kRowThreads / 64];
  __shared__ uint32_t sh[kRowThreads / 64];
  const size_t at = (size_t)blockIdx.x * H;
  float ss = 0.f, far = 0.f;
  for (int i = threadIdx.x; i < H; i += kRowThreads) {
    const float t = T::to_f32(hidden[at + i]) + T::to_f32(residual[at + i]);
    ss = fmaf(t, t, ss);
    far = fmaf(t * kFar, t * kFar, far);
    residual[at + i] = T::from_f32(t);  // read again below by this same thread only
  }
  const float sum = block_fsum<kRowThreads / 64>(ss, shf);
  float inv = rsqrtf(sum / (float)H + eps);
  if (sum_passes<T>(sum)) inv = far_inv(block_fsum<kRowThreads / 64>(far, shg), H, eps);
  auto normed = [&](int i) { return T::to_f32(residual[at + i]) * inv * T::to_f32(weight[i]); };
  uint32_t amax = 0;
  for (int i = threadIdx.x; i < H; i += kRowThreads) amax = max(amax, __float_as_uint(normed(i)) & 0x7FFFFFFF);
  const Int8Row row = int8_row(block_umax<kRowThreads / 64>(amax, sh));
  if (threadIdx.x == 0) scale[blockIdx.x] = row.s;
  for (int i = threadIdx.x; i < H; i += kRowThreads) {
    const float v[4] = {normed(i), 0.f, 0.f, 0.f};
    q[at + i] = (int8_t)(int8_codes4(v, row) & 0xFF);
  }
}

// Few rows: many threads for the latency of each; many: as many rows in flight as a CU
// holds (2048 rows of 4096, us: a wave a row 10.2, two units a thread 6.75; 28672 rows
// 66.3 / 61.5; 8192 rows of 2000 one unit a thread 11.3).
template <typename T, bool ODD>
static int launch_quant(const uint16_t* x, int rows, int H, int8_t* q, float* scale, hipStream_t st) {
  const int units = (H + 7) / 8;
  const bool many = rows >= 1024;
#define CEK_Q1(UPT) int8_quant_kernel<T, 1, UPT, ODD><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(x, rows, H, q, scale)
#define CEK_QW(WPR, UPT) int8_quant_kernel<T, WPR, UPT, ODD><<<(unsigned)rows, 64 * WPR, 0, st>>>(x, rows, H, q, scale)
  if (H < 8 || units > 8192) int8_quant_any_kernel<T><<<(unsigned)rows, kRowThreads, 0, st>>>(x, H, q, scale);
  else if (units <= 64) CEK_Q1(1);
  else if (units <= 128) CEK_Q1(2);
  else if (units <= 256) CEK_QW(4, 1);
  else if (many && units <= 512) CEK_QW(4, 2);
  else if (units <= 512) CEK_QW(8, 1);
  else if (many && units <= 1024) CEK_QW(4, 4);
  else if (many && units <= 2048) CEK_QW(4, 8);
  else if (units <= 1024) CEK_QW(16, 1);
  else if (units <= 2048) CEK_QW(16, 2);
  else if (units <= 4096) CEK_QW(16, 4);
  else CEK_QW(16, 8);
#undef CEK_Q1
#undef CEK_QW
  return check_launch();
}

template <typename T, bool ODD>
static int launch_norm(const uint16_t* h, uint16_t* r, const uint16_t* w, int rows, int H, float eps, int8_t* q,
                       float* scale, hipStream_t st) {
  const int units = (H + 7) / 8;
  const bool many = rows >= 1024;
#define CEK_N1(UPT) \
  int8_norm_kernel<T, 1, UPT, ODD><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(h, r, w, rows, H, eps, q, scale)
#define CEK_NW(WPR, UPT) int8_norm_kernel<T, WPR, UPT, ODD><<<(unsigned)rows, 64 * WPR, 0, st>>>(h, r, w, rows, H, eps, q, scale)
  if (H < 8 || units > 4096) int8_norm_any_kernel<T><<<(unsigned)rows, kRowThreads, 0, st>>>(h, r, w, H, eps, q, scale);
  else if (units <= 64) CEK_N1(1);
  else if (units <= 128) CEK_N1(2);
  else if (units <= 256) CEK_NW(4, 1);
  else if (many && units <= 512) CEK_NW(4, 2);
  else if (units <= 512) CEK_NW(8, 1);
  else if (many && units <= 768) CEK_NW(4, 3);
  else if (many && units <= 1024) CEK_NW(4, 4);
  else if (units <= 1024) CEK_NW(16, 1);
  else if (units <= 2048) CEK_NW(16, 2);
  else CEK_NW(16, 4);
#undef CEK_N1
#undef CEK_NW
  return check_launch();
}

// A launch takes up to 2^20 rows: a grid counts its threads in 32 bits.
template <typename T>
static int launch_rows(const void* x, void* residual, const void* weight, int64_t rows, int H, float eps, int8_t* q,
                       float* scale, hipStream_t st) {
  const uint16_t *xp = static_cast<const uint16_t*>(x), *w = static_cast<const uint16_t*>(weight);
  uint16_t* r = static_cast<uint16_t*>(residual);
  const bool odd = H % 8 != 0 || !aligned(x, 16) || !aligned(q, 8) || (r && (!aligned(r, 16) || !aligned(w, 16)));
  constexpr int64_t kMost = 1 << 20;
  for (int64_t t = 0; t < rows; t += kMost) {
    const int n = (int)(rows - t < kMost ? rows - t : kMost);
    const size_t at = (size_t)t * (size_t)H;
    const int rc = r     ? odd ? launch_norm<T, true>(xp + at, r + at, w, n, H, eps, q + at, scale + t, st)
                               : launch_norm<T, false>(xp + at, r + at, w, n, H, eps, q + at, scale + t, st)
                   : odd ? launch_quant<T, true>(xp + at, n, H, q + at, scale + t, st)
                         : launch_quant<T, false>(xp + at, n, H, q + at, scale + t, st);
    if (rc != CEK_OK) return rc;
  }
  return CEK_OK;
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
  return io_dtype == CEK_F16 ? launch_rows<F16>(x, nullptr, nullptr, rows, (int)H, 0.f, q, scale, st)
                             : launch_rows<BF16>(x, nullptr, nullptr, rows, (int)H, 0.f, q, scale, st);
}

extern "C" int cek_fused_add_rms_norm_quant_int8(const void* hidden, void* residual, const void* weight, int64_t rows,
                                                 int64_t H, float eps, int io_dtype, int8_t* q, float* scale,
                                                 void* stream) {
  if (rows < 0 || H <= 0 || rows > INT32_MAX || H > INT32_MAX / 2) return CEK_ERR_INVALID;
  if (io_dtype != CEK_F16 && io_dtype != CEK_BF16) return CEK_ERR_INVALID;
  if (rows == 0) return CEK_OK;
  if (!hidden || !residual || !weight || !q || !scale) return CEK_ERR_INVALID;
  hipStream_t st = (hipStream_t)stream;
  return io_dtype == CEK_F16 ? launch_rows<F16>(hidden, residual, weight, rows, (int)H, eps, q, scale, st)
                             : launch_rows<BF16>(hidden, residual, weight, rows, (int)H, eps, q, scale, st);
}
