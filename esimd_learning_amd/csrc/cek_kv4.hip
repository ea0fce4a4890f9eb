// cek_kv4.hip -- writes to and reads from the 4-bit key/value cache, gfx950
// (layout and number format: cek_kv4.h).
#include "cek_kv4.h"

namespace cek {

// One wave per (token, kv head, K or V): each lane holds hd / 64 values of the
// row, the extremes are a butterfly over the wave.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv4_write_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                        uint8_t* __restrict__ cache, const int64_t* __restrict__ slots,
                                                        int64_t T_rows, int64_t ks, int64_t vs, Kv4Dims dm) {
  constexpr int E = HD / 64;  // values per lane
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t t = item / (2 * dm.n_kv);
  if (t >= T_rows) return;
  const int h = (int)(item % (2 * dm.n_kv)) >> 1, is_v = (int)(item & 1);
  const int64_t slot = slots[t];
  const int bs = 1 << dm.bs_log2;
  if (slot < 0 || (slot >> dm.bs_log2) >= dm.num_blocks) return;
  const uint16_t* x = (is_v ? v + t * vs : k + t * ks) + (int64_t)h * HD;
  float f[E], lo = INFINITY, hi = -INFINITY;
  bool finite = true;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    f[e] = T::to_f32(x[lane * E + e]);
    lo = fminf(lo, f[e]);
    hi = fmaxf(hi, f[e]);
    finite = finite && __builtin_isfinite(f[e]);
  }
  hi = wave_max(hi);
  lo = -wave_max(-lo);
  const uint32_t p = kv4_params(lo, hi, __all(finite));
  const float s = kv4_step(p);
  const QuantDiv d = quant_div(s > 0.f ? s : 1.f);
  uint32_t w = 0;  // this lane's codes
#pragma unroll
  for (int e = 0; e < E; ++e) w |= kv4_code(f[e], kv4_centre(p), d, s > 0.f) << (4 * e);
  uint8_t* base = cache + (slot >> dm.bs_log2) * dm.block_stride + (int64_t)h * kv4_head_bytes(bs, HD);
  const int tok = (int)(slot & (bs - 1));
  // gather eight lanes' codes into words of four values
  constexpr int LPW = 4 / E;  // lanes per 16-bit word
  uint32_t word = w;
#pragma unroll
  for (int i = 1; i < LPW; ++i) word |= (uint32_t)__shfl_down((int)w, i, 64) << (4 * E * i);
  if (lane % LPW == 0) {
    const int u = lane / LPW;  // values 4u .. 4u + 3
    uint16_t* to = is_v ? reinterpret_cast<uint16_t*>(base + kv4_v_codes(bs, HD)) + ((tok >> 2) * (HD / 4) + u) * 4 + (tok & 3)
                        : reinterpret_cast<uint16_t*>(base) + tok * (HD / 4) + u;
    *to = (uint16_t)word;
  }
  if (lane == 0)
    *reinterpret_cast<uint32_t*>(base + (is_v ? kv4_v_params(bs, HD) : kv4_k_params(bs, HD)) + 4 * tok) = p;
}

// One wave per (row, kv head, K or V).
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv4_read_kernel(const uint8_t* __restrict__ cache, const int64_t* __restrict__ slots,
                                                       uint16_t* __restrict__ k, uint16_t* __restrict__ v,
                                                       int64_t T_rows, int64_t ks, int64_t vs, Kv4Dims dm) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t t = item / (2 * dm.n_kv);
  if (t >= T_rows) return;
  const int h = (int)(item % (2 * dm.n_kv)) >> 1, is_v = (int)(item & 1);
  const int64_t slot = slots[t];
  const int bs = 1 << dm.bs_log2;
  const bool in = slot >= 0 && (slot >> dm.bs_log2) < dm.num_blocks;
  const uint8_t* base = cache + (in ? (slot >> dm.bs_log2) * dm.block_stride : 0) + (int64_t)h * kv4_head_bytes(bs, HD);
  const int tok = in ? (int)(slot & (bs - 1)) : 0;
  uint16_t* y = (is_v ? v + t * vs : k + t * ks) + (int64_t)h * HD;
  const uint32_t p = *reinterpret_cast<const uint32_t*>(base + (is_v ? kv4_v_params(bs, HD) : kv4_k_params(bs, HD)) + 4 * tok);
  if (lane < HD / 4) {
    const uint16_t* from = is_v ? reinterpret_cast<const uint16_t*>(base + kv4_v_codes(bs, HD)) +
                                      ((tok >> 2) * (HD / 4) + lane) * 4 + (tok & 3)
                                : reinterpret_cast<const uint16_t*>(base) + tok * (HD / 4) + lane;
    const uint32_t w = *from;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[4 * lane + e] = in ? T::from_f32(kv4_value((w >> (4 * e)) & 15, p)) : 0;
  }
}

}  // namespace cek

using namespace cek;

extern "C" int cek_kv4_cache_write(const void* k, const void* v, void* cache, const int64_t* slots, int64_t T,
                                   int64_t n_kv, int64_t hd, int64_t block_size, int64_t num_blocks, int64_t k_stride,
                                   int64_t v_stride, int64_t block_stride, int io_dtype, void* stream) {
  Kv4Dims dm;
  const int rc = kv4_dims(n_kv, hd, block_size, num_blocks, block_stride, dm);
  if (rc != CEK_OK) return rc;
  if (io_dtype != CEK_F16 && io_dtype != CEK_BF16) return CEK_ERR_INVALID;
  if (T < 0 || T > INT32_MAX || k_stride < n_kv * hd || v_stride < n_kv * hd) return CEK_ERR_INVALID;
  if (T == 0) return CEK_OK;
  if (!k || !v || !cache || !slots || !aligned(cache, 16)) return CEK_ERR_INVALID;
  const int64_t wgs = (T * 2 * n_kv + 3) / 4;
  if (wgs > INT32_MAX) return CEK_ERR_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  const uint16_t *kp = static_cast<const uint16_t*>(k), *vp = static_cast<const uint16_t*>(v);
  uint8_t* cp = static_cast<uint8_t*>(cache);
#define CEK_GO(D)                                                                                                    \
  do {                                                                                                               \
    if (io_dtype == CEK_F16)                                                                                         \
      kv4_write_kernel<F16, D><<<(unsigned)wgs, 256, 0, st>>>(kp, vp, cp, slots, T, k_stride, v_stride, dm);         \
    else                                                                                                             \
      kv4_write_kernel<BF16, D><<<(unsigned)wgs, 256, 0, st>>>(kp, vp, cp, slots, T, k_stride, v_stride, dm);        \
  } while (0)
  CEK_KV4_HD(CEK_GO);
#undef CEK_GO
  return check_launch();
}

extern "C" int cek_kv4_cache_read(const void* cache, const int64_t* slots, void* k, void* v, int64_t T, int64_t n_kv,
                                  int64_t hd, int64_t block_size, int64_t num_blocks, int64_t k_stride, int64_t v_stride,
                                  int64_t block_stride, int io_dtype, void* stream) {
  Kv4Dims dm;
  const int rc = kv4_dims(n_kv, hd, block_size, num_blocks, block_stride, dm);
  if (rc != CEK_OK) return rc;
  if (io_dtype != CEK_F16 && io_dtype != CEK_BF16) return CEK_ERR_INVALID;
  if (T < 0 || T > INT32_MAX || k_stride < n_kv * hd || v_stride < n_kv * hd) return CEK_ERR_INVALID;
  if (T == 0) return CEK_OK;
  if (!k || !v || !cache || !slots || !aligned(cache, 16)) return CEK_ERR_INVALID;
  const int64_t wgs = (T * 2 * n_kv + 3) / 4;
  if (wgs > INT32_MAX) return CEK_ERR_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  uint16_t *kp = static_cast<uint16_t*>(k), *vp = static_cast<uint16_t*>(v);
  const uint8_t* cp = static_cast<const uint8_t*>(cache);
#define CEK_GO(D)                                                                                                   \
  do {                                                                                                              \
    if (io_dtype == CEK_F16)                                                                                        \
      kv4_read_kernel<F16, D><<<(unsigned)wgs, 256, 0, st>>>(cp, slots, kp, vp, T, k_stride, v_stride, dm);         \
    else                                                                                                            \
      kv4_read_kernel<BF16, D><<<(unsigned)wgs, 256, 0, st>>>(cp, slots, kp, vp, T, k_stride, v_stride, dm);        \
  } while (0)
  CEK_KV4_HD(CEK_GO);
#undef CEK_GO
  return check_launch();
}
