// cek_kv4.hip -- writes to and reads from the 4-bit key/value cache, gfx950
// (layout and number format: cek_kv4.h).
//
// Both move bytes: n_kv hd 4 bytes a token of 16-bit rows against n_kv (hd + 8) of
// cache.  hd / 8 lanes take a token's head row, eight values each (a 16-byte load or
// store; K's codes a 32-bit word, V's two 16-bit words eight bytes apart), so a
// wave has 8, 4 or 2 tokens.  V's 16-bit accesses of neighbouring tokens meet in the
// same cache lines.
//
// The write takes its loads and its arithmetic, about 18 vector operations a value, half
// of its time each and hardly at the same time: one row of K or V a wave, so that some
// waves load while others compute (8000 rows of 8 x 128 14.3 us; with four rows in
// flight a wave 16.0).  The read is bound by its 16-bit
// rows, stored past the caches (32768 rows of 8 x 128 27.1 us, 6.3 TB/s; 42 us through
// them): ROWS rows a wave in flight, four, or one where that leaves the GPU part
// empty (8 rows 4.0 -> 2.5 us).
#include <type_traits>

#include "cek_kv4.h"

namespace cek {

// Extremes of a row on its 16-bit patterns, two at a time: as integers with the
// lower bits of negative values flipped they are in the values' order, NaNs beyond
// the infinities (so that the extremes tell whether all are finite), and an
// integer minimum needs none of the care for NaNs that a float one takes.
typedef short s2 __attribute__((ext_vector_type(2)));
__device__ inline s2 kv4_order(uint32_t pair) {
  const s2 v = __builtin_bit_cast(s2, pair);
  return v ^ ((v >> (short)15) & (short)0x7FFF);
}
template <typename T>
__device__ inline float kv4_unorder(short key) {
  return T::to_f32((uint16_t)(key ^ ((key >> 15) & 0x7FFF)));
}
// op over the LPT lanes of a token (8, 16 or 32, aligned).
template <int LPT, typename OP>
__device__ inline s2 kv4_over_token(s2 v, OP op) {
  auto dpp = [&](auto ctrl) {
    const int y = __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF, 0xF, true);
    v = op(v, __builtin_bit_cast(s2, y));
  };
  dpp(std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  dpp(std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  dpp(std::integral_constant<int, 0x141>{});  // row_half_mirror
  if constexpr (LPT >= 16) dpp(std::integral_constant<int, 0x140>{});  // row_mirror
  if constexpr (LPT >= 32) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = op(__builtin_bit_cast(s2, (uint32_t)a[0]), __builtin_bit_cast(s2, (uint32_t)a[1]));
  }
  return v;
}

// Row i of a token: K's of heads 0 .. n_kv - 1, then V's.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv4_write_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                        uint8_t* __restrict__ cache, const int64_t* __restrict__ slots,
                                                        int64_t T_rows, int64_t ks, int64_t vs, int vec, Kv4Dims dm) {
  constexpr int LPT = HD / 8, TPW = 64 / LPT;
  const int lane = threadIdx.x & 63, j = lane % LPT;
  const int64_t t = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * TPW + lane / LPT;
  const int row = blockIdx.y, h = row < dm.n_kv ? row : row - dm.n_kv;
  const int bs = 1 << dm.bs_log2;
  const bool is_v = row >= dm.n_kv;
  u4 x = u4{0u, 0u, 0u, 0u};
  int64_t slot = -1;
  if (t < T_rows) {
    slot = slots[t];
    const uint16_t* src = (is_v ? v + t * vs : k + t * ks) + (int64_t)h * HD + 8 * j;
    if (vec) x = load_u4(src);
    else
      for (int e = 0; e < 4; ++e) x[e] = (uint32_t)src[2 * e] | ((uint32_t)src[2 * e + 1] << 16);
  }
  s2 lo = kv4_order(x[0]), hi = lo;
#pragma unroll
  for (int e = 1; e < 4; ++e) {
    const s2 y = kv4_order(x[e]);
    lo = __builtin_elementwise_min(lo, y);
    hi = __builtin_elementwise_max(hi, y);
  }
  lo = kv4_over_token<LPT>(lo, [](s2 a, s2 b) { return __builtin_elementwise_min(a, b); });
  hi = kv4_over_token<LPT>(hi, [](s2 a, s2 b) { return __builtin_elementwise_max(a, b); });
  const short bottom = lo[0] < lo[1] ? lo[0] : lo[1], top = hi[0] > hi[1] ? hi[0] : hi[1];
  const bool finite = top < (short)T::inf && bottom > (short)~T::inf;
  const uint32_t p = kv4_params(kv4_unorder<T>(bottom), kv4_unorder<T>(top), finite);
  const float s = kv4_step(p), m = kv4_centre(p);
  const QuantDiv d = quant_div(s > 0.f ? s : 1.f);
  float c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = kv4_code(T::to_f32((uint16_t)(x[e / 2] >> (16 * (e & 1)))), m, d);
  // four codes as one number below 2^16: exact
  const float a = fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]);
  const float b = fmaf(fmaf(fmaf(c[7], 16.f, c[6]), 16.f, c[5]), 16.f, c[4]);
  const uint32_t w = s > 0.f ? (uint32_t)a | ((uint32_t)b << 16) : 0x88888888u;
  if (slot < 0 || (slot >> dm.bs_log2) >= dm.num_blocks) return;
  uint8_t* base = cache + (slot >> dm.bs_log2) * dm.block_stride + (int64_t)h * kv4_head_bytes(bs, HD);
  const int tok = (int)(slot & (bs - 1));
  if (is_v) {
    uint16_t* to = reinterpret_cast<uint16_t*>(base + kv4_v_codes(bs, HD)) + (tok >> 2) * HD + 8 * j + (tok & 3);
    to[0] = (uint16_t)w;
    to[4] = (uint16_t)(w >> 16);
  } else {
    reinterpret_cast<uint32_t*>(base)[tok * LPT + j] = w;
  }
  if (j == 0) *reinterpret_cast<uint32_t*>(base + (is_v ? kv4_v_params(bs, HD) : kv4_k_params(bs, HD)) + 4 * tok) = p;
}

template <typename T, int HD, int ROWS>
__global__ __launch_bounds__(256) void kv4_read_kernel(const uint8_t* __restrict__ cache, const int64_t* __restrict__ slots,
                                                       uint16_t* __restrict__ k, uint16_t* __restrict__ v,
                                                       int64_t T_rows, int64_t ks, int64_t vs, int vec, Kv4Dims dm) {
  constexpr int LPT = HD / 8, TPW = 64 / LPT;
  const int lane = threadIdx.x & 63, j = lane % LPT;
  const int64_t t = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * TPW + lane / LPT;
  if (t >= T_rows) return;
  const int row0 = blockIdx.y * ROWS;
  const int bs = 1 << dm.bs_log2;
  const int64_t slot = slots[t];
  const bool in = slot >= 0 && (slot >> dm.bs_log2) < dm.num_blocks;
  const int tok = in ? (int)(slot & (bs - 1)) : 0;
  uint32_t w[ROWS], p[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = row0 + r, h = row < dm.n_kv ? row : row - dm.n_kv;
    w[r] = p[r] = 0;
    if (in && row < 2 * dm.n_kv) {
      const uint8_t* base = cache + (slot >> dm.bs_log2) * dm.block_stride + (int64_t)h * kv4_head_bytes(bs, HD);
      if (row < dm.n_kv) {
        w[r] = reinterpret_cast<const uint32_t*>(base)[tok * LPT + j];
        p[r] = *reinterpret_cast<const uint32_t*>(base + kv4_k_params(bs, HD) + 4 * tok);
      } else {
        const uint16_t* from =
            reinterpret_cast<const uint16_t*>(base + kv4_v_codes(bs, HD)) + (tok >> 2) * HD + 8 * j + (tok & 3);
        w[r] = (uint32_t)from[0] | ((uint32_t)from[4] << 16);
        p[r] = *reinterpret_cast<const uint32_t*>(base + kv4_v_params(bs, HD) + 4 * tok);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = row0 + r, h = row < dm.n_kv ? row : row - dm.n_kv;
    if (row >= 2 * dm.n_kv) break;
    u4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e] = (uint32_t)T::from_f32(kv4_value((w[r] >> (8 * e)) & 15, p[r])) |
             ((uint32_t)T::from_f32(kv4_value((w[r] >> (8 * e + 4)) & 15, p[r])) << 16);
    if (!in) y = u4{0u, 0u, 0u, 0u};
    uint16_t* dst = (row < dm.n_kv ? k + t * ks : v + t * vs) + (int64_t)h * HD + 8 * j;
    if (vec) __builtin_nontemporal_store(y, reinterpret_cast<u4*>(dst));
    else
      for (int e = 0; e < 8; ++e) dst[e] = (uint16_t)(y[e / 2] >> (16 * (e & 1)));
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
  const int64_t tokens = 4 * (512 / hd);  // of a workgroup
  const dim3 wgs((unsigned)((T + tokens - 1) / tokens), (unsigned)(2 * n_kv));
  const int vec = aligned(k, 16) && aligned(v, 16) && k_stride % 8 == 0 && v_stride % 8 == 0;
  hipStream_t st = (hipStream_t)stream;
  const uint16_t *kp = static_cast<const uint16_t*>(k), *vp = static_cast<const uint16_t*>(v);
  uint8_t* cp = static_cast<uint8_t*>(cache);
#define CEK_GO(D)                                                                                                    \
  do {                                                                                                               \
    if (io_dtype == CEK_F16)                                                                                         \
      kv4_write_kernel<F16, D><<<wgs, 256, 0, st>>>(kp, vp, cp, slots, T, k_stride, v_stride, vec, dm);         \
    else                                                                                                             \
      kv4_write_kernel<BF16, D><<<wgs, 256, 0, st>>>(kp, vp, cp, slots, T, k_stride, v_stride, vec, dm);        \
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
  const int64_t tokens = 4 * (512 / hd);  // of a workgroup
  // four rows a wave where that still gives every SIMD two waves
  const int64_t groups = (T + tokens - 1) / tokens;
  const int rows = groups * ((2 * n_kv + 3) / 4) >= 512 ? 4 : 1;
  const dim3 wgs((unsigned)groups, (unsigned)((2 * n_kv + rows - 1) / rows));
  const int vec = aligned(k, 16) && aligned(v, 16) && k_stride % 8 == 0 && v_stride % 8 == 0;
  hipStream_t st = (hipStream_t)stream;
  uint16_t *kp = static_cast<uint16_t*>(k), *vp = static_cast<uint16_t*>(v);
  const uint8_t* cp = static_cast<const uint8_t*>(cache);
#define CEK_READ(TY, D, N) \
  kv4_read_kernel<TY, D, N><<<wgs, 256, 0, st>>>(cp, slots, kp, vp, T, k_stride, v_stride, vec, dm)
#define CEK_GO(D)                              \
  do {                                         \
    if (io_dtype == CEK_F16) {                 \
      if (rows == 4) CEK_READ(F16, D, 4);      \
      else CEK_READ(F16, D, 1);                \
    } else {                                   \
      if (rows == 4) CEK_READ(BF16, D, 4);     \
      else CEK_READ(BF16, D, 1);               \
    }                                          \
  } while (0)
  CEK_KV4_HD(CEK_GO);
#undef CEK_GO
  return check_launch();
}
