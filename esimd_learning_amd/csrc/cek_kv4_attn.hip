// cek_kv4_attn.hip -- attention over the 4-bit paged key/value cache, gfx950
// (layout and number format: cek_kv4.h).
#include "cek_kv4.h"

namespace cek {

struct Kv4AttnArgs {
  const uint16_t* q;
  uint16_t* out;
  const uint8_t* cache;
  const int32_t *tables, *kv_lens, *cu_q;
  int64_t T, q_stride, out_stride, table_stride;
  Kv4Dims dm;
  int R, n_q, max_blocks, window;
  float scale;
};

// One wave per (row, head): a key per lane, then the row's values with each lane
// owning hd / 64 of them.
template <typename T, int HD>
__global__ __launch_bounds__(64) void kv4_attn_simple_kernel(Kv4AttnArgs a) {
  constexpr int E = HD / 64;
  __shared__ float qs[HD];
  const int lane = threadIdx.x, h = blockIdx.y;
  const int64_t t = blockIdx.x;
  if (t >= a.cu_q[a.R] || t < a.cu_q[0]) return;
  int lo = 0, hi = a.R;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int bs = 1 << a.dm.bs_log2;
  const int64_t kv = min((int64_t)max(a.kv_lens[lo], 0), (int64_t)a.max_blocks << a.dm.bs_log2);
  const int64_t pos = kv - (a.cu_q[lo + 1] - t);
  const int64_t first = a.window > 0 ? max((int64_t)0, pos - a.window + 1) : 0;
  const int kvh = h / (a.n_q / a.dm.n_kv);
  for (int e = 0; e < E; ++e) qs[lane * E + e] = T::to_f32(a.q[t * a.q_stride + (int64_t)h * HD + lane * E + e]);
  __syncthreads();
  float m = -1e30f, l = 0.f, o[E] = {};
  for (int64_t j0 = first & ~63; j0 <= pos; j0 += 64) {
    const int64_t j = j0 + lane;
    int32_t blk = -1;
    if (j >= first && j <= pos) blk = a.tables[(int64_t)lo * a.table_stride + (j >> a.dm.bs_log2)];
    if (blk >= a.dm.num_blocks) blk = -1;
    const int tok = (int)(j & (bs - 1));
    const uint8_t* base = a.cache + (int64_t)max(blk, 0) * a.dm.block_stride + (int64_t)kvh * kv4_head_bytes(bs, HD);
    float s = -INFINITY;
    if (blk >= 0) {
      const uint32_t p = *reinterpret_cast<const uint32_t*>(base + kv4_k_params(bs, HD) + 4 * tok);
      float acc = 0.f;
      for (int d = 0; d < HD; d += 8) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(base + tok * (HD / 2) + d / 2);
        for (int e = 0; e < 8; ++e) acc = fmaf(qs[d + e], kv4_value((w >> (4 * e)) & 15, p), acc);
      }
      s = acc * a.scale;
    }
    const float nm = fmaxf(m, wave_max(s));
    const float keep = __expf(m - nm), pr = __expf(s - nm);
    l = l * keep + wave_sum(pr);
    for (int e = 0; e < E; ++e) o[e] *= keep;
    m = nm;
    for (int i = 0; i < 64; ++i) {
      const int32_t bi = __shfl(blk, i, 64);
      if (bi < 0) continue;
      const float pi = __shfl(pr, i, 64);
      const int ti = (int)((j0 + i) & (bs - 1));
      const uint8_t* vb = a.cache + (int64_t)bi * a.dm.block_stride + (int64_t)kvh * kv4_head_bytes(bs, HD);
      const uint32_t p = *reinterpret_cast<const uint32_t*>(vb + kv4_v_params(bs, HD) + 4 * ti);
      const uint16_t* words = reinterpret_cast<const uint16_t*>(vb + kv4_v_codes(bs, HD)) + (ti >> 2) * HD + (ti & 3);
      for (int e = 0; e < E; ++e) {
        const int d = lane * E + e;
        o[e] = fmaf(pi, kv4_value((words[(d >> 2) * 4] >> (4 * (d & 3))) & 15, p), o[e]);
      }
    }
  }
  for (int e = 0; e < E; ++e)
    a.out[t * a.out_stride + (int64_t)h * HD + lane * E + e] = T::from_f32(l > 0.f || l != l ? o[e] / l : 0.f);
}

}  // namespace cek

using namespace cek;

extern "C" int64_t cek_kv4_attention_workspace_size(int64_t T, int64_t R, int64_t n_q, int64_t n_kv, int64_t hd,
                                                    int64_t max_q_len, int64_t max_kv_len) {
  return 0;
}

extern "C" int cek_kv4_attention(const void* q, const void* cache, const int32_t* block_tables, const int32_t* kv_lens,
                                 const int32_t* cu_q, void* out, int64_t T, int64_t R, int64_t n_q, int64_t n_kv,
                                 int64_t hd, int64_t block_size, int64_t num_blocks, int64_t q_stride, int64_t out_stride,
                                 int64_t block_stride, int64_t table_stride, int64_t max_blocks, float scale,
                                 int64_t max_q_len, int64_t max_kv_len, int64_t window, int io_dtype, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  Kv4AttnArgs a;
  const int rc = kv4_dims(n_kv, hd, block_size, num_blocks, block_stride, a.dm);
  if (rc != CEK_OK) return rc;
  if (io_dtype != CEK_F16 && io_dtype != CEK_BF16) return CEK_ERR_INVALID;
  if (T < 0 || T > INT32_MAX || R < 0 || R > INT32_MAX / 2 || n_q <= 0 || n_q % n_kv || n_q > 65535) return CEK_ERR_INVALID;
  if (q_stride < n_q * hd || out_stride < n_q * hd || max_blocks <= 0 || table_stride < max_blocks ||
      max_blocks * block_size > INT32_MAX || window < 0 || window > INT32_MAX || max_q_len < 0 || max_kv_len < 0 ||
      !(scale > 0.f) || !__builtin_isfinite(scale))
    return CEK_ERR_INVALID;
  if (T == 0 || R == 0) return CEK_OK;
  if (!q || !cache || !block_tables || !kv_lens || !cu_q || !out || !aligned(cache, 16)) return CEK_ERR_INVALID;
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.cache = static_cast<const uint8_t*>(cache);
  a.tables = block_tables;
  a.kv_lens = kv_lens;
  a.cu_q = cu_q;
  a.T = T;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.table_stride = table_stride;
  a.R = (int)R;
  a.n_q = (int)n_q;
  a.max_blocks = (int)max_blocks;
  a.window = (int)window;
  a.scale = scale;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)T, (unsigned)n_q);
#define CEK_GO(D)                                                                    \
  do {                                                                               \
    if (io_dtype == CEK_F16) kv4_attn_simple_kernel<F16, D><<<grid, 64, 0, st>>>(a); \
    else kv4_attn_simple_kernel<BF16, D><<<grid, 64, 0, st>>>(a);                    \
  } while (0)
  CEK_KV4_HD(CEK_GO);
#undef CEK_GO
  return check_launch();
}
