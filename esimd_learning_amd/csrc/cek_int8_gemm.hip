// cek_int8_gemm.hip -- products of int8 codes with a scale per token and one per
// output channel, and the gated block over a merged gate/up matrix, gfx950:
//   y[m, n] = Out((f32(sum_k a[m, k] b[n, k]) sb[n]) sa[m])
//   y[m, i] = Out(act(g) u), g and u such values of b's rows i and d + i, unrounded
#include "cek_int8_tile.h"
#include "cek_int8_few.h"
#include "cek_segs.h"

namespace cek {

// Split K: y from the parts' int32 sums [parts][M][NB] (NB = N, or 2 N for the gated
// block), added as integers: what one part would have given, bit for bit.  Four
// outputs of a row per thread.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void int8_join_kernel(const int32_t* __restrict__ P, const float* __restrict__ sa,
                                                        const float* __restrict__ sb, uint16_t* __restrict__ y, int M,
                                                        int N, int parts) {
  constexpr bool GLU = ACT >= 0;
  const uint32_t quads = (uint32_t)(N + 3) / 4, q = blockIdx.x * 256 + threadIdx.x;
  const int m = (int)(q / quads), n = (int)(q % quads) * 4;
  if (m >= M) return;
  const size_t NB = GLU ? 2 * (size_t)N : N, step = NB * M;
  const int32_t* p = P + m * NB + n;
  const float s0 = sa[m];
  if ((N & 3) == 0 && (reinterpret_cast<uintptr_t>(y) & 7) == 0 && (reinterpret_cast<uintptr_t>(sb) & 15) == 0) {
    i4 g{0, 0, 0, 0}, u{0, 0, 0, 0};
    // four parts at a time: their loads are out together, past the last they repeat it
    for (int k = 0; k < parts; k += 4) {
      i4 pg[4], pu[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int32_t* q = p + (size_t)min(k + j, parts - 1) * step;
        pg[j] = *reinterpret_cast<const i4*>(q);
        if constexpr (GLU) pu[j] = *reinterpret_cast<const i4*>(q + N);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k + j < parts) {
          g += pg[j];
          if constexpr (GLU) u += pu[j];
        }
    }
    const f4 sg = *reinterpret_cast<const f4*>(sb + n);
    f4 su = sg;
    if constexpr (GLU) su = *reinterpret_cast<const f4*>(sb + N + n);
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (GLU) o[e] = int8_glu<ACT>(g[e], u[e], s0, sg[e], su[e]);
      else o[e] = int8_scaled(g[e], s0, sg[e]);
    }
    *reinterpret_cast<uint2*>(y + (size_t)m * N + n) = make_uint2(int8_pack2<T>(o[0], o[1]), int8_pack2<T>(o[2], o[3]));
    return;
  }
  for (int e = 0; e < 4 && n + e < N; ++e) {
    int g = 0, u = 0;
    for (int k = 0; k < parts; ++k) {
      g += p[k * step + e];
      if constexpr (GLU) u += p[k * step + N + e];
    }
    float o;
    if constexpr (GLU) o = int8_glu<ACT>(g, u, s0, sb[n + e], sb[(size_t)N + n + e]);
    else o = int8_scaled(g, s0, sb[n + e]);
    y[(size_t)m * N + n + e] = T::from_f32(o);
  }
}

// ---- which tile, how many parts of K -----------------------------------------
// Time of a launch: rounds of 256 workgroups (one per CU), each a fixed part and a
// time per 128 values of K; a last round of fewer workgroups runs between the times
// of a nearly empty and a full chip.  Split K adds the join and its traffic.  Fitted
// to 730 launches over 41 shapes of 72 to 8192 rows (weights from HBM): 9% off on
// average, and the pick 0.2% above the fastest of all tiles and splits (geometric
// mean; 3% at worst).  They are plain products; the gated block goes by the same constants.
// Larger tiles move fewer operand bytes per product, smaller ones fill the chip sooner.
struct Int8Opt {
  int bm, bn;
  double fixed, step, fixed0, step0;  // us: a full round, and one with few workgroups
};
constexpr Int8Opt kInt8Opts[] = {
    {256, 256, 7.11, 1.441, 7.24, 1.075}, {256, 192, 7.22, 1.125, 7.36, 0.768}, {256, 128, 6.22, 0.851, 5.12, 0.582},
    {128, 256, 6.15, 0.874, 5.26, 0.648}, {128, 192, 6.22, 0.722, 4.07, 0.547}, {128, 128, 5.52, 0.559, 3.55, 0.404},
    {64, 128, 4.27, 0.399, 3.25, 0.280}};
constexpr int kInt8Tiles = sizeof(kInt8Opts) / sizeof(kInt8Opts[0]);
constexpr int kInt8Parts[] = {1, 2, 3, 4, 6, 8, 12};
constexpr int64_t kInt8MaxWorkspace = int64_t(1) << 28;

static double int8_us(const Int8Opt& o, int64_t M, int64_t NB, int64_t steps, int parts) {
  const int64_t n = (M + o.bm - 1) / o.bm * ((NB + o.bn - 1) / o.bn) * parts, full = n / kCUs, rest = n % kCUs;
  const double s = (double)((steps + parts - 1) / parts), f = (double)rest / kCUs;
  constexpr double kStart = 2.51;  // of a round's fixed part, what only the first one takes
  double t = kStart + (double)full * (o.fixed - kStart + s * o.step);
  if (rest) t += o.fixed0 + (o.fixed - o.fixed0) * f - kStart + s * (o.step0 + (o.step - o.step0) * f);
  if (parts > 1) t += 3.97 + 3.07e-7 * 4.0 * (double)parts * (double)M * (double)NB;
  return t;
}

struct Int8Plan {
  int cfg, parts;  // cfg < 0: the kernels for few rows
};
// NB: rows of b.
static int64_t int8_parts_bytes(int parts, int64_t M, int64_t NB) {
  return parts > 1 ? ((int64_t)parts * M * NB * 4 + 15) / 16 * 16 : 0;
}
static Int8Plan int8_plan(int64_t M, int64_t NB, int64_t K, bool glu, int64_t ws_bytes) {
  Int8Plan best{0, 1};
  double us = 0;
  const int64_t steps = (K + 127) / 128;
  for (int c = 0; c < kInt8Tiles; ++c)
    for (int parts : kInt8Parts) {
      if (parts > 1 && (steps < 4 * parts || (double)M * (double)NB * 4 * parts > (double)kInt8MaxWorkspace ||
                        int8_parts_bytes(parts, M, NB) > ws_bytes))
        break;
      const double t = int8_us(kInt8Opts[c], M, NB, steps, parts);
      if ((c == 0 && parts == 1) || t < us) {
        us = t;
        best = Int8Plan{c, parts};
      }
    }
  if (int8_few_takes(M, NB, K, glu, us)) return Int8Plan{-1, 1};
  return best;
}

// (a grid counts its threads in 32 bits)
static bool int8_sizes_ok(int64_t M, int64_t N, int64_t K, int64_t NB) {
  return M >= 0 && N >= 0 && K > 0 && K % 16 == 0 && K <= kInt8MaxK && M <= (1 << 24) && NB <= (1 << 24);
}
static int64_t int8_workspace(int64_t M, int64_t N, int64_t K, bool glu) {
  if (N > INT32_MAX || !int8_sizes_ok(M, N, K, glu ? 2 * N : N) || M == 0 || N == 0) return 0;
  const int64_t NB = glu ? 2 * N : N;
  return int8_parts_bytes(int8_plan(M, NB, K, glu, INT64_MAX).parts, M, NB);
}

template <class C, class T, int ACT>
static int launch_int8_tile(Int8Args& g, hipStream_t st) {
  g.tiles_m = (g.M + C::BM - 1) / C::BM;
  g.tiles_n = (g.N + C::BO - 1) / C::BO;
  const int64_t n = (int64_t)g.tiles_m * g.tiles_n * g.parts;
  if (n > INT32_MAX / C::NT) return CEK_ERR_UNSUPPORTED;
  if (g.parts == 1) {
    int8_tile_kernel<C, T, ACT, false><<<(unsigned)n, C::NT, 0, st>>>(g);
    return check_launch();
  }
  int8_tile_kernel<C, T, ACT, true><<<(unsigned)n, C::NT, 0, st>>>(g);
  const int rc = check_launch();
  if (rc != CEK_OK) return rc;
  // (a workspace of at most 2^28 bytes: M is below 2^26 / N / parts)
  int8_join_kernel<T, ACT><<<(unsigned)(((int64_t)g.M * ((g.N + 3) / 4) + 255) / 256), 256, 0, st>>>(g.part, g.sa, g.sb, g.y,
                                                                                                     g.M, g.N, g.parts);
  return check_launch();
}

static int int8_args(const void* a, const void* sa, const void* b, const void* sb, const void* y, int64_t M, int64_t N,
                     int64_t K, int64_t NB, int out_dtype, const void* ws, int64_t ws_bytes) {
  if (!int8_sizes_ok(M, N, K, NB)) return CEK_ERR_INVALID;
  if (ws_bytes < 0 || (ws && !aligned(ws, 16))) return CEK_ERR_INVALID;
  if (out_dtype != CEK_F16 && out_dtype != CEK_BF16) return CEK_ERR_INVALID;
  if (M == 0 || N == 0) return CEK_OK;
  if (!a || !sa || !b || !sb || !y || !aligned(a, 16) || !aligned(b, 16) || !aligned(sa, 4) || !aligned(sb, 4) ||
      !aligned(y, 2))
    return CEK_ERR_INVALID;
  return CEK_OK;
}

template <class T, int ACT>
static int launch_int8_t(Int8Args& g, int cfg, hipStream_t st) {
  constexpr bool G = ACT >= 0;
  switch (cfg) {
    case 0: return launch_int8_tile<Int8Tile<256, 256, 2, 4, 2, 2, G>, T, ACT>(g, st);
    case 1: return launch_int8_tile<Int8Tile<256, 192, 4, 2, 2, 3, G>, T, ACT>(g, st);
    case 2: return launch_int8_tile<Int8Tile<256, 128, 4, 2, 3, 3, G>, T, ACT>(g, st);
    case 3: return launch_int8_tile<Int8Tile<128, 256, 2, 4, 3, 3, G>, T, ACT>(g, st);
    case 4: return launch_int8_tile<Int8Tile<128, 192, 4, 2, 3, 4, G>, T, ACT>(g, st);
    case 5: return launch_int8_tile<Int8Tile<128, 128, 2, 4, 4, 5, G>, T, ACT>(g, st);
    case 6: return launch_int8_tile<Int8Tile<64, 128, 2, 4, 5, 6, G>, T, ACT>(g, st);
    default: return CEK_ERR_UNSUPPORTED;
  }
}

template <int ACT>
static int launch_int8(const int8_t* a, const float* sa, const int8_t* b, const float* sb, void* y, int64_t M, int64_t N,
                       int64_t K, int out_dtype, void* ws, int64_t ws_bytes, hipStream_t st) {
  const Int8Plan p = int8_plan(M, ACT >= 0 ? 2 * N : N, K, ACT >= 0, ws ? ws_bytes : 0);
  if (p.cfg < 0)
    return launch_int8_few(Int8Few{reinterpret_cast<const uint8_t*>(a), sa, reinterpret_cast<const uint8_t*>(b), sb,
                                   static_cast<uint16_t*>(y), (int)M, (int)N, (int)K, out_dtype == CEK_BF16, ACT},
                           st);
  Int8Args g{reinterpret_cast<const uint8_t*>(a), sa, reinterpret_cast<const uint8_t*>(b), sb, static_cast<uint16_t*>(y),
             static_cast<int32_t*>(ws), (int)M, (int)N, (int)K, 0, 0, p.parts};
  return out_dtype == CEK_F16 ? launch_int8_t<F16, ACT>(g, p.cfg, st) : launch_int8_t<BF16, ACT>(g, p.cfg, st);
}

}  // namespace cek

using namespace cek;

extern "C" int64_t cek_gemm_int8_a8w8_workspace_size(int64_t M, int64_t N, int64_t K) {
  return int8_workspace(M, N, K, false);
}
extern "C" int64_t cek_gemm_int8_a8w8_glu_workspace_size(int64_t M, int64_t d, int64_t K) {
  return int8_workspace(M, d, K, true);
}

extern "C" int cek_gemm_int8_plan(int64_t M, int64_t N, int64_t K, int gated, int64_t workspace_bytes) {
  if (N > INT32_MAX) return -1;
  const int64_t NB = gated ? 2 * N : N;
  if (!int8_sizes_ok(M, N, K, NB) || M == 0 || N == 0) return -1;
  const Int8Plan p = int8_plan(M, NB, K, gated != 0, workspace_bytes);
  return p.cfg < 0 ? -1 : 16 * p.cfg + p.parts;
}

extern "C" int cek_gemm_int8_few_plan(int64_t M, int64_t N, int64_t K, int gated, int64_t workspace_bytes) {
  if (N > INT32_MAX) return -1;
  const int64_t NB = gated ? 2 * N : N;
  if (!int8_sizes_ok(M, N, K, NB) || M == 0 || N == 0) return -1;
  return int8_plan(M, NB, K, gated != 0, workspace_bytes).cfg < 0 ? int8_few_form(M, N, K, gated != 0) : 0;
}

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
  if (d > INT32_MAX) return CEK_ERR_INVALID;
  const int rc = int8_args(a, sa, b, sb, y, M, d, K, 2 * d, out_dtype, workspace, workspace_bytes);
  if (rc != CEK_OK || M == 0 || d == 0) return rc;
  return activation == CEK_SILU ? launch_int8<CEK_SILU>(a, sa, b, sb, y, M, d, K, out_dtype, workspace, workspace_bytes,
                                                        (hipStream_t)stream)
                                : launch_int8<CEK_GELU_TANH>(a, sa, b, sb, y, M, d, K, out_dtype, workspace,
                                                             workspace_bytes, (hipStream_t)stream);
}
