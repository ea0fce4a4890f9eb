// cek_int8_stream.hip -- int8 products of a few rows of a (up to 64), gfx950: the weights
// are read from HBM once, and that is what bounds them.
#include <algorithm>
#include <type_traits>

#include "cek_int8_few.h"
#include "cek_segs.h"

namespace cek {

// ---- one to four rows --------------------------------------------------------
// v_dot4 on 16-byte units: thread u of a workgroup holds a's values of unit u of
// every 4 KB of K, for all M rows, and multiplies them with the same unit of R
// weight rows, so that a wave's load reads 1 KB of one row.  The sums meet in the
// lanes of a wave, then of four waves in LDS.  One row of 14336 x 4096 10.2 us (5.75 TB/s;
// a read alone 9.7), gated 4 x 14336 x 4096 21.6 (5.4 TB/s).
// TPR threads per weight row: 256, or fewer where K is shorter than 4 KB.
template <int M, int R, int CH, int TPR, bool GLU>
__global__ __launch_bounds__(256) void int8_dot_kernel(Int8Few p) {
  constexpr int RT = GLU ? 2 * R : R;  // weight rows of a thread: R gate rows, then their up rows
  constexpr int G = 256 / TPR, W = TPR / 64;
  __shared__ int red[4][M * RT];
  const int units = p.K / 16, tid = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  const int n0 = (blockIdx.x * G + grp) * R;
  int acc[RT][M];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) acc[r][m] = 0;
  for (int u0 = 0; u0 < units; u0 += TPR * CH) {
    u4 w[RT][CH], x[M][CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int u = min(u0 + TPR * c + tid, units - 1);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const size_t row = (size_t)min(n0 + r % R, p.N - 1) + (r >= R ? (size_t)p.N : 0);
        w[r][c] = load_u4_stream(p.b + row * p.K + 16 * u);
      }
#pragma unroll
      for (int m = 0; m < M; ++m) x[m][c] = load_u4(p.a + (size_t)m * p.K + 16 * u);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const bool in = u0 + TPR * c + tid < units;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const u4 xv = in ? x[m][c] : u4{0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][m] = __builtin_amdgcn_sdot4((int)w[r][c][e], (int)xv[e], acc[r][m], false);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) acc[r][m] = wave_isum(acc[r][m]);
  if ((tid & 63) == 0) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int m = 0; m < M; ++m) red[threadIdx.x >> 6][r * M + m] = acc[r][m];
  }
  __syncthreads();
  if (tid < M * R) {
    const int r = tid / M, m = tid % M, n = n0 + r;
    auto sum = [&](int i) {
      int s = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) s += red[grp * W + w][i];
      return s;
    };
    if (n < p.N) {
      if constexpr (GLU) int8_store(p, m, n, sum(tid), sum(tid + M * R), p.sa[m], p.sb[n], p.sb[(size_t)p.N + n]);
      else int8_store(p, m, n, sum(tid), 0, p.sa[m], p.sb[n], 0.f);
    }
  }
}

template <int M, int R, bool GLU>
static int launch_dot_r(const Int8Few& p, hipStream_t st) {
#define CEK_I8D(CH, TPR) \
  int8_dot_kernel<M, R, CH, TPR, GLU><<<(unsigned)(((int64_t)p.N + R * (256 / TPR) - 1) / (R * (256 / TPR))), 256, 0, st>>>(p)
  if (p.K <= 1024) CEK_I8D(1, 64);
  else if (p.K <= 2048) CEK_I8D(1, 128);
  else if (p.K <= 4096) CEK_I8D(1, 256);
  else CEK_I8D(2, 256);
#undef CEK_I8D
  return check_launch();
}
// Weight rows of a thread, measured (us): N = 14336, K = 4096, one row 2 / 4 / 8 10.30 /
// 10.46 / 10.75; N = 28672, K = 1024 7.12 / 6.56 / 6.78; N = 512, K = 16384 3.8 / 4.2 / 6.1.
// The gated block's two outputs are four rows: one row of d = 14336 19.46 (four
// outputs 19.46, one 21.0).
static int dot_rows(int64_t N, int64_t K, bool glu) { return !glu && K <= 2048 && N >= 8192 ? 4 : 2; }
template <int M>
static int launch_dot_m(const Int8Few& p, hipStream_t st) {
  if (p.act >= 0) return launch_dot_r<M, 2, true>(p, st);
  return dot_rows(p.N, p.K, false) == 4 ? launch_dot_r<M, 4, false>(p, st) : launch_dot_r<M, 2, false>(p, st);
}

static int launch_int8_dot(const Int8Few& p, hipStream_t st) {
  switch (p.M) {
    case 1: return launch_dot_m<1>(p, st);
    case 2: return launch_dot_m<2>(p, st);
    case 3: return launch_dot_m<3>(p, st);
    case 4: return p.act >= 0 ? launch_dot_r<4, 2, true>(p, st) : CEK_ERR_UNSUPPORTED;
    default: return CEK_ERR_UNSUPPORTED;
  }
}

// ---- up to 64 rows -----------------------------------------------------------
// Weights and activations stream through LDS rings that loader waves fill with
// direct-to-LDS loads (1 KB: two rows x 512 bytes); eight consumer waves take 64 K
// values of a stage's 512 each over all 16 x 16 blocks of the workgroup (AR rows of a
// x RW of b) and meet in LDS at the end.  One barrier a stage.  Weights from HBM: 16 x 4096 x
// 14336 13.0 us (4.5 TB/s; a read alone 9.8), 37 x 10750 x 2576 10.0 (a read 5.6), 48 x 4096 x
// 4096 8.1.  Beside the read it is the bytes of a that bound them: a CU loads AR rows of a
// beside its RW rows of b.  Activations straight to the consumers' registers (16 rows x 64
// bytes a load) take 15.7 in the place of 13.1 and 11.1 in the place of 8.3.
constexpr int kConsumers = 8;

template <int AR_, int RW_, bool GLU_>
struct Int8Stream {
  static constexpr int AR = AR_, RW = RW_;
  static constexpr bool GLU = GLU_;
  static constexpr int KS = 512, MB = (AR + 15) / 16, NT = (RW + 15) / 16;
  static constexpr int WL = 2, AL = AR >= 64 ? 4 : 2;
  static constexpr int THREADS = 64 * (kConsumers + WL + AL);
  static constexpr int LDSB = AR <= 16 && RW <= 24 ? 81920 : 163840;  // two workgroups per CU, or one
  static constexpr int RING = LDSB - 512;
  static constexpr int ASZ = AR * KS, WSZ = RW * KS, SLOT = ASZ + WSZ;
  static constexpr int AM = ASZ / 1024 / AL, WM = WSZ / 1024 / WL;    // loads per loader wave and stage
  static constexpr int PER = AM > WM ? AM : WM, R0 = RING / SLOT, R1 = R0 > 24 ? 24 : R0;
  static constexpr int R = R1 > 62 / PER + 1 ? 62 / PER + 1 : R1;
  static_assert(AM * AL * 1024 == ASZ && WM * WL * 1024 == WSZ, "loads");
  static_assert(R >= 2 && (!GLU || RW % 8 == 0), "rings; four gate rows beside four up rows");
};

// A loader wave: MINE loads a stage, of the 1 KB pieces who + WAVES m, through a ring of
// R slots SLOT bytes apart.  A slot holds rows of 512 bytes one after another, unit u
// of row r at u ^ (r & 15).  Row offsets vo, this lane's byte offset of its unit within
// the stage ku; units past the row are zeros and no traffic (37 x 10750 x 2576, whose last
// stage holds 16 of 512 values, 10.3 -> 10.1 us).  The wave takes part in the S stage
// barriers: before barrier i stage i has landed, after it stage i - 1's slot is free.
template <int MINE, int WAVES, int R, int SLOT>
__device__ __forceinline__ void int8_stream_load(uint8_t* slots, const uint32_t (&vo)[MINE], const uint32_t (&ku)[MINE],
                                                 int K, int S, int k_first, __amdgpu_buffer_rsrc_t even,
                                                 __amdgpu_buffer_rsrc_t odd, int who) {
  auto issue = [&](int s, int slot) {
    const uint32_t k0 = (uint32_t)(s + k_first >= S ? s + k_first - S : s + k_first) * 512;
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
      const uint32_t off = k0 + ku[m] < (uint32_t)K ? vo[m] + k0 + ku[m] : 0x80000000u;
#if defined(__HIP_DEVICE_COMPILE__)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(m & 1 ? odd : even, (lds_ptr_t)(slots + slot * SLOT + 1024 * (who + WAVES * m)),
                                               16, off, 0, 0, 0);
#endif
    }
  };
#pragma unroll
  for (int s = 0; s < R; ++s)
    if (s < S) issue(s, s);
  if (S >= R) {
    wait_vmcnt<(R - 1) * MINE>();
    bare_barrier();
    int slot = 0;
    for (int s = R; s < S; ++s) {
      wait_vmcnt<(R - 2) * MINE>();
      bare_barrier();
      issue(s, slot);
      slot = slot + 1 == R ? 0 : slot + 1;
    }
  }
  auto drain = [&](auto self, auto rc) {
    constexpr int r = decltype(rc)::value;
    if (S >= R ? r < R - 1 : r < S) {
      wait_vmcnt<r * MINE>();
      bare_barrier();
    }
    if constexpr (r > 0) self(self, std::integral_constant<int, r - 1>{});
  };
  drain(drain, std::integral_constant<int, R - 1>{});
}

template <class C>
__global__ __launch_bounds__(C::THREADS, (C::LDSB > 81920 ? 3 : 6)) void int8_stream_kernel(Int8Few p) {
  constexpr int MB = C::MB, NT = C::NT, R = C::R;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[C::LDSB];
  float* const sw = reinterpret_cast<float*>(smem + C::RING);  // [RW]
  float* const sx = sw + 64;                                   // [M]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  constexpr int RO = C::GLU ? C::RW / 2 : C::RW;               // outputs of a workgroup
  const int n0 = blockIdx.x * RO, K = p.K, S = (K + C::KS - 1) / C::KS;
  const int rows = min(RO, p.N - n0);
  const int k_first = p.N >= 8192 ? (int)((blockIdx.x >> 3) % (unsigned)S) : 0;
  // weight row r of the workgroup: of the gated block four gate rows, their up rows, four more
  // (the weights' loader waves take pairs of rows in turn: an even load is gate, an odd one up)
  auto out_of = [](int r) { return C::GLU ? (r >> 3) * 4 + (r & 3) : r; };

  i4 acc[MB][NT];
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[b][t] = i4{0, 0, 0, 0};

  if (wave >= kConsumers + C::WL) {
    const int who = wave - kConsumers - C::WL;
    uint32_t vo[C::AM], ku[C::AM];
#pragma unroll
    for (int m = 0; m < C::AM; ++m) {
      const int row = 2 * (who + C::AL * m) + (lane >> 5);
      vo[m] = (uint32_t)min(row, p.M - 1) * (uint32_t)K;
      ku[m] = 16u * (uint32_t)((lane & 31) ^ (row & 15));
    }
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.a), 0, (int)((uint32_t)p.M * (uint32_t)K), 0x00020000);
    int8_stream_load<C::AM, C::AL, R, C::SLOT>(smem, vo, ku, K, S, k_first, r, r, who);
  } else if (wave >= kConsumers) {
    const int who = wave - kConsumers;
    uint32_t vo[C::WM], ku[C::WM];
#pragma unroll
    for (int m = 0; m < C::WM; ++m) {
      const int row = 2 * (who + C::WL * m) + (lane >> 5);
      vo[m] = (uint32_t)min(out_of(row), rows - 1) * (uint32_t)K;
      ku[m] = 16u * (uint32_t)((lane & 31) ^ (row & 15));
    }
    auto rsrc = [&](size_t first) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.b + first * K), 0, (int)((uint32_t)rows * (uint32_t)K), 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t rg = rsrc(n0), ru = C::GLU ? rsrc((size_t)p.N + n0) : rg;
    int8_stream_load<C::WM, C::WL, R, C::SLOT>(smem + C::ASZ, vo, ku, K, S, k_first, rg, ru, who);
  } else {
    if (wave == 0 && lane < C::RW) sw[lane] = p.sb[(C::GLU && (lane & 4) ? (size_t)p.N : 0) + min(n0 + out_of(lane), p.N - 1)];
    if (wave == 1 && lane < p.M) sx[lane] = p.sa[lane];
    const int r16 = lane & 15, g = lane >> 4, unit = 4 * wave + g;
    int ao[MB], wo[NT];
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      const int row = min(16 * b + r16, C::AR - 1);
      ao[b] = row * C::KS + 16 * (unit ^ (row & 15));
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = min(16 * t + r16, C::RW - 1);
      wo[t] = C::ASZ + row * C::KS + 16 * (unit ^ (row & 15));
    }
    const uint8_t* at = smem;
    int ks = k_first;
    for (int i = 0; i < S; ++i) {
      lds_barrier();  // stage i has landed; this wave's reads of stage i - 1 are done
      if (ks * C::KS + wave * 64 < K) {
        u4 av[MB], wv[NT];
#pragma unroll
        for (int b = 0; b < MB; ++b) av[b] = *reinterpret_cast<const u4*>(at + ao[b]);
#pragma unroll
        for (int t = 0; t < NT; ++t) wv[t] = *reinterpret_cast<const u4*>(at + wo[t]);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int b = 0; b < MB; ++b) acc[b][t] = mfma_i8(av[b], wv[t], acc[b][t]);
      }
      ks = ks + 1 == S ? 0 : ks + 1;
      at = at + C::SLOT == smem + R * C::SLOT ? smem : at + C::SLOT;
    }
  }

  // The eight waves' sums meet in LDS: D row 4 (lane >> 4) + v of a block is row m of a,
  // column lane & 15 the weight row.
  constexpr int BL = MB * NT;
  static_assert(kConsumers * BL * 1024 <= C::RING, "the sums take the slots' place");
  i4* const red = reinterpret_cast<i4*>(smem);  // [8][BL][64]
  lds_barrier();  // the slots are done with
  if (wave < kConsumers) {
#pragma unroll
    for (int j = 0; j < BL; ++j) red[(wave * BL + j) * 64 + lane] = acc[j / NT][j % NT];
  }
  lds_barrier();
  for (int q = threadIdx.x; q < BL * 64; q += C::THREADS) {
    const int blk = q / 64, r = 16 * (blk % NT) + (q & 15), m0 = 16 * (blk / NT) + 4 * ((q & 63) >> 4);
    const int n = n0 + out_of(r);
    if (r >= C::RW || n >= p.N || m0 >= p.M || (C::GLU && (q & 4))) continue;
    i4 c = red[q], u{0, 0, 0, 0};
    if constexpr (C::GLU) u = red[q + 4];
#pragma unroll
    for (int w = 1; w < kConsumers; ++w) {
      c += red[w * BL * 64 + q];
      if constexpr (C::GLU) u += red[w * BL * 64 + q + 4];
    }
    const float sg = sw[r], su = C::GLU ? sw[r + 4] : 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (m0 + v < p.M) int8_store(p, m0 + v, n, c[v], u[v], sx[m0 + v], sg, su);
  }
}

template <int AR, bool GLU>
static int launch_stream_ar(const Int8Few& p, int rw, hipStream_t st) {
  const unsigned grid = (unsigned)((p.N + (GLU ? rw / 2 : rw) - 1) / (GLU ? rw / 2 : rw));
#define CEK_I8S(RW) int8_stream_kernel<Int8Stream<AR, RW, GLU>><<<grid, (Int8Stream<AR, RW, GLU>::THREADS), 0, st>>>(p)
  switch (rw) {
    case 8: CEK_I8S(8); break;
    case 12:
      if constexpr (!GLU) CEK_I8S(12);
      else return CEK_ERR_UNSUPPORTED;
      break;
    case 16: CEK_I8S(16); break;
    case 24: CEK_I8S(24); break;
    case 32: CEK_I8S(32); break;
    case 40: CEK_I8S(40); break;
    case 48: CEK_I8S(48); break;
    case 56: CEK_I8S(56); break;
    case 64: CEK_I8S(64); break;
    default: return CEK_ERR_UNSUPPORTED;
  }
#undef CEK_I8S
  return check_launch();
}

// Rows of a that a workgroup holds.
static int stream_rows(int64_t M) { return M <= 8 ? 8 : (int)((M + 15) / 16 * 16); }
template <bool GLU>
static int launch_stream_g(const Int8Few& p, int rw, hipStream_t st) {
  switch (stream_rows(p.M)) {
    case 8: return launch_stream_ar<8, GLU>(p, rw, st);
    case 16: return launch_stream_ar<16, GLU>(p, rw, st);
    case 32: return launch_stream_ar<32, GLU>(p, rw, st);
    case 48: return launch_stream_ar<48, GLU>(p, rw, st);
    case 64: return launch_stream_ar<64, GLU>(p, rw, st);
    default: return CEK_ERR_UNSUPPORTED;
  }
}

// Weight rows per workgroup and the launch's time in us: a CU's workgroups cost their
// weight and activation bytes, and each after the first its start and end, less where two
// share a CU (the rings of one cover the other's); no launch takes less than its start and
// the weights at the rate HBM gives.  Fitted to 540 launches over 62 shapes (weights from
// HBM): the pick is 1.5% above the fastest count up to 16 rows.  Above 16 the constants are
// fitted to 66 shapes of 34 to 64 rows, 9% off, for the choice between these kernels and the
// tiles: 0.8% above the faster of the two on average, 40% at worst (34 x 14336 x 8192 by
// tiles 31 to 32 us, by rings 22.4; 64 x 14336 x 4096 19.8 and 16.7).  These are plain
// products; the gated block goes by the same constants (64 x 14336 x 4096 by tiles 29.8, by
// rings 34.4; 40 rows 27.3 and 27.9).
static int stream_plan(int64_t M, int64_t NB, int64_t K, bool glu, double* us) {
  const bool few = M <= 16;
  const double start = few ? 2.61 : 2.97, weight = few ? 0.0234e-3 : 0.0416e-3, act = few ? 0.0103e-3 : 0.0084e-3,
               next = few ? 5.06 : 3.48;
  const int rows[] = {8, 12, 16, 24, 32, 40, 48, 56, 64};
  const int ar = stream_rows(M);
  int best = 0;
  for (int r : rows) {
    if (glu && r == 12) continue;
    const int64_t per_cu = ((NB + r - 1) / r + kCUs - 1) / kCUs;
    const double t = start + (double)per_cu * (r * weight + ar * act) * (double)K +
                     (double)(per_cu - 1) * (few && r <= 24 ? 0.77 : next);
    if (!best || t < *us) {
      *us = t;
      best = r;
    }
  }
  *us = std::max(*us, start + (double)NB * (double)K / 6.0e6);
  return best;
}

// Up to three rows (four of the gated block) v_dot4, us at N = 14336, K = 4096: one row 10.3
// against 12.1 of the rings, three 11.8 against 12.3, four 12.8 against 12.4; the block's
// four 21.9 against 23.2.
static bool int8_dot_takes(int64_t M, bool glu) { return M <= (glu ? 4 : 3); }

bool int8_few_takes(int64_t M, int64_t NB, int64_t K, bool glu, double tile_us) {
  if (M > 64) return false;
  // Up to 32 rows only wide matrices of short rows go to the tiles: there a workgroup of the
  // rings is mostly start and end, and a CU has several.  Rings / tiles, us: 28672 x 512 with
  // 16 rows 7.4 / 6.2, 28672 x 1024 10.3 / 9.0 but 43008 x 1024 14.0 / 15.5; with 32 rows
  // 21504 x 2048 13.7 / 11.8, 131072 x 2048 61 / 54, 43008 x 2048 23.4 / 23.9, 28672 x 4096
  // 25.2 / 26.9; 16384 x 512 4.7 / 5.4.  No limit in K alone is right for all of these: up to
  // 16 rows this one gives K = 1024 to the rings, which costs 28672 and 131072 wide matrices
  // 5 to 14%, and from 17 rows K = 2048 to the tiles, which costs 43008 wide ones 2 to 7%.
  if (M <= 32) return int8_dot_takes(M, glu) || NB <= 16384 || K > (M > 16 ? 2048 : 512);
  double us;
  stream_plan(M, NB, K, glu, &us);
  return us <= tile_us;
}

int int8_few_form(int64_t M, int64_t N, int64_t K, bool glu) {
  if (int8_dot_takes(M, glu)) return 16 * (int)M + dot_rows(N, K, glu);
  double us;
  return 256 * stream_rows(M) + stream_plan(M, glu ? 2 * N : N, K, glu, &us);
}

int launch_int8_few(const Int8Few& p, hipStream_t st) {
  const bool glu = p.act >= 0;
  if (int8_dot_takes(p.M, glu)) return launch_int8_dot(p, st);
  double us;
  const int rw = stream_plan(p.M, glu ? 2 * (int64_t)p.N : p.N, p.K, glu, &us);
  return glu ? launch_stream_g<true>(p, rw, st) : launch_stream_g<false>(p, rw, st);
}

}  // namespace cek
