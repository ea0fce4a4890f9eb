// cek_kv4_attn.hip -- attention over the 4-bit paged key/value cache, gfx950
// (layout and number format: cek_kv4.h).
//
//   out_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i . k_j), j in row i's range
//
// with k = mk + sk (ck - 7.5), v = mv + sv (cv - 7.5) per token and head:
//
//   q . k       = sk (q . ck) + (mk - 7.5 sk) sum(q)
//   sum_j w v   = sum_j (w sv)(cv) - 7.5 sum_j (w sv) + sum_j w mv
//
// so the matrix products run on the codes themselves and the parameters are
// applied to scores and weights, one value a token instead of hd.  Codes enter
// the fp16 MFMA as they lie: a 32-bit word & 0x000F000F is a pair of fp16
// subnormals c 2^-24, & 0x00F000F0 a pair c 2^-20 -- exact, one AND (and a shift
// for every second pair) where a conversion would take three operations.  The
// powers of two are taken back in q (2^-4 for the second kind) and in the sums.
//
// Layout: everything stays in registers.  A wave takes 32 tokens at a time and
// QT tiles of 16 rows (row = query token x query head of the kv head).  It forms
// S^T = K Q^T (MFMA rows: tokens, columns: rows), so that a lane holds eight
// weights of one row, which are -- without a shuffle, since the order within a
// contraction is free -- the operand of O^T = V^T P^T; V's words hold four tokens
// side by side for that.  Each code byte is read once, 1 KB a load instruction.
//
// Weights: with M a running maximum of the exponents and 2^E above every sv so
// far, P = exp2(x - M - E + 9) makes P sv at most 2^9 as it comes and 2^15 with
// the 2^6 that a maximum may lag behind (it moves, and the sums are rescaled,
// only where a score exceeds it by more): fp16 holds P sv to half a step (2^-12
// of the value) down to 2^-23 of the largest.  Sums are fp32; 7.5 sum(P sv) is
// taken by an MFMA over the rounded weights, so that a weight's rounding acts
// on v's distance from its centre alone.
#include <algorithm>
#include <type_traits>

#include "cek_kv4.h"

namespace cek {

struct Kv4AttnArgs {
  const uint16_t* q;
  uint16_t* out;
  const uint8_t* cache;
  const int32_t *tables, *kv_lens, *cu_q;
  float* part;     // split keys: rows of hd sums
  float* part_ml;  // and their (reference exponent, sum of weights)
  int4* meta;      // per query token: first partial row, parts, rows a tile, place in its request
  int64_t T, q_stride, out_stride, table_stride;
  Kv4Dims dm;
  int R, group, max_blocks, window;
  int rows_above, rows_upto;  // this launch serves requests with that many rows
  int target;                 // work items (per kv head) to split the keys into; 0: not split
  int part_row0;              // first partial row of this launch
  int vec_q, vec_out;
  float scale;
};

constexpr int kAttnWaves = 4;
constexpr int kAttnHead = 6, kAttnBase = 9;  // exponents: lag of a maximum, where the largest weight lies
constexpr float kAttnNone = -1e30f;

typedef const __attribute__((address_space(4))) int32_t* const_i32;  // scalar loads

// One request as the work list sees it.
struct Kv4Work {
  int r, q0, rows, kv, n_new, lo, tile, chunk, nch, item0, keys;
};

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ inline int wave_scan_incl(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    if (lane >= off) x += y;
  }
  return x;
}

// Work item -> (request, row tile, part of the keys).  A request has
// ceil(rows / BR) tiles and its keys (from the first that any row sees, down to
// a multiple of 32) in parts of C, the same for the whole call: C = the sum over
// requests of tiles x keys, over `target`, at least 128 and a multiple of 128.
// Every wave of the grid computes the same from the lengths; items of a call
// number at most target + tiles, which is the grid.
template <int BR>
__device__ inline bool kv4_find_work(const Kv4AttnArgs& a, int item, Kv4Work& w) {
  const int lane = threadIdx.x & 63;
  const int64_t reach = (int64_t)a.max_blocks << a.dm.bs_log2;
  auto request = [&](int r, int& q0, int& rows, int& kv, int& n_new, int& lo, int& tiles) {
    q0 = n_new = rows = kv = lo = tiles = 0;
    if (r >= a.R) return;
    q0 = max(0, a.cu_q[r]);
    n_new = (int)min((int64_t)a.cu_q[r + 1], a.T) - q0;
    if (n_new <= 0) return;
    const int64_t n = (int64_t)n_new * a.group;
    if (n <= a.rows_above || n > a.rows_upto) return;
    rows = (int)n;
    kv = (int)min((int64_t)max(a.kv_lens[r], 0), reach);
    lo = a.window > 0 ? max(0, kv - n_new - a.window + 1) & ~31 : 0;
    tiles = (rows + BR - 1) / BR;
  };
  int q0, rows, kv, n_new, lo, tiles;
  int C = INT32_MAX;
  if (a.target > 0) {
    float total = 0.f;
    for (int base = 0; base < a.R; base += 64) {
      request(base + lane, q0, rows, kv, n_new, lo, tiles);
      total += (float)tiles * (float)(kv - lo);
    }
    total = wave_sum(total);
    C = max(1, (int)ceilf(total * 1.001f / ((float)a.target * 128.f))) * 128;
  }
  int first = 0;
  for (int base = 0; base < a.R; base += 64) {
    request(base + lane, q0, rows, kv, n_new, lo, tiles);
    const int nch = a.target > 0 ? max(1, (int)(((unsigned)(kv - lo) + (unsigned)C - 1u) / (unsigned)C)) : 1;
    const int incl = first + wave_scan_incl(tiles * nch);
    const uint64_t above = __ballot(incl > item);
    if (above) {
      const int at = __builtin_ctzll(above);
      auto get = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
      w.r = base + at;
      w.q0 = get(q0);
      w.rows = get(rows);
      w.kv = get(kv);
      w.n_new = get(n_new);
      w.lo = get(lo);
      w.nch = get(nch);
      const int t = get(tiles);
      w.item0 = get(incl) - t * w.nch;
      const int at_tile = uniform((item - w.item0) / w.nch);
      w.tile = t - 1 - at_tile;  // the last rows, which see most keys, first
      w.chunk = item - w.item0 - at_tile * w.nch;
      w.keys = C;
      return true;
    }
    first = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// Parameters of 16 tokens that do not exist.
__device__ const uint8_t kv4_zeros[64] __attribute__((aligned(16))) = {};

__device__ inline uint32_t pack_h2(float a, float b) {
  return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});
}

// KVSPLIT: the workgroup's four waves share QT x 16 rows and take every fourth 32
// tokens each; else each wave has QT x 16 rows of its own and all the tokens.
template <typename T, int HD, int QT, bool KVSPLIT>
__global__ __launch_bounds__(256, 2) void kv4_attn_kernel(Kv4AttnArgs a) {
  constexpr int ND = HD / 32;                    // 32-bit words per lane, part and 16 tokens
  constexpr int NP = HD >= 128 ? HD / 128 : 1;   // parts of a row: 128 values, or 64
  constexpr int NH = HD >= 128 ? 2 : 1;          // runs of four values per lane and part
  constexpr int PW = HD / NP;                    // values of a part
  constexpr int BR = QT * 16 * (KVSPLIT ? 1 : kAttnWaves);
  constexpr int LSTR = HD + 4;                   // LDS row stride: rows 4 banks apart
  __shared__ float lds_o[KVSPLIT ? kAttnWaves * 16 * LSTR : 1];
  __shared__ float lds_ml[KVSPLIT ? kAttnWaves * 16 * 2 : 1];

  Kv4Work w;
  if (!kv4_find_work<BR>(a, blockIdx.x, w)) return;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.y;
  const int bs = 1 << a.dm.bs_log2;
  const int row0 = w.tile * BR + (KVSPLIT ? 0 : wave * QT * 16);  // this wave's first row in the request

  if (a.meta && kvh == 0 && w.chunk == 0) {
    // for the launch that joins the parts
    const int t0 = w.tile * BR / a.group, t1 = min(w.rows, (w.tile + 1) * BR);
    for (int t = t0 + (int)threadIdx.x; t * a.group < t1; t += 256)
      a.meta[w.q0 + t] = int4{a.part_row0 + w.item0 * a.dm.n_kv * BR, w.nch, BR, t};
  }

  // ---- q: this lane's 16-bit values of row c of each tile, in the order of K's words ----
  u4 qf[QT][ND];        // MFMA operands
  float qsum[QT], qmul[QT];
  int pos[QT];          // position of the row; padding rows see everything
  int pmin = INT32_MAX, pmax = -1;  // over this wave's rows
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int rr = row0 + i * 16 + c;
    const bool real = rr < w.rows;
    const int t = rr / a.group, h = kvh * a.group + rr % a.group;
    const uint16_t* src = a.q + (int64_t)(w.q0 + (real ? t : 0)) * a.q_stride + (int64_t)(real ? h : 0) * HD;
    pos[i] = real ? w.kv - w.n_new + t : INT32_MAX - 1;
    if (row0 + i * 16 < w.rows) {
      // uniform: rows are in order of position
      pmin = uniform(min(pmin, w.kv - w.n_new + (row0 + i * 16) / a.group));
      pmax = uniform(max(pmax, w.kv - w.n_new + (min(row0 + i * 16 + 16, w.rows) - 1) / a.group));
    }
    uint32_t raw[ND][4];
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      const int d0 = (n / (PW / 32)) * PW + g * (PW / 4) + (n % (PW / 32)) * 8;
      if (a.vec_q) {
        const u4 x = load_u4(src + d0);
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[n][e] = real ? x[e] : 0;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          raw[n][e] = real ? (uint32_t)src[d0 + 2 * e] | ((uint32_t)src[d0 + 2 * e + 1] << 16) : 0;
      }
    }
    float top = 0.f;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        top = fmaxf(top, fmaxf(fabsf(T::to_f32(raw[n][e] & 0xFFFF)), fabsf(T::to_f32(raw[n][e] >> 16))));
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    // the row times 2^k, its largest value in 2^13 .. 2^14: exact in fp16 down to 2^-33 of it
    int k = 0;
    if (top > 0.f) k = min(120, 140 - (int)((__float_as_uint(top) >> 23) & 255));
    const float up = ldexpf(1.f, k);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = T::to_f32(raw[n][e] & 0xFFFF) * up;
        f[2 * e + 1] = T::to_f32(raw[n][e] >> 16) * up;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += f[e];
      // word & 0x000F000F: values 0, 4; & 0x00F000F0: 1, 5 (16 c); the same of word >> 8: 2, 6 and 3, 7
      qf[i][n] = u4{pack_h2(f[0], f[4]), pack_h2(f[1] * 0.0625f, f[5] * 0.0625f), pack_h2(f[2], f[6]),
                    pack_h2(f[3] * 0.0625f, f[7] * 0.0625f)};
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    qsum[i] = sum * 0x1p-24f;
    qmul[i] = ldexpf(a.scale * 1.4426950408889634f, 24 - k);
  }

  // ---- the range of keys ----
  const int window = a.window > 0 ? a.window : INT32_MAX;  // pos - window stays in range
  const int t_lo = a.window > 0 ? max(0, pmin - a.window + 1) & ~31 : 0;
  const int begin = uniform((w.nch > 1 ? max(t_lo, w.lo + w.chunk * w.keys) : t_lo) + (KVSPLIT ? 32 * wave : 0));
  const int end = uniform(
      w.nch > 1 ? (int)min((int64_t)pmax + 1, (int64_t)w.lo + ((int64_t)w.chunk + 1) * w.keys) : pmax + 1);
  constexpr int STEP = KVSPLIT ? 32 * kAttnWaves : 32;

  f4 o[QT][NP][NH][4];
  f4 wsum[QT];
  float l[QT], z[QT], m[QT], ref[QT];
  int ev = -80;
  float sv_top = -1.f;  // 2^ev, or -1 before the first tokens
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    l[i] = z[i] = 0.f;
    m[i] = ref[i] = kAttnNone;
    wsum[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NP * NH * 4; ++x) o[i][x / (NH * 4)][x / 4 % NH][x % 4] = f4{0.f, 0.f, 0.f, 0.f};
  }

  const uint8_t* head = a.cache + (int64_t)kvh * kv4_head_bytes(bs, HD);
  const uint32_t k_lane = c * (HD / 2) + g * (PW / 8);
  const uint32_t v_lane = kv4_v_codes(bs, HD) + g * HD * 2 + c * (PW / 8);
  const uint32_t kp_lane = kv4_k_params(bs, HD) + 16 * g;
  const uint32_t vp_lane = kv4_v_params(bs, HD) + 16 * g;
  const const_i32 table = (const_i32)(uintptr_t)(a.tables + (int64_t)w.r * a.table_stride);

  struct Blocks { int b[2]; };
  // the blocks of 32 tokens; behind the last key (a half of them may lie there) none
  auto blocks_of = [&](int t0) {
    Blocks x;
    x.b[0] = uniform(table[t0 >> a.dm.bs_log2]);
    x.b[1] = uniform(table[min(t0 + 16, w.kv - 1) >> a.dm.bs_log2]);
    if (t0 + 16 >= w.kv) x.b[1] = -1;
    return x;
  };
  // A block outside the cache holds no token: block 0 is read in its place.
  auto at_block = [&](int t0, const Blocks& x, int i, int& tok) {
    const int b = x.b[i];
    tok = (t0 + 16 * i) & (bs - 1);
    return head + (int64_t)(b < 0 || b >= a.dm.num_blocks ? 0 : b) * a.dm.block_stride;
  };
  auto load_codes = [&](const uint8_t* base, uint32_t at, uint32_t (&to)[ND], uint32_t part) {
    if constexpr (HD == 64) {
      const uint2 x = *reinterpret_cast<const uint2*>(base + at);
      to[0] = x.x, to[1] = x.y;
    } else {
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const u4 x = load_u4(base + p * part + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) to[4 * p + e] = x[e];
      }
    }
  };
  uint32_t kc[2][ND], vc[2][ND];  // the codes of 32 tokens, 16 and 16
  u4 kp[2], vp[2];                // their parameters, of tokens 4 g ..
  float none[2];                  // 0, or -infinity where the block lies outside the cache
  auto load_k = [&](int t0, const Blocks& x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int tok;
      const uint8_t* base = at_block(t0, x, i, tok);
      load_codes(base + tok * (HD / 2), k_lane, kc[i], PW / 2);  // 64 bytes of a row and part of 128 values
    }
  };
  auto load_v = [&](int t0, const Blocks& x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int tok;
      const uint8_t* base = at_block(t0, x, i, tok);
      load_codes(base + tok * (HD / 2), v_lane, vc[i], PW * 2);  // 256 bytes of four tokens and part
    }
  };
  auto load_params = [&](int t0, const Blocks& x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int tok;
      const uint8_t* base = at_block(t0, x, i, tok) + 4 * tok;
      const bool out = x.b[i] < 0 || x.b[i] >= a.dm.num_blocks;
      // tokens that do not exist have parameters 0, whatever lies in block 0
      kp[i] = load_u4(out ? kv4_zeros + 16 * g : base + kp_lane);
      vp[i] = load_u4(out ? kv4_zeros + 16 * g : base + vp_lane);
      none[i] = out ? -INFINITY : 0.f;
    }
  };

  auto sees = [&](int i, int t0, int h, int e) {  // row c of tile i the token 16 h + 4 g + e at t0
    const int t = t0 + 16 * h + 4 * g + e;
    return (t <= pos[i]) & (t < end) & (t > pos[i] - window);  // no branches
  };

  // Scores of 32 tokens: x (exponents / qmul), their maxima xm and that of the V steps.
  float x[QT][2][4], xm[QT], top;
  auto scores = [&](int t0, auto mask) {
    constexpr bool masked = decltype(mask)::value;
    if constexpr (masked) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool out = t0 + 16 * h + 4 * g + e >= end;  // no token: whatever lies there
          kp[h][e] = out ? 0u : kp[h][e];
          vp[h][e] = out ? 0u : vp[h][e];
        }
    }
    // S^T: tokens 16 h + 4 g + e of row c
    f4 acc[QT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < QT; ++i) acc[i][h] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        const uint32_t y = kc[h][n], y8 = y >> 8;
        const u4 f = u4{y & 0x000F000Fu, y & 0x00F000F0u, y8 & 0x000F000Fu, y8 & 0x00F000F0u};
#pragma unroll
        for (int i = 0; i < QT; ++i) acc[i][h] = mfma16x16x32<F16>(f, qf[i][n], acc[i][h]);
      }
    }
    top = -1.f;
#pragma unroll
    for (int i = 0; i < QT; ++i) xm[i] = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float xh[QT];
#pragma unroll
      for (int i = 0; i < QT; ++i) xh[i] = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float sk = kv4_step(kp[h][e]), mk = fmaf(-7.5f, sk, kv4_centre(kp[h][e]));
        top = fmaxf(top, kv4_step(vp[h][e]));
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          x[i][h][e] = fmaf(sk, acc[i][h][e], mk * qsum[i]);
          if constexpr (masked) x[i][h][e] = sees(i, t0, h, e) ? x[i][h][e] : -INFINITY;
          xh[i] = fmaxf(xh[i], x[i][h][e]);
        }
      }
#pragma unroll
      for (int i = 0; i < QT; ++i) xm[i] = fmaxf(xm[i], xh[i] + none[h]);
    }
  };
  auto grows = [&]() {
    bool y = top > sv_top;
#pragma unroll
    for (int i = 0; i < QT; ++i) y = y | (xm[i] * qmul[i] > m[i] + (float)kAttnHead);
    return __any(y);
  };
  // New references, and the sums so far brought to them.
  auto rescale = [&]() {
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    ev = max(ev, (int)((__float_as_uint(fmaxf(top, 0.f)) >> 23) & 255) - 126);
    sv_top = __uint_as_float((uint32_t)(ev + 127) << 23);
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      float t = fmaxf(m[i], xm[i] * qmul[i]);
      t = fmaxf(t, __shfl_xor(t, 16, 64));
      t = fmaxf(t, __shfl_xor(t, 32, 64));
      m[i] = t;
      const float nr = t + (float)(ev - kAttnBase);
      const float f = __builtin_amdgcn_exp2f(ref[i] - nr);
      ref[i] = nr;
      l[i] *= f;
      z[i] *= f;
      wsum[i] *= f;
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int b = 0; b < 4; ++b) o[i][p][h][b] *= f;
    }
  };
  // Weights and the sums over them.  As soon as the registers of one kind of
  // operand are used, the next tile's (at t1, in blocks nx) are loaded into them.
  auto accumulate = [&](int t0, int t1, const Blocks& nx, auto mask) {
    constexpr bool masked = decltype(mask)::value;
    load_k(t1, nx);
    u4 pf[QT];  // the weights times sv, fp16: tokens 4 g .. of both halves
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float pv[QT][4], off[QT];
#pragma unroll
      for (int i = 0; i < QT; ++i) off[i] = none[h] - ref[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float sv = kv4_step(vp[h][e]), mv = kv4_centre(vp[h][e]);
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          const float p = __builtin_amdgcn_exp2f(fmaf(x[i][h][e], qmul[i], off[i]));
          pv[i][e] = p * sv;
          if constexpr (masked) {
            const bool ok = sees(i, t0, h, e);
            l[i] += ok ? p : 0.f;
            z[i] = ok ? fmaf(p, mv, z[i]) : z[i];
            pv[i][e] = ok ? pv[i][e] : 0.f;
          } else {
            l[i] += p;
            z[i] = fmaf(p, mv, z[i]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        pf[i][2 * h] = pack_h2(pv[i][0], pv[i][1]);
        pf[i][2 * h + 1] = pack_h2(pv[i][2], pv[i][3]);
      }
    }
    load_params(t1, nx);
    // O^T: values 4 (NH c + h) + b of each part, in rows c
    const u4 halves = u4{0x47804780u, 0x47804780u, 0x47804780u, 0x47804780u};  // 7.5
#pragma unroll
    for (int i = 0; i < QT; ++i) wsum[i] = mfma16x16x32<F16>(halves, pf[i], wsum[i]);
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int n = (p * NH + h) * 2;
        const uint32_t a0 = vc[0][n], a1 = vc[0][n + 1], b0 = vc[1][n], b1 = vc[1][n + 1];
        u4 f[4];
        f[0] = u4{a0 & 0x000F000Fu, a1 & 0x000F000Fu, b0 & 0x000F000Fu, b1 & 0x000F000Fu};
        f[1] = u4{a0 & 0x00F000F0u, a1 & 0x00F000F0u, b0 & 0x00F000F0u, b1 & 0x00F000F0u};
        f[2] = u4{(a0 >> 8) & 0x000F000Fu, (a1 >> 8) & 0x000F000Fu, (b0 >> 8) & 0x000F000Fu, (b1 >> 8) & 0x000F000Fu};
        f[3] = u4{(a0 >> 8) & 0x00F000F0u, (a1 >> 8) & 0x00F000F0u, (b0 >> 8) & 0x00F000F0u, (b1 >> 8) & 0x00F000F0u};
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int i = 0; i < QT; ++i) o[i][p][h][b] = mfma16x16x32<F16>(f[b], pf[i], o[i][p][h][b]);
      }
    load_v(t1, nx);
  };

  // Tiles in order: those that the window cuts, those that every row sees whole (up
  // to `full`), those that the rows' own positions or the end cut.  The cut ones
  // mask, and rescale without asking.
  if (begin < end) {
    const int last = begin + (end - 1 - begin) / STEP * STEP;
    const int full = uniform(min(pmin - 31, end - 32));
    Blocks nb = blocks_of(begin);
    load_k(begin, nb);
    load_params(begin, nb);
    load_v(begin, nb);
    nb = blocks_of(min(begin + STEP, last));
    int t0 = begin;
    auto advance = [&](auto mask) {
      const Blocks nx = nb;
      nb = blocks_of(min(t0 + 2 * STEP, last));  // a tile ahead of the loads that need them
      accumulate(t0, min(t0 + STEP, last), nx, mask);
      t0 += STEP;
    };
    auto cut_to = [&](int to) {
      while (t0 < to) {
        scores(t0, std::true_type{});
        rescale();
        advance(std::true_type{});
      }
    };
    if (a.window > 0) cut_to(min(end, pmax - a.window + 1));
    while (t0 <= full) {
      scores(t0, std::false_type{});
      if (grows()) rescale();
      advance(std::false_type{});
    }
    cut_to(end);
  }

  // ---- the end: sums over the lanes of a row, parts to the workspace, rows out ----
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    l[i] += __shfl_xor(l[i], 16, 64);
    l[i] += __shfl_xor(l[i], 32, 64);
    z[i] += __shfl_xor(z[i], 16, 64);
    z[i] += __shfl_xor(z[i], 32, 64);
    const float off = z[i] - wsum[i][0];  // every row of the MFMA's result holds 7.5 sum(P sv)
    // lane (c, g): values p PW + g PW / 4 + 4 NH e + 4 h + b of row c
    auto value = [&](int p, int e, int h, int b) {
      return fmaf(o[i][p][h][b][e], b & 1 ? 0x1p20f : 0x1p24f, off);
    };
    if constexpr (KVSPLIT) {
      if (i > 0) __syncthreads();
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int h = 0; h < NH; ++h)
            *reinterpret_cast<f4*>(&lds_o[(wave * 16 + c) * LSTR + p * PW + g * (PW / 4) + 4 * NH * e + 4 * h]) =
                f4{value(p, e, h, 0), value(p, e, h, 1), value(p, e, h, 2), value(p, e, h, 3)};
      if (g == 0) {
        lds_ml[(wave * 16 + c) * 2] = ref[i];
        lds_ml[(wave * 16 + c) * 2 + 1] = l[i];
      }
      __syncthreads();
      // thread (row, sixteenth of the row)
      const int row = threadIdx.x >> 4, seg = threadIdx.x & 15;
      const int rr = w.tile * BR + i * 16 + row;
      float top = kAttnNone, den = 0.f, y[HD / 16] = {};
#pragma unroll
      for (int v = 0; v < kAttnWaves; ++v) top = fmaxf(top, lds_ml[(v * 16 + row) * 2]);
#pragma unroll
      for (int v = 0; v < kAttnWaves; ++v) {
        const float lv = lds_ml[(v * 16 + row) * 2 + 1];
        const float f = __builtin_amdgcn_exp2f(lds_ml[(v * 16 + row) * 2] - top);
        den = fmaf(lv, f, den);
#pragma unroll
        for (int e = 0; e < HD / 16; e += 4) {
          const f4 s = *reinterpret_cast<const f4*>(&lds_o[(v * 16 + row) * LSTR + seg * (HD / 16) + e]);
#pragma unroll
          for (int b = 0; b < 4; ++b) y[e + b] = fmaf(s[b], f, y[e + b]);
        }
      }
      if (rr < w.rows) {
        if (w.nch > 1) {
          const int64_t pr = a.part_row0 + ((int64_t)(w.item0 + w.tile * w.nch + w.chunk) * a.dm.n_kv + kvh) * BR + i * 16 + row;
#pragma unroll
          for (int e = 0; e < HD / 16; e += 4)
            *reinterpret_cast<f4*>(a.part + pr * HD + seg * (HD / 16) + e) = f4{y[e], y[e + 1], y[e + 2], y[e + 3]};
          if (seg == 0) {
            a.part_ml[2 * pr] = top;
            a.part_ml[2 * pr + 1] = den;
          }
        } else {
          const float inv = den != 0.f ? 1.0f / den : 0.f;
          uint16_t* dst = a.out + (int64_t)(w.q0 + rr / a.group) * a.out_stride +
                          (int64_t)(kvh * a.group + rr % a.group) * HD + seg * (HD / 16);
          uint32_t u[HD / 32];
#pragma unroll
          for (int e = 0; e < HD / 32; ++e)
            u[e] = (uint32_t)T::from_f32(den != 0.f ? y[2 * e] * inv : 0.f) |
                   ((uint32_t)T::from_f32(den != 0.f ? y[2 * e + 1] * inv : 0.f) << 16);
          if (a.vec_out) {
#pragma unroll
            for (int e = 0; e < HD / 32; e += 2) *reinterpret_cast<uint2*>(dst + 2 * e) = uint2{u[e], u[e + 1]};
          } else {
#pragma unroll
            for (int e = 0; e < HD / 16; ++e) dst[e] = (uint16_t)(u[e / 2] >> (16 * (e & 1)));
          }
        }
      }
    } else {
      const int rr = row0 + i * 16 + c;
      if (rr < w.rows) {
        if (w.nch > 1) {
          const int64_t pr = a.part_row0 + ((int64_t)(w.item0 + w.tile * w.nch + w.chunk) * a.dm.n_kv + kvh) * BR +
                             wave * QT * 16 + i * 16 + c;
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int h = 0; h < NH; ++h)
                *reinterpret_cast<f4*>(a.part + pr * HD + p * PW + g * (PW / 4) + 4 * NH * e + 4 * h) =
                    f4{value(p, e, h, 0), value(p, e, h, 1), value(p, e, h, 2), value(p, e, h, 3)};
          if (g == 0) {
            a.part_ml[2 * pr] = ref[i];
            a.part_ml[2 * pr + 1] = l[i];
          }
        } else {
          const float inv = l[i] != 0.f ? 1.0f / l[i] : 0.f;
          uint16_t* dst = a.out + (int64_t)(w.q0 + rr / a.group) * a.out_stride +
                          (int64_t)(kvh * a.group + rr % a.group) * HD + g * (PW / 4);
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int h = 0; h < NH; ++h) {
                uint16_t y[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) y[b] = T::from_f32(l[i] != 0.f ? value(p, e, h, b) * inv : 0.f);
                uint16_t* to = dst + p * PW + 4 * NH * e + 4 * h;
                if (a.vec_out) {
                  *reinterpret_cast<uint2*>(to) =
                      uint2{(uint32_t)y[0] | ((uint32_t)y[1] << 16), (uint32_t)y[2] | ((uint32_t)y[3] << 16)};
                } else {
#pragma unroll
                  for (int b = 0; b < 4; ++b) to[b] = y[b];
                }
              }
        }
      }
    }
  }
}

// Joins the parts of a row: one workgroup per (query token, query head), its waves
// taking every fourth part.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv4_attn_join_kernel(Kv4AttnArgs a) {
  constexpr int E = HD / 64;
  const int t = blockIdx.x, h = blockIdx.y;
  if (t < a.cu_q[0] || t >= a.cu_q[a.R]) return;
  const int4 mt = a.meta[t];
  const int nch = mt.y, BR = mt.z;
  if (nch <= 1) return;
  const int rr = mt.w * a.group + h % a.group, tile = rr / BR;
  const int64_t pr0 = mt.x + ((int64_t)tile * nch * a.dm.n_kv + h / a.group) * BR + rr % BR;
  const int64_t step = (int64_t)a.dm.n_kv * BR;
  __shared__ float so[kAttnWaves][HD], sl[kAttnWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float top = kAttnNone;
  for (int p = lane; p < nch; p += 64) top = fmaxf(top, a.part_ml[2 * (pr0 + p * step)]);
  top = wave_max(top);
  float den = 0.f, y[E] = {};
#pragma unroll 4
  for (int p = wave; p < nch; p += kAttnWaves) {
    const int64_t pr = pr0 + p * step;
    const float lp = a.part_ml[2 * pr + 1];
    const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * pr] - top);
    den = fmaf(lp, f, den);
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = fmaf(a.part[pr * HD + lane * E + e], f, y[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[wave][lane * E + e] = y[e];
  if (lane == 0) sl[wave] = den;
  __syncthreads();
  den = sl[0] + sl[1] + sl[2] + sl[3];
  for (int d = threadIdx.x; d < HD; d += 256) {
    const float v = so[0][d] + so[1][d] + so[2][d] + so[3][d];
    a.out[(int64_t)t * a.out_stride + (int64_t)h * HD + d] = T::from_f32(den != 0.f ? v / den : 0.f);
  }
}

}  // namespace cek

using namespace cek;

namespace {

// What the host knows of a call: which kernels, their tiles and how the keys are
// split.  Requests with more than kAttnFewRows rows (query tokens x heads of a kv
// head) go to the kernel whose waves have rows of their own.
constexpr int kAttnFewRows = 64;
constexpr int kAttnSplitWgs = 512;  // workgroups to split the keys for

struct AttnPlan {
  bool few, many;
  int qt_few, qt_many;
  int64_t items_few, items_many;  // bounds of the work items per kv head
  int target_few, target_many;    // 0: the keys stay whole
  int64_t part_rows_few, part_rows;
  int64_t bytes;
};

AttnPlan attn_plan(int64_t T, int64_t R, int64_t n_q, int64_t n_kv, int64_t hd, int64_t max_q_len, int64_t max_kv_len) {
  AttnPlan p{};
  const int64_t group = n_q / n_kv;
  if (max_q_len <= 0 || max_q_len > T) max_q_len = T;
  const int64_t rows = max_q_len * group;
  p.many = rows > kAttnFewRows;
  p.few = !p.many || R > 1;
  const int64_t few_rows = p.many ? group : rows;  // of a request, as a rule
  p.qt_few = few_rows <= 16 || hd == 256 ? 1 : 2;
  p.qt_many = hd == 256 ? 1 : 2;
  const int64_t seqs = std::min(R, T);
  p.items_few = T * group / (16 * p.qt_few) + seqs;
  if (p.many) p.items_few = std::min(p.items_few, seqs * (kAttnFewRows / (16 * p.qt_few)));
  p.items_many = T * group / (64 * p.qt_many) + seqs;
  const bool long_keys = max_kv_len <= 0 || max_kv_len > 256;
  auto target = [&](int64_t items) {
    return long_keys && items * n_kv < 4 * kAttnSplitWgs ? (int)std::max<int64_t>(1, (kAttnSplitWgs + n_kv - 1) / n_kv) : 0;
  };
  if (p.few) p.target_few = target(p.many ? seqs : p.items_few);
  if (p.many) p.target_many = target(p.items_many);
  p.items_few += p.target_few;
  p.items_many += p.target_many;
  p.part_rows_few = p.target_few ? p.items_few * n_kv * 16 * p.qt_few : 0;
  p.part_rows = p.part_rows_few + (p.target_many ? p.items_many * n_kv * 64 * p.qt_many : 0);
  if (p.target_few || p.target_many) p.bytes = p.part_rows * (hd + 2) * 4 + T * 16;
  return p;
}

template <typename T, int HD>
void launch_attn(const AttnPlan& p, Kv4AttnArgs a, int64_t n_kv, int64_t n_q, hipStream_t st) {
  if (p.few) {
    Kv4AttnArgs b = a;
    b.rows_above = 0;
    b.rows_upto = p.many ? kAttnFewRows : INT32_MAX;
    b.target = p.target_few;
    b.part_row0 = 0;
    const dim3 grid((unsigned)p.items_few, (unsigned)n_kv);
    if (p.qt_few == 1) kv4_attn_kernel<T, HD, 1, true><<<grid, 256, 0, st>>>(b);
    else if constexpr (HD != 256) kv4_attn_kernel<T, HD, 2, true><<<grid, 256, 0, st>>>(b);
  }
  if (p.many) {
    Kv4AttnArgs b = a;
    b.rows_above = p.few ? kAttnFewRows : 0;
    b.rows_upto = INT32_MAX;
    b.target = p.target_many;
    b.part_row0 = (int)p.part_rows_few;
    const dim3 grid((unsigned)p.items_many, (unsigned)n_kv);
    kv4_attn_kernel<T, HD, HD == 256 ? 1 : 2, false><<<grid, 256, 0, st>>>(b);
  }
  if (p.target_few || p.target_many) {
    kv4_attn_join_kernel<T, HD><<<dim3((unsigned)a.T, (unsigned)n_q), 256, 0, st>>>(a);
  }
}

}  // namespace

extern "C" int64_t cek_kv4_attention_workspace_size(int64_t T, int64_t R, int64_t n_q, int64_t n_kv, int64_t hd,
                                                    int64_t max_q_len, int64_t max_kv_len) {
  if (T <= 0 || R <= 0 || n_kv <= 0 || n_q <= 0 || n_q % n_kv || (hd != 64 && hd != 128 && hd != 256)) return 0;
  return attn_plan(T, R, n_q, n_kv, hd, max_q_len, max_kv_len).bytes;
}

extern "C" int cek_kv4_attention(const void* q, const void* cache, const int32_t* block_tables, const int32_t* kv_lens,
                                 const int32_t* cu_q, void* out, int64_t T, int64_t R, int64_t n_q, int64_t n_kv,
                                 int64_t hd, int64_t block_size, int64_t num_blocks, int64_t q_stride, int64_t out_stride,
                                 int64_t block_stride, int64_t table_stride, int64_t max_blocks, float scale,
                                 int64_t max_q_len, int64_t max_kv_len, int64_t window, int io_dtype, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  Kv4AttnArgs a{};
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
  if (T * (n_q / n_kv) > INT32_MAX / 2) return CEK_ERR_UNSUPPORTED;  // rows of a kv head
  if (workspace_bytes < 0 || (workspace && !aligned(workspace, 16))) return CEK_ERR_INVALID;
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
  a.group = (int)(n_q / n_kv);
  a.max_blocks = (int)max_blocks;
  a.window = (int)window;
  a.scale = scale;
  a.vec_q = aligned(q, 16) && q_stride % 8 == 0;
  a.vec_out = aligned(out, 8) && out_stride % 4 == 0;
  AttnPlan p = attn_plan(T, R, n_q, n_kv, hd, max_q_len, max_kv_len);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) {
    p.items_few -= p.target_few;
    p.items_many -= p.target_many;
    p.target_few = p.target_many = 0;
  } else if (p.bytes > 0) {
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + p.part_rows * hd;
    a.meta = reinterpret_cast<int4*>(a.part_ml + p.part_rows * 2);
  }
  if (p.items_few > INT32_MAX || p.items_many > INT32_MAX || p.part_rows > INT32_MAX) return CEK_ERR_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
#define CEK_GO(D)                                                       \
  do {                                                                  \
    if (io_dtype == CEK_F16) launch_attn<F16, D>(p, a, n_kv, n_q, st);  \
    else launch_attn<BF16, D>(p, a, n_kv, n_q, st);                     \
  } while (0)
  CEK_KV4_HD(CEK_GO);
#undef CEK_GO
  return check_launch();
}
