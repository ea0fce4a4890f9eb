// cek_kv4_attn_rows.hip -- attention over the 4-bit cache for many rows a request
// (prompt chunks), gfx950.  The mathematics is cek_kv4_attn.hip's.
//
// What bounds it: arithmetic.  Per 16 rows and 32 tokens the matrix products take
// 272 cycles of a SIMD (17 MFMA), the softmax between them about 70 vector
// operations and 8 exponentials, 370.  Unpacking codes and parameters (130 more)
// does not depend on the rows: a workgroup of four waves, each with QT x 16 rows of
// its own, does it once for all of them.  The tokens come in stages of 64 (32 at head
// size 256); the waves load a share of a stage's codes two stages ahead, unpack it
// one stage ahead into LDS, as the operands the MFMA takes and in their order (so
// that every LDS access is 16 bytes a lane in a row), and meet at one barrier a
// stage.  Two workgroups a CU: while one's waves are in the products the other's
// may be in the softmax.
//
// Four chunks of 1900 tokens on 1900 .. 4100 keys, 32 / 8 heads of 128, fp16: 415 us,
// 639 TFLOP/s.  Of a SIMD's cycles the matrix cores are busy 27%, vector instructions
// 48% and exponentials 10%, and hardly at the same time: 85% together.  (With one
// power of two for all rows of a tile, which saves a multiplication a score but mixes
// the rows' ranges, 394.)  No gain came from priorities for the products, from products
// and softmax of different rows interleaved, from fewer maxima, nor from the next
// product's operands read ahead; the largest step of 32 tokens found while unpacking,
// once for all waves, cost 12 us.
#include <type_traits>

#include "cek_kv4_attn.h"

namespace cek {

template <typename T, int HD, int QT>
__global__ __launch_bounds__(256, 2) void kv4_attn_rows_kernel(Kv4AttnArgs a) {
  constexpr int ND = HD / 32;                   // K operands of 16 tokens (32 values each)
  constexpr int NP = HD >= 128 ? HD / 128 : 1;  // parts of a row: 128 values, or 64
  constexpr int NH = HD >= 128 ? 2 : 1;         // runs of four values per lane and part
  constexpr int PW = HD / NP;                   // values of a part
  constexpr int KW = PW / 32;                   // K words of a lane, part and 16 tokens
  constexpr int ST = HD == 256 ? 32 : 64;       // tokens of a stage
  constexpr int NS = ST / 16, NG = ST / 32;     // runs of 16 and of 32
  constexpr int NV = NP * NH * 4;               // V operands of 32 tokens
  constexpr int BR = QT * 16 * kAttnWaves;
  static_assert(BR == attn_rows_br(HD), "rows of a tile");
  __shared__ u4 k_op[2][NS * ND][64], v_op[2][NG * NV][64];
  __shared__ float par[2][4][ST];  // K step and offset, V step and centre, of a stage's tokens
  __shared__ float gone[2][NS];    // -infinity for 16 tokens in no block

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  // heads side by side: the tiles that see most keys first, of all heads
  const int wg = uniform((int)(blockIdx.x / (unsigned)a.dm.n_kv)), kvh = blockIdx.x - wg * a.dm.n_kv;
  const int bs = 1 << a.dm.bs_log2;
  Kv4List<BR, 1> list{a};
  const auto mine = list.request(lane);
  int u = wg, u_end = u + 1;
  if (a.wgs > 0) {
    // (costs and leads made a chunk of 1000 on 4000 keys slower, by 2 .. 7 us of 71)
    list.share(mine, list.unit_for(mine, a.wgs, 256, 512), 0);
    list.deal(a.wgs, 0);
    u = list.begin_of(wg);
    u_end = list.begin_of(wg + 1);
  }
  for (Kv4Work w; u < u_end && list.find(mine, u, u_end, w); u += w.span) {
  if (w.units == 0) continue;
  const int row0 = w.tile * BR + wave * QT * 16;  // this wave's first row in the request
  // Partial rows: of a tile's first stretch in 2 wg + 1, of the others in 2 wg.
  const bool whole = w.units == w.all;
  const int64_t part0 = a.part_row0 + ((int64_t)(2 * wg + (w.unit == 0)) * a.dm.n_kv + kvh) * BR;
  if (a.meta && kvh == 0 && w.unit == 0 && (int)threadIdx.x < BR) {
    // for the launch that joins the parts: the first one's row and their number
    const int rr = w.tile * BR + (int)threadIdx.x;
    const int parts = whole ? 1 : list.owner_of(w.first + w.all - 1) - wg + 1;
    if (rr < w.rows) a.meta[(int64_t)w.q0 * a.group + rr] = int4{(int)part0 + (int)threadIdx.x, parts, a.dm.n_kv * BR, BR};
  }

  // ---- rows and the range of keys: the wave's, and the workgroup's ----
  int pos[QT];          // position of the row; padding rows see everything
  const uint16_t* qsrc[QT];
  bool real[QT];
  auto pos_of = [&](int rr) { return kv4_pos(w.kv, w.n_new, rr / a.group); };
  const int tile_end = min(w.rows, (w.tile + 1) * BR), wave_end = min(tile_end, row0 + QT * 16);
  const int pmin = uniform(row0 < w.rows ? pos_of(row0) : INT32_MAX - 1), pmax = uniform(row0 < w.rows ? pos_of(wave_end - 1) : -1);
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int rr = row0 + i * 16 + c;
    real[i] = rr < w.rows;
    const int t = rr / a.group, h = kvh * a.group + rr % a.group;
    qsrc[i] = a.q + (int64_t)(w.q0 + (real[i] ? t : 0)) * a.q_stride + (int64_t)(real[i] ? h : 0) * HD;
    pos[i] = real[i] ? kv4_pos(w.kv, w.n_new, t) : INT32_MAX - 1;
  }
  const int window = a.window > 0 ? a.window : INT32_MAX;  // pos - window stays in range
  const int first_pos = uniform(pos_of(w.tile * BR)), last_pos = uniform(pos_of(tile_end - 1));
  const int t_lo = a.window > 0 ? max(0, first_pos - a.window + 1) & ~31 : 0;
  const int begin = uniform(list.len ? max(t_lo, w.lo + w.unit * list.len) : t_lo);
  const int end = uniform(
      list.len ? (int)min((int64_t)last_pos + 1, (int64_t)w.lo + (int64_t)(w.unit + w.units) * list.len) : last_pos + 1);

  // ---- q: 16-bit values on their way ----
  uint32_t raw[QT][ND][4];
#pragma unroll
  for (int i = 0; i < QT; ++i)
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      const int d0 = (n / KW) * PW + g * (PW / 4) + (n % KW) * 8;
      if (a.vec_q) {
        const u4 x = load_u4(qsrc[i] + d0);
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[i][n][e] = x[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[i][n][e] = (uint32_t)qsrc[i][d0 + 2 * e] | ((uint32_t)qsrc[i][d0 + 2 * e + 1] << 16);
      }
    }

  // ---- a stage's codes and parameters ----
  // This wave's shares: K words of 16 tokens and a part; V words of 32 tokens, a part
  // and a run (head size 64: half of the operands of 32 tokens); wave 0 all K
  // parameters, wave 1 all V parameters.
  const int k_run = HD == 256 ? wave >> 1 : wave, k_part = HD == 256 ? wave & 1 : 0;
  const int v_grp = HD == 256 ? 0 : wave >> 1, v_part = HD == 256 ? wave >> 1 : 0, v_run = HD == 64 ? 0 : wave & 1;
  const uint8_t* head = a.cache + (int64_t)kvh * kv4_head_bytes(bs, HD);
  const const_i32 table = (const_i32)(uintptr_t)(a.tables + (int64_t)w.r * a.table_stride);
  const uint32_t k_lane = c * (HD / 2) + k_part * (PW / 2) + g * (PW / 8);
  const uint32_t v_lane = kv4_v_codes(bs, HD) + v_part * (PW * 2) + g * HD * 2 + c * (PW / 8) + v_run * 8;
  const uint32_t p_base = wave == 1 ? kv4_v_params(bs, HD) : kv4_k_params(bs, HD);
  const int last = begin < end ? begin + (end - 1 - begin) / ST * ST : begin;
  // the blocks of this wave's shares of a stage, and (waves 0 and 1) of a lane's token
  struct Blocks { int k, va, vb, p; } nb;
  const int p_tok = 16 * min(g, NS - 1) + c;
  auto blocks_of = [&](int t0) {
    auto at = [&](int t) { return min(t, w.kv - 1) >> a.dm.bs_log2; };
    Blocks x;
    x.k = table[at(t0 + 16 * k_run)];
    x.va = table[at(t0 + 32 * v_grp)];
    x.vb = table[at(t0 + 32 * v_grp + 16)];
    x.p = wave < 2 ? a.tables[(int64_t)w.r * a.table_stride + at(t0 + p_tok)] : 0;
    return x;
  };
  auto outside = [&](int b) { return (uint32_t)b >= (uint32_t)a.dm.num_blocks; };
  // a block outside the cache holds no token: block 0 is read in its place
  auto at_block = [&](int b) {
    return head + (uint64_t)(uint32_t)(outside(b) ? 0 : b) * (uint32_t)a.dm.block_stride;
  };
  u4 kc;              // KW words
  uint2 va, vb;       // four values of four tokens: of the first and the second 16
  uint32_t pw = 0;    // a token's parameters
  float p_none = 0.f; // -infinity where it lies in no block
  auto load = [&](int t0, const Blocks& x) {
    auto tok = [&](int t) { return (t0 + t) & (bs - 1); };
    const uint8_t* kb = at_block(x.k) + tok(16 * k_run) * (HD / 2);
    if constexpr (KW == 4) {
      kc = load_u4(kb + k_lane);
    } else {
      const uint2 y = *reinterpret_cast<const uint2*>(kb + k_lane);
      kc = u4{y.x, y.y, 0u, 0u};
    }
    va = *reinterpret_cast<const uint2*>(at_block(x.va) + tok(32 * v_grp) * (HD / 2) + v_lane);
    vb = *reinterpret_cast<const uint2*>(at_block(x.vb) + tok(32 * v_grp + 16) * (HD / 2) + v_lane);
    if (wave < 2) {
      // parameters 0 for tokens that do not exist, whatever lies there
      const bool out = outside(x.p);
      p_none = out ? -INFINITY : 0.f;
      pw = *reinterpret_cast<const uint32_t*>(at_block(x.p) + 4 * tok(p_tok) + p_base);
      pw = (out | (t0 + p_tok >= end)) ? 0u : pw;
    }
  };
  if (begin < end) {
    nb = blocks_of(begin);
    load(begin, nb);
    nb = blocks_of(min(begin + ST, last));
  }

  // ---- q as MFMA operands: each row times its own power of two, so that what
  // other rows hold (an infinity, values far larger) leaves it as it is ----
  __syncthreads();  // (of the stretch before, nothing is read any more)
  u4 qf[QT][ND];
  float qsum[QT], qmul[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    float top_q = 0.f;
#pragma unroll
    for (int n = 0; n < 4 * ND; ++n) {
      if (!real[i]) raw[i][n / 4][n % 4] = 0;
      const uint32_t x = raw[i][n / 4][n % 4];
      top_q = fmaxf(top_q, fmaxf(fabsf(T::to_f32(x & 0xFFFF)), fabsf(T::to_f32(x >> 16))));
    }
    top_q = over_rows(top_q, [](float p, float q) { return fmaxf(p, q); });
    int k2 = 0;
    if (top_q > 0.f) k2 = min(120, 140 - (int)((__float_as_uint(top_q) >> 23) & 255));
    const float up = ldexpf(1.f, k2);
    qmul[i] = ldexpf(1.f, 24 - k2);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = T::to_f32(raw[i][n][e] & 0xFFFF) * up;
        f[2 * e + 1] = T::to_f32(raw[i][n][e] >> 16) * up;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += f[e];
      // word & 0x000F000F: values 0, 4; & 0x00F000F0: 1, 5 (16 c); the same of word >> 8: 2, 6 and 3, 7
      qf[i][n] = u4{pack_h2(f[0], f[4]), pack_h2(f[1] * 0.0625f, f[5] * 0.0625f), pack_h2(f[2], f[6]),
                    pack_h2(f[3] * 0.0625f, f[7] * 0.0625f)};
    }
    qsum[i] = over_rows(sum, [](float p, float q) { return p + q; }) * 0x1p-24f;
  }

  // The loaded stage into LDS.
  auto unpack = [&](int buf) {
#pragma unroll
    for (int n = 0; n < KW; ++n) {
      const uint32_t x = kc[n], x8 = x >> 8;
      k_op[buf][k_run * ND + k_part * KW + n][lane] =
          u4{x & 0x000F000Fu, x & 0x00F000F0u, x8 & 0x000F000Fu, x8 & 0x00F000F0u};
    }
    u4* const to = &v_op[buf][v_grp * NV + (v_part * NH + v_run) * 4][lane];
    if (HD != 64 || (wave & 1) == 0) {
      to[0] = v_operand<0>(va.x, va.y, vb.x, vb.y);
      to[64] = v_operand<4>(va.x, va.y, vb.x, vb.y);
    }
    if (HD != 64 || (wave & 1) == 1) {
      to[128] = v_operand<0>(va.x >> 8, va.y >> 8, vb.x >> 8, vb.y >> 8);
      to[192] = v_operand<4>(va.x >> 8, va.y >> 8, vb.x >> 8, vb.y >> 8);
    }
    if (wave == 0 && lane < ST) {
      const float s = kv4_step(pw) * a.scale;
      par[buf][0][lane] = s;
      par[buf][1][lane] = fmaf(-7.5f, s, kv4_centre(pw) * a.scale);
      if (c == 0) gone[buf][g] = p_none;
    }
    if (wave == 1 && lane < ST) {
      par[buf][2][lane] = v_step_of(pw);
      par[buf][3][lane] = kv4_centre(pw);
    }
  };

  f4 o[QT][NP][NH][4];
  f4 wsum[QT];
  float l[QT], z[QT], m[QT], ref[QT];
  float sv_top[QT];  // 2^E, above every V step that the row has seen
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    l[i] = z[i] = 0.f;
    m[i] = ref[i] = kAttnNone;
    sv_top[i] = kAttnStep;
    wsum[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NP * NH * 4; ++x) o[i][x / (NH * 4)][x / 4 % NH][x % 4] = f4{0.f, 0.f, 0.f, 0.f};
  }

  // 32 tokens from t0 on, the stage's group j.
  auto step = [&](int t0, int buf, int j, auto mask) {
    constexpr bool masked = decltype(mask)::value;
    auto sees = [&](int i, int h, int e) {
      const int t = t0 + 16 * h + 4 * g + e;
      return (t <= pos[i]) & (t < end) & (t > pos[i] - window);  // no branches
    };
    // all reads of one product ahead of it: K's and the parameters first, V's behind
    // the first product, so that they come while the weights are computed
    u4 kf[2 * ND], vf[NV];
    f4 acc[QT][2], sk[2], mk[2], sv[2], mv[2];
    float none[2];
    float step_top = 0.f;
#pragma unroll
    for (int n = 0; n < 2 * ND; ++n) kf[n] = k_op[buf][2 * j * ND + n][lane];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = 32 * j + 16 * h + 4 * g;
      sk[h] = *reinterpret_cast<const f4*>(&par[buf][0][at]);
      mk[h] = *reinterpret_cast<const f4*>(&par[buf][1][at]);
      sv[h] = *reinterpret_cast<const f4*>(&par[buf][2][at]);
      none[h] = gone[buf][2 * j + h];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < QT; ++i) acc[i][h] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int i = 0; i < QT; ++i) acc[i][h] = mfma16x16x32<F16>(kf[h * ND + n], qf[i][n], acc[i][h]);
    }
#pragma unroll
    for (int x = 0; x < NV; ++x) vf[x] = v_op[buf][j * NV + x][lane];
#pragma unroll
    for (int h = 0; h < 2; ++h) mv[h] = *reinterpret_cast<const f4*>(&par[buf][3][32 * j + 16 * h + 4 * g]);
    __builtin_amdgcn_sched_barrier(0);
    // the exponents / qmul, in place of the sums
    float xm[QT], top[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      xm[i] = -INFINITY;
      top[i] = 0.f;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (!masked)
#pragma unroll
        for (int e = 0; e < 4; ++e) step_top = fmaxf(step_top, sv[h][e]);
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        float xh = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y = fmaf(sk[h][e], acc[i][h][e], mk[h][e] * qsum[i]);
          if constexpr (masked) {
            const bool ok = sees(i, h, e);
            y = ok ? y : -INFINITY;
            top[i] = fmaxf(top[i], ok ? sv[h][e] : 0.f);
          }
          acc[i][h][e] = y;
          xh = fmaxf(xh, y);
        }
        xm[i] = fmaxf(xm[i], xh + none[h]);
      }
    }
    if constexpr (!masked)
#pragma unroll
      for (int i = 0; i < QT; ++i) top[i] = step_top;
    bool grow = masked;
#pragma unroll
    for (int i = 0; i < QT; ++i) grow = grow | (top[i] > sv_top[i]) | (xm[i] * qmul[i] > m[i] + (float)kAttnHead);
    if (masked || __any(grow)) {
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        top[i] = over_rows(top[i], [](float p, float q) { return fmaxf(p, q); });
        const float x = over_rows(xm[i], [](float p, float q) { return fmaxf(p, q); }) * qmul[i];
        // a row moves for what it has seen itself, whatever the others saw
        const bool move = masked | (top[i] > sv_top[i]) | (x > m[i] + (float)kAttnHead);
        sv_top[i] = move ? fmaxf(sv_top[i], above_step(top[i])) : sv_top[i];
        m[i] = move ? fmaxf(m[i], x) : m[i];
        const float nr = move ? attn_ref(m[i], sv_top[i]) : ref[i];
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
    }
    u4 pf[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float pv[4];
        const float off = none[h] - ref[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(acc[i][h][e], qmul[i], off));
          pv[e] = p * sv[h][e];
          if constexpr (masked) {
            const bool ok = sees(i, h, e);
            l[i] += ok ? p : 0.f;
            z[i] = ok ? fmaf(p, mv[h][e], z[i]) : z[i];
            pv[e] = ok ? pv[e] : 0.f;
          } else {
            l[i] += p;
            z[i] = fmaf(p, mv[h][e], z[i]);
          }
        }
        pf[i][2 * h] = pack_h2(pv[0], pv[1]);
        pf[i][2 * h + 1] = pack_h2(pv[2], pv[3]);
      }
    const u4 halves = u4{0x38003800u, 0x38003800u, 0x38003800u, 0x38003800u};  // 0.5
#pragma unroll
    for (int i = 0; i < QT; ++i) wsum[i] = mfma16x16x32<F16>(halves, pf[i], wsum[i]);
#pragma unroll
    for (int x = 0; x < NV; ++x)
#pragma unroll
      for (int i = 0; i < QT; ++i)
        o[i][x / (NH * 4)][x / 4 % NH][x % 4] = mfma16x16x32<F16>(vf[x], pf[i], o[i][x / (NH * 4)][x / 4 % NH][x % 4]);
  };

  if (begin < end) {
    unpack(0);
    load(min(begin + ST, last), nb);
    nb = blocks_of(min(begin + 2 * ST, last));
    __syncthreads();
    // Each wave: stages before its first key, cut by the window, seen whole, cut by
    // the rows' positions, behind its last key -- the same number of barriers for all.
    int t0 = begin, buf = 0;
    const int from = a.window > 0 ? pmin - a.window + 1 : 0;                  // its first key
    const int full0 = a.window > 0 ? pmax - a.window + 1 : 0;                 // first key that all rows see
    const int full1 = min(pmin + 1, end), to = min(pmax + 1, end);            // behind the last such, behind the last
    auto stages = [&](int upto, auto what) {
      for (; t0 < upto; t0 += ST, buf ^= 1) {
        if (t0 + ST <= last) unpack(buf ^ 1);
        load(min(t0 + 2 * ST, last), nb);
        nb = blocks_of(min(t0 + 3 * ST, last));
        what();
        __syncthreads();
      }
    };
    auto idle = [&]() {};
    auto cut = [&]() {
#pragma unroll 1
      for (int j = 0; j < NG; ++j)
        if (t0 + 32 * j < to && t0 + 32 * j + 32 > from) step(t0 + 32 * j, buf, j, std::true_type{});
    };
    auto all = [&]() {
#pragma unroll
      for (int j = 0; j < NG; ++j) step(t0 + 32 * j, buf, j, std::false_type{});
    };
    auto down = [&](int t) { return begin + (t - begin) / ST * ST; };       // to a stage's begin, t >= begin
    const int e0 = down(max(min(from, end), begin)), e1 = max(full0 > begin ? down(full0 + ST - 1) : begin, e0);
    stages(min(e0, end), idle);
    stages(min(min(e1, to), end), cut);
    stages(down(max(full1, begin)), all);
    stages(to, cut);
    stages(end, idle);
  }

  // ---- the end: sums over the lanes of a row, rows out ----
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    l[i] = over_rows(l[i], [](float p, float q) { return p + q; });
    z[i] = over_rows(z[i], [](float p, float q) { return p + q; });
    const float off = z[i] + wsum[i][0];  // every row of the MFMA's result holds sum(P sv) / 2
    // lane (c, g): values p PW + g PW / 4 + 4 NH e + 4 h + b of row c
    auto value = [&](int p, int e, int h, int b) {
      return fmaf(o[i][p][h][b][e], b & 1 ? 0.0625f : 1.0f, off);
    };
    const int rr = row0 + i * 16 + c;
    if (rr >= w.rows) continue;
    if (!whole) {
      const int64_t pr = part0 + wave * QT * 16 + i * 16 + c;
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

void launch_attn_rows(const Kv4AttnArgs& a, int hd, int io_dtype, dim3 grid, hipStream_t st) {
#define CEK_GO(D)                                                                                              \
  do {                                                                                                         \
    if (io_dtype == CEK_F16) kv4_attn_rows_kernel<F16, D, D == 256 ? 1 : 2><<<grid, 256, 0, st>>>(a);          \
    else kv4_attn_rows_kernel<BF16, D, D == 256 ? 1 : 2><<<grid, 256, 0, st>>>(a);                             \
  } while (0)
  CEK_KV4_HD(CEK_GO);
#undef CEK_GO
}

}  // namespace cek
