// cek_kv4_attn.hip -- attention over the 4-bit paged key/value cache, gfx950
// (layout and number format: cek_kv4.h).
//
//   out_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i . k_j), j in row i's range
//
// with k = mk + sk (ck - 7.5), v = mv + sv (cv - 7.5) per token and head:
//
//   q . k       = sk (q . ck) + (mk - 7.5 sk) sum(q)
//   sum_j w v   = sum_j (w sv)(cv - 8) + sum_j (w sv) / 2 + sum_j w mv
//
// so the matrix products run on the codes themselves and the parameters are
// applied to scores and weights, one value a token instead of hd.  K's codes
// enter the fp16 MFMA as they lie: a 32-bit word & 0x000F000F is a pair of fp16
// subnormals c 2^-24, & 0x00F000F0 a pair c 2^-20 -- exact, one AND (and a shift
// for every second pair) where a conversion would take three operations.  The
// powers of two are taken back in q (2^-4 for the second kind) and in the scores --
// exactly, so that a row's largest score less its maximum is 0 at any size.
// V's take an OR and a packed subtraction more (v_pair).
//
// Layout: everything stays in registers.  A wave takes 32 tokens at a time and
// QT tiles of 16 rows (row = query token x query head of the kv head).  It forms
// S^T = K Q^T (MFMA rows: tokens, columns: rows), so that a lane holds eight
// weights of one row, which are -- without a shuffle, since the order within a
// contraction is free -- the operand of O^T = V^T P^T; V's words hold four tokens
// side by side for that.  Each tile of rows reads each code byte once, 1 KB a load
// instruction; the tiles of one request read them again, from HBM or the L2.
//
// Weights: with M a running maximum of a row's exponents and 2^E above every sv that
// the row has seen, P = exp2(x - M - E + 9) makes P sv at most 2^9 as it comes and
// 2^15 with the 2^6 that a maximum may lag behind (it moves, and the sums are
// rescaled, only where a score exceeds it by more): fp16 holds P sv to half a step
// (2^-12 of the value) down to 2^-23 of the largest, and to 2^-34 of that below.
// M, E and the power of two of q are the row's own and move for what it sees itself:
// no other row, and no token that it does not see, changes its bits.  Sums are fp32;
// sum(P sv) / 2 is taken by an MFMA over the rounded weights, so that a weight's
// rounding acts on v's distance from its centre alone.
//
// What bounds it: the codes' bytes from HBM, and for short keys the latency of one
// launch.  64 requests of 308 .. 16000 keys, 32 / 8 heads of 128, bf16: 57.8 us for
// 288 MB (5.0 TB/s; a kernel that only reads them 40); one of 131071 keys 33.1 us
// (143 MB; 20); 16 of 5 drafts on up to 6000 keys, window 4096, 16 heads of 256,
// fp16: 43.8 us (174 MB; 24); one of 700 keys 10.4 us, of which 5 in the six tiles
// that each wave takes one after another.  What lies between: launch, work list,
// table and first tiles before the loop, 5 us; the join's launch, 5; and workgroups
// that end up to 10 us before the last one.
#include <algorithm>
#include <type_traits>

#include "cek_kv4_attn.h"

namespace cek {

// Parameters of tokens that do not exist: K's and, 4 bs bytes on, V's.
__device__ const uint8_t kv4_zeros[4 * 256 + 64] __attribute__((aligned(16))) = {};

typedef uint32_t u2 __attribute__((ext_vector_type(2)));

__device__ inline __amdgpu_buffer_rsrc_t kv4_rsrc(const uint8_t* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000);
}
__device__ inline uint32_t lds_offset(const void* p) { return (uint32_t)(uintptr_t)(lds_ptr_t)p; }

// LDS reads behind a wave's own direct loads, in asm with their wait: the compiler
// would wait for every direct load in flight before any LDS read.  A lane's
// codes of 32 tokens (K or V: two loads of 16 tokens, HALF bytes apart) and the
// parameters of its tokens (one or two loads each).
template <int HD, int HALF>
__device__ inline void read_codes(uint32_t at, uint32_t (&to)[2][HD / 32]) {
  if constexpr (HD == 64) {
    u2 a, b;
    asm volatile("ds_read_b64 %0, %2\n\tds_read_b64 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(a), "=&v"(b)
                 : "v"(at), "n"(HALF)
                 : "memory");
    to[0][0] = a[0], to[0][1] = a[1], to[1][0] = b[0], to[1][1] = b[1];
  } else if constexpr (HD == 128) {
    u4 a, b;
    asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(a), "=&v"(b)
                 : "v"(at), "n"(HALF)
                 : "memory");
#pragma unroll
    for (int e = 0; e < 4; ++e) to[0][e] = a[e], to[1][e] = b[e];
  } else {
    u4 x[4];
    asm volatile(
        "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:1024\n\t"
        "ds_read_b128 %2, %4 offset:%5\n\tds_read_b128 %3, %4 offset:%6\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
        : "v"(at), "n"(HALF), "n"(HALF + 1024)
        : "memory");
#pragma unroll
    for (int e = 0; e < 16; ++e) to[e / 8][e % 8] = x[e / 4][e % 4];
  }
}
__device__ inline void read_params(uint32_t at, u4 (&k)[2], u4 (&v)[2]) {
  asm volatile(
      "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:64\n\t"
      "ds_read_b128 %2, %4 offset:128\n\tds_read_b128 %3, %4 offset:192\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(k[0]), "=&v"(k[1]), "=&v"(v[0]), "=&v"(v[1])
      : "v"(at)
      : "memory");
}
__device__ inline void read_params(uint32_t at, u4 (&k)[1], u4 (&v)[1]) {
  asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:128\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(k[0]), "=&v"(v[0])
               : "v"(at)
               : "memory");
}

// Workgroups that a CU holds at once (waves a SIMD): by registers and LDS.
constexpr int attn_held(int hd, int qt) { return hd == 256 ? 2 : (hd == 64 ? 5 - qt : 4 - qt); }

// Few rows a request: the workgroup's four waves share QT x 16 rows and take every
// fourth 32 tokens each.
// FOLD: tiles of 8 rows, in the MFMA's columns twice, so that columns 0 .. 7 have
// the scores of the first 16 tokens at hand and columns 8 .. 15 those of the second
// 16: half the arithmetic between the two products.
template <typename T, int HD, int QT, bool FOLD>
__global__ __launch_bounds__(256, attn_held(HD, QT)) void kv4_attn_kernel(Kv4AttnArgs a) {
  constexpr int ND = HD / 32;                    // 32-bit words per lane, part and 16 tokens
  constexpr int NP = HD >= 128 ? HD / 128 : 1;   // parts of a row: 128 values, or 64
  constexpr int NH = HD >= 128 ? 2 : 1;          // runs of four values per lane and part
  constexpr int PW = HD / NP;                    // values of a part
  constexpr int RT = FOLD ? 8 : 16;              // rows of a tile
  constexpr int NX = FOLD ? 1 : 2;               // groups of four tokens a lane has scores of
  constexpr int BR = QT * RT;
  constexpr int LSTR = HD + 4;                   // LDS row stride: rows 4 banks apart
  constexpr int CODES = HD >= 128 ? 4 * NP * 1024 : 2048;  // bytes of 32 tokens' codes
  constexpr int SLOT = CODES + 256;                        // and parameters
  constexpr int HALF = CODES / 2;                          // 16 tokens: K codes, V codes
  constexpr int DEPTH = 2;                 // slots a wave
  constexpr int LOADS = CODES / 1024 + 1;                  // load instructions of a slot
  constexpr int OUT_BYTES = kAttnWaves * 16 * (LSTR + 2) * 4;
  constexpr int RING_BYTES = kAttnWaves * DEPTH * SLOT;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[RING_BYTES > OUT_BYTES ? RING_BYTES : OUT_BYTES];
  float* const lds_o = reinterpret_cast<float*>(lds);
  float* const lds_ml = lds_o + kAttnWaves * 16 * LSTR;

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int wg = uniform((int)(blockIdx.x / (unsigned)a.dm.n_kv)), kvh = blockIdx.x - wg * a.dm.n_kv;
  const int bs = 1 << a.dm.bs_log2;
  Kv4List<BR, attn_held(HD, QT)> list{a};
  const auto mine = list.request(lane);
  int u = wg, u_end = u + 1;
  if (a.wgs > 0) {
    // (units of cost: 4, 5, 6, 8 on 64 ragged requests 56.2, 56.4, 55.3, 56.3 us; 2, 4, 5, 6
    // on 16 with drafts, heads of 256, 45.0, 43.0, 44.2, 45.3; leads matter by 1 us)
    list.share(mine, 32 * kAttnWaves, HD == 256 ? 4 : 6);
    list.deal(a.wgs, attn_held(HD, QT) == 2 ? 8 : (attn_held(HD, QT) == 3 ? 6 : 4));
    u = list.begin_of(wg);
    u_end = list.begin_of(wg + 1);
  }
  for (Kv4Work w; u < u_end && list.find(mine, u, u_end, w); u += w.span) {
  if (w.units == 0) continue;
  const int row0 = w.tile * BR;  // the first row in the request
  // Partial rows: of a tile's first stretch in 2 wg + 1, of the others in 2 wg.
  const bool whole = w.units == w.all;
  const int64_t part0 =
      a.part_row0 + ((int64_t)(2 * wg + (w.unit == 0)) * a.dm.n_kv + kvh) * BR;
  if (a.meta && kvh == 0 && w.unit == 0 && (int)threadIdx.x < BR) {
    // for the launch that joins the parts: the first one's row and their number
    const int rr = w.tile * BR + (int)threadIdx.x;
    const int parts = whole ? 1 : list.owner_of(w.first + w.all - 1) - wg + 1;
    if (rr < w.rows) a.meta[(int64_t)w.q0 * a.group + rr] = int4{(int)part0 + (int)threadIdx.x, parts, a.dm.n_kv * BR, BR};
  }

  // ---- rows and the range of keys ----
  int pos[QT];          // position of the row; padding rows see everything
  int pmin = INT32_MAX, pmax = -1;  // over this wave's rows
  const uint16_t* qsrc[QT];
  bool real[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int rr = row0 + i * RT + (FOLD ? c & 7 : c);
    real[i] = rr < w.rows;
    const int t = rr / a.group, h = kvh * a.group + rr % a.group;
    qsrc[i] = a.q + (int64_t)(w.q0 + (real[i] ? t : 0)) * a.q_stride + (int64_t)(real[i] ? h : 0) * HD;
    pos[i] = real[i] ? kv4_pos(w.kv, w.n_new, t) : INT32_MAX - 1;
    if (row0 + i * RT < w.rows) {
      // uniform: rows are in order of position
      pmin = uniform(min(pmin, kv4_pos(w.kv, w.n_new, (row0 + i * RT) / a.group)));
      pmax = uniform(max(pmax, kv4_pos(w.kv, w.n_new, (min(row0 + i * RT + RT, w.rows) - 1) / a.group)));
    }
  }
  const int window = a.window > 0 ? a.window : INT32_MAX;  // pos - window stays in range
  const int t_lo = a.window > 0 ? max(0, pmin - a.window + 1) & ~31 : 0;
  const int begin = uniform((list.len ? max(t_lo, w.lo + w.unit * list.len) : t_lo) + 32 * wave);
  const int end = uniform(
      list.len ? (int)min((int64_t)pmax + 1, (int64_t)w.lo + (int64_t)(w.unit + w.units) * list.len) : pmax + 1);
  constexpr int STEP = 32 * kAttnWaves;

  // ---- q: this lane's 16-bit values of its row of each tile, in the order of K's
  // words; on their way while the codes' addresses are found ----
  uint32_t raw[QT][ND][4];
#pragma unroll
  for (int i = 0; i < QT; ++i)
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      const int d0 = (n / (PW / 32)) * PW + g * (PW / 4) + (n % (PW / 32)) * 8;
      if (a.vec_q) {
        const u4 x = load_u4(qsrc[i] + d0);
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[i][n][e] = x[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[i][n][e] = (uint32_t)qsrc[i][d0 + 2 * e] | ((uint32_t)qsrc[i][d0 + 2 * e + 1] << 16);
      }
    }

  // ---- codes and parameters: through a ring of LDS slots ----
  // Each wave keeps the next DEPTH tiles' loads in flight without a register: a
  // lane reads back what it loaded itself (the codes), so that nothing but the
  // wave's own vmcnt orders the two.
  const int head_bytes = kv4_head_bytes(bs, HD);
  const uint8_t* head = a.cache + (int64_t)kvh * head_bytes;
  const const_i32 table = (const_i32)(uintptr_t)(a.tables + (int64_t)w.r * a.table_stride);
  struct Blocks { int b[2]; };
  auto blocks_of = [&](int t0) {
    return Blocks{{table[t0 >> a.dm.bs_log2], table[min(t0 + 16, w.kv - 1) >> a.dm.bs_log2]}};
  };
  uint8_t* const ring = lds + wave * (DEPTH * SLOT);
  // hd 64: K and V of 16 tokens in one load, 32 lanes each
  const uint32_t k_lane = HD >= 128 ? c * (HD / 2) + g * 16 : (lane & 31) * 16 + (lane >> 5) * kv4_v_codes(bs, HD);
  const uint32_t v_lane = kv4_v_codes(bs, HD) + g * HD * 2 + c * 16;
  // parameters, 16 lanes each: K's of the first and the second 16 tokens, V's
  const uint32_t p_lane = (g & 2 ? 4 * bs : 0) + 4 * c;
  // The 32 tokens at t0 into a slot; returns which halves lie in no block (bits 0
  // and 1; the second one may lie behind the last key).  No code is read there (the
  // buffer has no bytes) and the parameters are 0.
  auto fetch = [&](int t0, const Blocks& x, int slot) -> int {
    uint8_t* const to = ring + slot * SLOT;
    int outs = 0;
    const uint8_t* par[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool out = ((uint32_t)x.b[h] >= (uint32_t)a.dm.num_blocks) | (t0 + 16 * h >= w.kv);
      outs |= (int)out << h;
      const uint64_t at = (uint64_t)(uint32_t)(out ? 0 : x.b[h]) * (uint32_t)a.dm.block_stride;
      const auto src = kv4_rsrc(head + at, out ? 0 : head_bytes);
      const int tok = (t0 + 16 * h) & (bs - 1);
      // (aux 2: not kept in the caches, since a tile of rows reads each code once)
#define CEK_FETCH(lane_off, dst, bytes, off) \
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (lds_ptr_t)(dst), bytes, lane_off, off, 0, 2)
      // a part of 128 values and 16 tokens: 64 bytes of each K row, 256 of each four tokens of V
      CEK_FETCH(k_lane, to + h * HALF, 16, tok * (HD / 2));
      if constexpr (HD == 256) CEK_FETCH(k_lane, to + h * HALF + 1024, 16, tok * (HD / 2) + 64);
      if constexpr (HD >= 128) CEK_FETCH(v_lane, to + h * HALF + NP * 1024, 16, tok * (HD / 2));
      if constexpr (HD == 256) CEK_FETCH(v_lane, to + h * HALF + 3 * 1024, 16, tok * (HD / 2) + 256);
#undef CEK_FETCH
      par[h] = out ? kv4_zeros : head + at + kv4_k_params(bs, HD) + 4 * tok;
    }
    __builtin_amdgcn_global_load_lds((g & 1 ? par[1] : par[0]) + p_lane, (lds_ptr_t)(to + CODES), 4, 0, 0);
    return outs;
  };
  const int last = begin + (end - 1 - begin) / STEP * STEP;
  Blocks nb;                       // of the tile DEPTH ahead
  int outs = 0;                    // two bits a slot, the present tile's first: halves outside the cache
  if (begin < end) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      nb = blocks_of(min(begin + i * STEP, last));
      outs |= fetch(min(begin + i * STEP, last), nb, i) << (2 * i);
    }
    nb = blocks_of(min(begin + DEPTH * STEP, last));
  }

  // ---- q as MFMA operands ----
  u4 qf[QT][ND];
  float qsum[QT], qmul[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    float top = 0.f;
    if (!real[i])
#pragma unroll
      for (int n = 0; n < 4 * ND; ++n) raw[i][n / 4][n % 4] = 0;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        top = fmaxf(top, fmaxf(fabsf(T::to_f32(raw[i][n][e] & 0xFFFF)), fabsf(T::to_f32(raw[i][n][e] >> 16))));
    top = over_rows(top, [](float p, float q) { return fmaxf(p, q); });
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
        f[2 * e] = T::to_f32(raw[i][n][e] & 0xFFFF) * up;
        f[2 * e + 1] = T::to_f32(raw[i][n][e] >> 16) * up;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += f[e];
      // word & 0x000F000F: values 0, 4; & 0x00F000F0: 1, 5 (16 c); the same of word >> 8: 2, 6 and 3, 7
      qf[i][n] = u4{pack_h2(f[0], f[4]), pack_h2(f[1] * 0.0625f, f[5] * 0.0625f), pack_h2(f[2], f[6]),
                    pack_h2(f[3] * 0.0625f, f[7] * 0.0625f)};
    }
    sum = over_rows(sum, [](float p, float q) { return p + q; });
    qsum[i] = sum * 0x1p-24f;
    qmul[i] = ldexpf(1.f, 24 - k);
  }

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

  auto token = [&](int h, int e) { return 16 * (FOLD ? c >> 3 : h) + 4 * g + e; };
  auto sees = [&](int i, int t0, int h, int e) {  // this lane's row of tile i that token at t0
    const int t = t0 + token(h, e);
    return (t <= pos[i]) & (t < end) & (t > pos[i] - window);  // no branches
  };

  uint32_t kc[2][ND], vc[2][ND];  // the codes of 32 tokens, 16 and 16
  u4 kp[NX], vp[NX];              // the parameters of this lane's tokens, 4 g .. of 16
  float none[NX];                 // 0, or -infinity where those lie in no block
  int slot = 0;
  const uint32_t ring_at = lds_offset(ring);
  const uint32_t k_at = ring_at + (HD >= 128 ? lane * 16 : c * 32 + g * 8);
  const uint32_t v_at = ring_at + (HD >= 128 ? NP * 1024 + lane * 16 : 512 + lane * 8);
  const uint32_t p_at = ring_at + CODES + 16 * g + (FOLD ? (c >> 3) * 64 : 0);
  // The present tile from its slot: K codes and parameters once they are there,
  // V codes later, and then the slot to the tile DEPTH ahead.
  auto read_k = [&]() {
    wait_vmcnt<(DEPTH - 1) * LOADS>();
    const uint32_t at = slot * SLOT;
    if constexpr (FOLD) {
      none[0] = outs >> (c >> 3) & 1 ? -INFINITY : 0.f;
    } else {
      none[0] = outs & 1 ? -INFINITY : 0.f;
      none[1] = outs & 2 ? -INFINITY : 0.f;
    }
    read_params(p_at + at, kp, vp);
    read_codes<HD, HALF>(k_at + at, kc);
  };
  auto read_v = [&]() { read_codes<HD, HALF>(v_at + slot * SLOT, vc); };
  auto refill = [&](int t0) {
    const Blocks nx = nb;
    nb = blocks_of(min(t0 + (DEPTH + 1) * STEP, last));  // a tile ahead of the loads that need them
    outs = (outs >> 2) | (fetch(min(t0 + DEPTH * STEP, last), nx, slot) << (2 * (DEPTH - 1)));
    slot = slot + 1 == DEPTH ? 0 : slot + 1;
  };

  // Scores of 32 tokens: x (exponents / qmul), their maxima xm and those of the V steps.
  float x[QT][NX][4], xm[QT], top[QT];
  auto scores = [&](int t0, auto mask) {
    constexpr bool masked = decltype(mask)::value;
    if constexpr (masked) {
#pragma unroll
      for (int h = 0; h < NX; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool out = t0 + token(h, e) >= end;  // no token: whatever lies there
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
    float step_top = 0.f;  // of the lane's tokens, where all rows see them
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      xm[i] = -INFINITY;
      top[i] = 0.f;
    }
    if constexpr (FOLD) {
#pragma unroll
      for (int i = 0; i < QT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][0][e] = c < 8 ? acc[i][0][e] : acc[i][1][e];
    }
#pragma unroll
    for (int h = 0; h < NX; ++h) {
      float xh[QT];
#pragma unroll
      for (int i = 0; i < QT; ++i) xh[i] = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float sk = kv4_step(kp[h][e]) * a.scale, mk = fmaf(-7.5f, sk, kv4_centre(kp[h][e]) * a.scale);
        if constexpr (!masked) step_top = fmaxf(step_top, v_step_of(vp[h][e]));
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          x[i][h][e] = fmaf(sk, acc[i][h][e], mk * qsum[i]);
          if constexpr (masked) {
            const bool ok = sees(i, t0, h, e);
            x[i][h][e] = ok ? x[i][h][e] : -INFINITY;
            top[i] = fmaxf(top[i], ok ? v_step_of(vp[h][e]) : 0.f);
          }
          xh[i] = fmaxf(xh[i], x[i][h][e]);
        }
      }
#pragma unroll
      for (int i = 0; i < QT; ++i) xm[i] = fmaxf(xm[i], xh[i] + none[h]);
    }
    if constexpr (!masked)
#pragma unroll
      for (int i = 0; i < QT; ++i) top[i] = step_top;
  };
  auto grows = [&]() {
    bool y = false;
#pragma unroll
    for (int i = 0; i < QT; ++i) y = y | (top[i] > sv_top[i]) | (xm[i] * qmul[i] > m[i] + (float)kAttnHead);
    return __any(y);
  };
  // Over the lanes that hold one row.
  auto over_row = [&](float v, auto op) {
    if constexpr (FOLD) v = op(v, CEK_DPP_F32(v, 0x128));  // row_ror 8
    return over_rows(v, op);
  };
  // New references, and the sums so far brought to them.
  auto rescale = [&](auto mask) {
    constexpr bool masked = decltype(mask)::value;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      const float t = over_row(xm[i], [](float p, float q) { return fmaxf(p, q); }) * qmul[i];
      // a row moves for what it has seen itself, whatever the others saw
      top[i] = over_row(top[i], [](float p, float q) { return fmaxf(p, q); });
      const bool move = masked | (top[i] > sv_top[i]) | (t > m[i] + (float)kAttnHead);
      sv_top[i] = move ? fmaxf(sv_top[i], above_step(top[i])) : sv_top[i];
      m[i] = move ? fmaxf(m[i], t) : m[i];
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
  };
  // Weights and the sums over them.
  auto accumulate = [&](int t0, auto mask) {
    constexpr bool masked = decltype(mask)::value;
    u4 pf[QT];  // the weights times sv, fp16: tokens 4 g .. of both halves
#pragma unroll
    for (int h = 0; h < NX; ++h) {
      float pv[QT][4], off[QT];
#pragma unroll
      for (int i = 0; i < QT; ++i) off[i] = none[h] - ref[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float sv = v_step_of(vp[h][e]), mv = kv4_centre(vp[h][e]);
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
    if constexpr (FOLD) {
      // the other half's weights, of columns 0 .. 7 (8 .. 15 hold nothing that is used)
#pragma unroll
      for (int i = 0; i < QT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) pf[i][2 + e] = __builtin_amdgcn_mov_dpp(pf[i][e], 0x128, 0xF, 0xF, true);  // row_ror 8
    }
    read_v();
    refill(t0);
    // O^T: values 4 (NH c + h) + b of each part, in rows c
    const u4 halves = u4{0x38003800u, 0x38003800u, 0x38003800u, 0x38003800u};  // 0.5
#pragma unroll
    for (int i = 0; i < QT; ++i) wsum[i] = mfma16x16x32<F16>(halves, pf[i], wsum[i]);
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int n = (p * NH + h) * 2;
        const uint32_t a0 = vc[0][n], a1 = vc[0][n + 1], b0 = vc[1][n], b1 = vc[1][n + 1];
        const u4 f[4] = {v_operand<0>(a0, a1, b0, b1), v_operand<4>(a0, a1, b0, b1),
                         v_operand<0>(a0 >> 8, a1 >> 8, b0 >> 8, b1 >> 8),
                         v_operand<4>(a0 >> 8, a1 >> 8, b0 >> 8, b1 >> 8)};
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int i = 0; i < QT; ++i) o[i][p][h][b] = mfma16x16x32<F16>(f[b], pf[i], o[i][p][h][b]);
      }
  };

  // Tiles in order: those that the window cuts, those that every row sees whole (up
  // to `full`), those that the rows' own positions or the end cut.  The cut ones
  // mask, and rescale without asking.
  if (begin < end) {
    const int full = uniform(min(pmin - 31, end - 32));
    int t0 = begin;
    auto cut_to = [&](int to) {
      for (; t0 < to; t0 += STEP) {
        read_k();
        scores(t0, std::true_type{});
        rescale(std::true_type{});
        accumulate(t0, std::true_type{});
      }
    };
    if (a.window > 0) cut_to(min(end, pmax - a.window + 1));
    for (; t0 <= full; t0 += STEP) {
      read_k();
      scores(t0, std::false_type{});
      if (grows()) rescale(std::false_type{});
      accumulate(t0, std::false_type{});
    }
    cut_to(end);
    wait_vmcnt<0>();  // loads in flight land in LDS that is about to be used, or given back
  }
  __syncthreads();

  // ---- the end: sums over the lanes of a row, parts to the workspace, rows out ----
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    l[i] = over_row(l[i], [](float p, float q) { return p + q; });
    z[i] = over_row(z[i], [](float p, float q) { return p + q; });
    const float off = z[i] + wsum[i][0];  // every row of the MFMA's result holds sum(P sv) / 2
    // lane (c, g): values p PW + g PW / 4 + 4 NH e + 4 h + b of row c
    auto value = [&](int p, int e, int h, int b) {
      return fmaf(o[i][p][h][b][e], b & 1 ? 0.0625f : 1.0f, off);
    };
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
    const int rr = w.tile * BR + i * RT + row;
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
    if (row < RT && rr < w.rows) {
      if (!whole) {
        const int64_t pr = part0 + i * RT + row;
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
  }
  __syncthreads();  // the rows have been read: LDS is free for the next stretch's codes
  }
}

// Largest of the 64 lanes, uniform, by DPP (wave_sum_dpp's pattern).
__device__ inline float wave_max_dpp(float v) {
  v = fmaxf(v, CEK_DPP_F32(v, 0xB1));
  v = fmaxf(v, CEK_DPP_F32(v, 0x4E));
  v = fmaxf(v, CEK_DPP_F32(v, 0x141));
  v = fmaxf(v, CEK_DPP_F32(v, 0x140));
  return over_rows(v, [](float p, float q) { return fmaxf(p, q); });
}

// The parts of a row that several workgroups share.  Part 0 is its first
// workgroup's, part p that of the p-th after it, two row tiles on each.
struct Kv4Parts {
  int64_t t, row0;
  int h, n, step;
  // Row t, head h of the call; n is 0 where there is nothing to join.
  __device__ inline Kv4Parts(const Kv4AttnArgs& a, int64_t item, int n_q) {
    t = item / n_q;
    h = (int)(item - t * n_q);
    n = 0;
    if (t >= a.T) return;
    const int kvh = h / a.group;
    const int c0 = a.cu_q[0], c1 = a.cu_q[a.R];
    const int4 mt = a.meta[t * a.group + h - kvh * a.group];
    row0 = mt.x + (int64_t)kvh * mt.w;
    step = mt.z;
    n = mt.y;
    // (rows that offsets out of order left without a worker: whatever the workspace
    // held -- no more parts than workgroups share a tile, each in a row of its own)
    const bool no = (t < c0) | (t >= c1) | (mt.y <= 1) | (mt.y > a.max_parts) | (mt.x < 0) | (mt.z <= 0) | (mt.w < 0);
    if (no || row(n - 1) >= a.part_rows) n = 0;
  }
  __device__ inline int64_t row(int p) const { return row0 + (int64_t)step * (p > 0 ? 2 * p - 1 : 0); }
};

// Joins them: HD / 4 lanes a row, eight parts at a time on their way.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv4_attn_join_kernel(Kv4AttnArgs a, int n_q) {
  constexpr int L = HD / 4, AHEAD = 8;
  const Kv4Parts parts(a, (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L, n_q);
  if (parts.n == 0) return;
  const int d0 = (threadIdx.x % L) * 4;
  float top = kAttnNone, den = 0.f;
  f4 y = f4{0.f, 0.f, 0.f, 0.f};
  for (int base = 0; base < parts.n; base += AHEAD) {
    f4 v[AHEAD];
    float2 ml[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int64_t row = parts.row(min(base + i, parts.n - 1));
      ml[i] = *reinterpret_cast<const float2*>(a.part_ml + 2 * row);
      v[i] = *reinterpret_cast<const f4*>(a.part + row * HD + d0);
    }
    float nt = top;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) nt = fmaxf(nt, ml[i].x);
    const float keep = __builtin_amdgcn_exp2f(top - nt);
    top = nt;
    den *= keep;
    y *= keep;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      // (a part of weight 0 counts too: what it holds may be NaN)
      const bool in = base + i < parts.n;
      const float f = __builtin_amdgcn_exp2f(ml[i].x - nt);
      den = in ? fmaf(f, ml[i].y, den) : den;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = in ? fmaf(v[i][e], f, y[e]) : y[e];
    }
  }
  const float inv = den != 0.f ? 1.0f / den : 0.f;
  uint16_t u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = T::from_f32(den != 0.f ? y[e] * inv : 0.f);
  uint16_t* const dst = a.out + parts.t * a.out_stride + (int64_t)parts.h * HD + d0;
  if (a.vec_out) {
    *reinterpret_cast<uint2*>(dst) =
        uint2{(uint32_t)u[0] | ((uint32_t)u[1] << 16), (uint32_t)u[2] | ((uint32_t)u[3] << 16)};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) dst[e] = u[e];
  }
}

// Few rows of many parts: a workgroup for 32 values of a row, eight groups of
// threads taking every eighth part.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv4_attn_join_wide_kernel(Kv4AttnArgs a, int n_q) {
  constexpr int G = 8, AHEAD = 8;  // groups; parts of a group that are loaded at once
  const int tid = threadIdx.x, lane = tid & 63, grp = tid >> 5;
  const Kv4Parts parts(a, blockIdx.x, n_q);
  if (parts.n == 0) return;
  const int d0 = (int)blockIdx.y * 32 + (tid & 31);
  float top = kAttnNone, den = 0.f, y = 0.f;
  for (int base = 0; base < parts.n; base += 64) {
    // a lane for a part: references and sums; then the parts' rows by their weights
    const bool in = base + lane < parts.n;
    const int64_t mine = parts.row(in ? base + lane : 0);
    const float r = in ? a.part_ml[2 * mine] : kAttnNone, l = in ? a.part_ml[2 * mine + 1] : 0.f;
    const int n = min(64, parts.n - base);
    float v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) v[i] = a.part[parts.row(base + min(grp + G * i, n - 1)) * HD + d0];
    const float nt = fmaxf(top, wave_max_dpp(r)), keep = __builtin_amdgcn_exp2f(top - nt);
    const float f = __builtin_amdgcn_exp2f(r - nt);
    top = nt;
    den = fmaf(den, keep, wave_sum_dpp(f * l));
    y *= keep;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int p = grp + G * i;
      const float w = __shfl(f, p, 64);
      y = p < n ? fmaf(v[i], w, y) : y;
    }
  }
  __shared__ float so[G][32];
  so[grp][tid & 31] = y;
  __syncthreads();
  if (tid < 32) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) v += so[i][tid];
    a.out[parts.t * a.out_stride + (int64_t)parts.h * HD + d0] = T::from_f32(den != 0.f ? v / den : 0.f);
  }
}

}  // namespace cek

using namespace cek;

namespace {

// What the host knows of a call: which kernels, their tiles, and whether the keys
// are shared.  Requests with more than kAttnFewRows rows (query tokens x heads of a
// kv head) go to the kernel whose waves have rows of their own.  16 requests of 4000
// keys, bf16, us at 16 / 32 / 64 / 128 rows in this kernel and in that one: 8 kv heads
// of 128, 29 / 36 / 53 / 90 and 62 / 64 / 69 / 80; 4 of 64, 20 / 24 / 30 / 42 and 31 /
// 33 / 35 / 42; 4 of 256, 30 / 42 / 67 / 108 and 46 / 49 / 58 / 87.
constexpr int kAttnFewRows = 64;
constexpr int kAttnCus = 256;

struct AttnPlan {
  bool few, many;
  bool fold;                      // tiles of 8 rows in the kernel for few rows
  int qt_few;
  int64_t tiles_few, tiles_many;  // bounds of the row tiles per kv head
  int wgs_few, wgs_many;          // workgroups per kv head that share the keys; 0: one for each tile
  int64_t part_rows_few, part_rows;
  int64_t bytes;
};

AttnPlan attn_plan(int64_t T, int64_t R, int64_t n_q, int64_t n_kv, int64_t hd, int64_t max_q_len, int64_t max_kv_len) {
  AttnPlan p{};
  const int64_t group = n_q / n_kv;
  if (max_q_len <= 0 || max_q_len > T) max_q_len = T;
  const int64_t rows = max_q_len * group;
  p.many = rows > kAttnFewRows;
  // (all requests of one length: none for it)
  p.few = !p.many || T < R * max_q_len;
  const int64_t few_rows = p.many ? group : rows;  // of a request, as a rule
  p.fold = few_rows <= 8;
  p.qt_few = few_rows <= 16 || hd == 256 ? 1 : 2;
  const int64_t br_few = p.fold ? 8 : 16 * p.qt_few;
  const int64_t seqs = std::min(R, T);
  p.tiles_few = T * group / br_few + seqs;
  if (p.many) p.tiles_few = std::min(p.tiles_few, seqs * (kAttnFewRows / br_few));
  p.tiles_many = T * group / attn_rows_br((int)hd) + seqs;
  // As many workgroups as the CUs hold at once, each with an equal share of all
  // keys.  Not for short keys, where joining the parts would take longer than
  // they, nor for more row tiles than workgroups of the kernel for many rows.
  const bool long_keys = max_kv_len <= 0 || max_kv_len > 1024;
  if (p.few && long_keys) p.wgs_few = (int)std::max<int64_t>(1, kAttnCus * attn_held((int)hd, p.qt_few) / n_kv);
  if (p.many && long_keys && p.tiles_many * n_kv < 2 * kAttnCus)
    p.wgs_many = (int)std::max<int64_t>(1, 2 * kAttnCus / n_kv);
  p.part_rows_few = (int64_t)2 * p.wgs_few * n_kv * br_few;
  p.part_rows = p.part_rows_few + (int64_t)2 * p.wgs_many * n_kv * attn_rows_br((int)hd);
  if (p.part_rows > 0) p.bytes = p.part_rows * (hd + 2) * 4 + T * group * 16;
  return p;
}

template <typename T, int HD>
void launch_attn(const AttnPlan& p, Kv4AttnArgs a, int64_t n_kv, int64_t n_q, hipStream_t st) {
  if (p.few) {
    Kv4AttnArgs b = a;
    b.rows_above = 0;
    b.rows_upto = p.many ? kAttnFewRows : INT32_MAX;
    b.wgs = p.wgs_few;
    b.part_row0 = 0;
    const dim3 grid((unsigned)((p.wgs_few ? p.wgs_few : p.tiles_few) * n_kv));
    if (p.fold) kv4_attn_kernel<T, HD, 1, true><<<grid, 256, 0, st>>>(b);
    else if (p.qt_few == 1) kv4_attn_kernel<T, HD, 1, false><<<grid, 256, 0, st>>>(b);
    else if constexpr (HD != 256) kv4_attn_kernel<T, HD, 2, false><<<grid, 256, 0, st>>>(b);
  }
  if (p.many) {
    Kv4AttnArgs b = a;
    b.rows_above = p.few ? kAttnFewRows : 0;
    b.rows_upto = INT32_MAX;
    b.wgs = p.wgs_many;
    b.part_row0 = (int)p.part_rows_few;
    const dim3 grid((unsigned)((p.wgs_many ? p.wgs_many : p.tiles_many) * n_kv));
    launch_attn_rows(b, HD, T::code, grid, st);
  }
  if (p.part_rows > 0) {
    const int64_t rows = a.T * n_q;
    if (rows <= 512) kv4_attn_join_wide_kernel<T, HD><<<dim3((unsigned)rows, HD / 32), 256, 0, st>>>(a, (int)n_q);
    else kv4_attn_join_kernel<T, HD><<<(unsigned)((rows * (HD / 4) + 255) / 256), 256, 0, st>>>(a, (int)n_q);
  }
}

}  // namespace

extern "C" int64_t cek_kv4_attention_workspace_size(int64_t T, int64_t R, int64_t n_q, int64_t n_kv, int64_t hd,
                                                    int64_t max_q_len, int64_t max_kv_len) {
  if (T <= 0 || R <= 0 || n_kv <= 0 || n_q <= 0 || n_q % n_kv || (hd != 64 && hd != 128 && hd != 256)) return 0;
  // sizes that the call refuses
  if (T > INT32_MAX || n_q > 65535 || n_kv > 4096 || max_q_len < 0 || max_kv_len < 0 ||
      T * (n_q / n_kv) > INT32_MAX / 4 || R > 1 << 26)
    return 0;
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
  // rows of a kv head, and requests: their tiles with what each costs stay below 2^30
  if (T * (n_q / n_kv) > INT32_MAX / 4 || R > 1 << 26) return CEK_ERR_UNSUPPORTED;
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
  a.scale = scale * 1.4426950408889634f;  // weights are powers of two
  a.vec_q = aligned(q, 16) && q_stride % 8 == 0;
  a.vec_out = aligned(out, 8) && out_stride % 4 == 0;
  AttnPlan p = attn_plan(T, R, n_q, n_kv, hd, max_q_len, max_kv_len);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) {
    p.wgs_few = p.wgs_many = 0;  // whole keys
    p.part_rows = 0;
  } else if (p.bytes > 0) {
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + p.part_rows * hd;
    a.meta = reinterpret_cast<int4*>(a.part_ml + p.part_rows * 2);
    a.part_rows = (int)std::min<int64_t>(p.part_rows, INT32_MAX);
    a.max_parts = std::max(p.wgs_few, p.wgs_many);
  }
  if (p.tiles_few * n_kv > INT32_MAX || p.tiles_many * n_kv > INT32_MAX || p.part_rows > INT32_MAX || T * n_q > INT32_MAX)
    return CEK_ERR_UNSUPPORTED;
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
