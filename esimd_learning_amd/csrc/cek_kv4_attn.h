// cek_kv4_attn.h -- what the attention kernels over the 4-bit cache share: their
// arguments, the work list and the arithmetic's constants (cek_kv4_attn.hip says
// what they mean).
#pragma once

#include "cek_kv4.h"

namespace cek {

struct Kv4AttnArgs {
  const uint16_t* q;
  uint16_t* out;
  const uint8_t* cache;
  const int32_t *tables, *kv_lens, *cu_q;
  float* part;     // split keys: rows of hd sums
  float* part_ml;  // and their (reference exponent, sum of weights)
  int4* meta;      // per row of a kv head: first part's row, parts, rows a slot, rows a tile
  int64_t T, q_stride, out_stride, table_stride;
  Kv4Dims dm;
  int R, group, max_blocks, window;
  int rows_above, rows_upto;  // this launch serves requests with that many rows
  int wgs;                    // workgroups per kv head that share the keys; 0: keys stay whole
  int part_row0;              // first partial row of this launch
  int part_rows;              // of all
  int max_parts;              // of a row
  int vec_q, vec_out;
  float scale;
};

constexpr int kAttnWaves = 4;
constexpr int kAttnHead = 6, kAttnBase = 9;  // exponents: lag of a maximum, where the largest weight lies
constexpr float kAttnNone = -3e38f;

typedef const __attribute__((address_space(4))) int32_t* const_i32;  // scalar loads

// A stretch of work: units [unit, unit + units) of the keys of one tile of rows.
struct Kv4Work {
  int r, q0, rows, kv, n_new, lo, tile;
  int unit, units, all;  // all: the tile's units
  int first, span;       // the tile's first unit in the list; how far the stretch reaches there
};

// The position of a request's new row t.  Rows before position 0 see no key: -1, from
// which a window of up to 2^31 - 1 can be taken without an overflow.
__device__ inline int kv4_pos(int kv, int n_new, int t) { return max(kv - n_new + t, -1); }

// The work list: every request has ceil(rows / BR) tiles of rows, and each tile its
// keys (from the first that any row sees, down to a multiple of 32) in units of
// `len` tokens, or in one.  Tiles lie one after another, a request's last one
// first (its rows see most keys).  Every wave of the grid computes its place
// from the lengths alone.
//
// Shared keys are dealt so that the workgroups end together, which equal shares do
// not do (64 requests of 308 .. 16000 keys ended between 29 and 59 us):
//   - a stretch costs its rows, its first loads and its sums' way out, as much as
//     `cost` units: in the list every tile has that many more, without keys, ahead
//     (62 -> 55 us);
//   - of the HELD workgroups that a CU holds the first is served first.  The grid's
//     first 256 workgroups are the first ones of their CUs, the next 256 the second
//     ones: each such layer gets less than the one before it, by `lead` 32nds.
template <int BR, int HELD>
struct Kv4List {
  const Kv4AttnArgs& a;
  int len = 0;    // tokens of a unit; 0: all of a tile's
  int cost = 0;   // units that a stretch costs
  int total = 0;  // units and costs, where the keys are shared

  struct Req { int q0, rows, kv, n_new, lo, tiles; };
  __device__ inline Req request(int r) const {
    Req x;
    const int at = min(r, a.R - 1);
    const int c0 = a.cu_q[at], c1 = a.cu_q[at + 1], kv = a.kv_lens[at];
    x.q0 = max(0, c0);
    x.n_new = (int)min((int64_t)c1, a.T) - x.q0;
    const int64_t n = (int64_t)x.n_new * a.group;
    const bool mine = (r < a.R) & (x.n_new > 0) & (n > a.rows_above) & (n <= a.rows_upto);
    x.rows = mine ? (int)n : 0;
    x.kv = (int)min((int64_t)max(kv, 0), (int64_t)a.max_blocks << a.dm.bs_log2);
    x.lo = a.window > 0 ? max(0, kv4_pos(x.kv, x.n_new, 0) - a.window + 1) & ~31 : 0;
    x.tiles = (x.rows + BR - 1) / BR;
    return x;
  }
  __device__ inline int units(const Req& x) const {
    return len ? (int)(((unsigned)max(x.kv - x.lo, 1) + (unsigned)len - 1u) / (unsigned)len) : 1;
  }
  // Tokens of a unit, from `least` to `most`, that give n workgroups four units each.
  __device__ inline int unit_for(const Req& first, int n, int least, int most) const {
    const int lane = threadIdx.x & 63;
    float keys = (float)first.tiles * (float)(first.kv - first.lo);
    for (int base = 64; base < a.R; base += 64) {
      const Req x = request(base + lane);
      keys += (float)x.tiles * (float)(x.kv - x.lo);
    }
    keys = wave_sum_dpp(keys);
    int step = least;
    while (step < most && keys > 4.f * (float)n * (float)step) step *= 2;
    return uniform(step);
  }
  // Units of `step` tokens, or as many times that as keep their number in 30 bits
  // (offsets that do not ascend may count rows so often that none does: no work then).
  __device__ inline void share(const Req& first, int step, int cost_) {
    const int lane = threadIdx.x & 63;
    cost = cost_;
    for (len = step;; len *= 2) {
      float sum = (float)first.tiles * (float)(units(first) + cost);
      int n = first.tiles * (units(first) + cost);
      for (int base = 64; base < a.R; base += 64) {
        const Req x = request(base + lane);
        sum += (float)x.tiles * (float)(units(x) + cost);
        n += x.tiles * (units(x) + cost);
      }
      total = __builtin_amdgcn_readlane(wave_scan_incl(n), 63);
      if (wave_sum_dpp(sum) < 0x1p30f) return;
      if (len >= 1 << 29) {
        total = 0;
        return;
      }
    }
  }
  // Of n workgroups each layer has `size`, the last one the rest; layer l's units
  // begin at base[l], its first more[l] workgroups have each[l] + 1, the others each[l].
  // (Below four units a workgroup one layer has all: no workgroup without units lies
  // between two with some, so that a tile's parts are those of consecutive ones.)
  int size = 0, base[HELD], each[HELD], more[HELD];
  __device__ inline void deal(int n, int lead) {
    constexpr unsigned S = 32 * HELD;
    const int lane = threadIdx.x & 63;
    size = total / 4 < n ? 0 : n / HELD;
    // a lane for a layer: one division for all of them
    const unsigned whole = (unsigned)total / S, rest = (unsigned)total % S;
    auto begin = [&](int l) {  // 32nds of an even share, of the layers before l
      const unsigned upto = l * (32 + lead * (HELD - l));
      return l < HELD ? (size ? (int)(whole * upto + rest * upto / S) : 0) : total;
    };
    const int l = min(lane, HELD - 1), from = begin(l), units = begin(l + 1) - from;
    const int workers = l + 1 < HELD ? size : n - (HELD - 1) * size;
    const int quot = (int)((unsigned)units / (unsigned)max(workers, 1)), over = units - quot * workers;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      base[i] = __builtin_amdgcn_readlane(from, i);
      each[i] = __builtin_amdgcn_readlane(quot, i);
      more[i] = __builtin_amdgcn_readlane(over, i);
    }
  }
  __device__ inline int begin_of(int j) const {
    int u = 0;
#pragma unroll
    for (int l = 0; l < HELD; ++l) {
      const int i = j - l * size;
      u = l == 0 || i >= 0 ? base[l] + each[l] * i + min(i, more[l]) : u;
    }
    return u;
  }
  __device__ inline int owner_of(int u) const {
    int at = 0, b = base[0], e = each[0], m = more[0];
#pragma unroll
    for (int l = 1; l < HELD; ++l) {
      const bool in = u >= base[l];
      at = in ? l * size : at;
      b = in ? base[l] : b;
      e = in ? each[l] : e;
      m = in ? more[l] : m;
    }
    const int i = u - b, far = m * (e + 1);
    return uniform(at + (i < far ? (int)((unsigned)i / (unsigned)(e + 1)) : m + (int)((unsigned)(i - far) / (unsigned)max(e, 1))));
  }
  // The stretch that starts at unit u, up to unit `to` (without units where it has
  // no more than costs); false behind the last one.
  __device__ inline bool find(const Req& first, int u, int to, Kv4Work& w) const {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.R; base += 64) {
      const Req x = base == 0 ? first : request(base + lane);
      const int n = units(x) + cost;
      const int incl = before + wave_scan_incl(x.tiles * n);
      const uint64_t above = __ballot(incl > u);
      if (above) {
        const int at = __builtin_ctzll(above);
        auto get = [&](int y) { return __builtin_amdgcn_readlane(y, at); };
        w.r = base + at;
        w.q0 = get(x.q0);
        w.rows = get(x.rows);
        w.kv = get(x.kv);
        w.n_new = get(x.n_new);
        w.lo = get(x.lo);
        const int all = get(n), tiles = get(x.tiles), start = get(incl) - tiles * all;
        const int nth = uniform((u - start) / all);
        w.tile = tiles - 1 - nth;
        w.all = all - cost;
        w.first = start + nth * all + cost;
        w.span = min(w.first + w.all, to) - u;
        w.unit = max(u - w.first, 0);
        w.units = max(u + w.span - w.first, 0) - w.unit;
        return true;
      }
      before = __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
  }
};

// v of lanes l, l ^ 16, l ^ 32, l ^ 48, joined by op.
template <typename OP>
__device__ inline float over_rows(float v, OP op) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// V's step as the products take it: of a row that is one value throughout (step 0)
// 2^-40 of that value, which changes nothing that fp32 holds and keeps the weights,
// up to 2^15 over the largest step, times the value in fp32's range.
__device__ inline float v_step_of(uint32_t p) { return fmaxf(kv4_step(p), fabsf(kv4_centre(p)) * 0x1p-40f); }

// The least power of two above a step; kAttnStep at least.
constexpr float kAttnStep = 0x1p-80f;
__device__ inline float above_step(float s) {
  return fmaxf(kAttnStep, __uint_as_float((__float_as_uint(s) & 0x7F800000u) + 0x00800000u));
}
// A row's reference, from its maximum m and 2^E.  From 2^22 on fp32 has no room for E
// beside m: the reference is m alone, and the largest weight 1.
__device__ inline float attn_ref(float m, float power) {
  const int e = (int)(__float_as_uint(power) >> 23) - 127;
  return fabsf(m) < 0x1p22f ? m + (float)(e - kAttnBase) : m;
}

__device__ inline uint32_t pack_h2(float a, float b) {
  return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});
}

// V's operand of four words: the nibbles at bits SHIFT (0: values c - 8; 4: 16 (c - 8))
// of each half, put into the mantissa of 1024 and taken back to zero.  Signed, so that
// sums over many keys stay as small as what they stand for: the MFMA aligns what it
// adds to the largest addend, and sums of codes 0 .. 15 lost 2^-17 of themselves over
// 640 keys a wave (a request of 123258 keys: outputs off by 0.0009 of their norm, now
// 0.0003).
template <int SHIFT>
__device__ inline uint32_t v_pair(uint32_t w) {
  const uint32_t x = (w & (0x000F000Fu << SHIFT)) | 0x64006400u;
  const _Float16 zero = (_Float16)(-1024 - (8 << SHIFT));
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, x) + h2{zero, zero});
}
template <int SHIFT>
__device__ inline u4 v_operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return u4{v_pair<SHIFT>(a), v_pair<SHIFT>(b), v_pair<SHIFT>(c), v_pair<SHIFT>(d)};
}

// The kernel for many rows (cek_kv4_attn_rows.hip): tiles of attn_rows_br(hd) rows.
constexpr int attn_rows_br(int hd) { return hd == 256 ? 64 : 128; }
void launch_attn_rows(const Kv4AttnArgs& a, int hd, int io_dtype, dim3 grid, hipStream_t st);

}  // namespace cek
