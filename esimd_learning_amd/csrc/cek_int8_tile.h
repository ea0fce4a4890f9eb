// cek_int8_tile.h -- the tiled int8 product (and gated block), gfx950.
//
// A workgroup of eight waves computes BM x BN sums in 16 x 16 x 64 matrix instructions (on
// random codes 4060 TOPS of these alone, 3450 of 32 x 32 x 32: the clock falls less), 128 K
// values a step.  A step's rows of a and b go from memory straight to LDS, into rings of
// slots of 128 bytes a row, by four of the waves (by all eight: 4096 x 4096 x 14336 171 ->
// 178 us); one barrier a step says that the next slots are full and the last ones free.
//
// What bounds it: large tiles the matrix cores, whose clock the power limit holds at 1.6 to
// 2.0 GHz (256 x 256: 2480 cycles a step, 2048 of them matrix instructions, 2220 without the
// loads); smaller ones the loads: a CU takes 1 KB of direct-to-LDS loads in 17.5 cycles
// from its L2, but in 38 to 45 where the lines come from HBM, whatever their depth, row
// pitch or sharing (touching them ahead of the loads made every shape 5 to 10% slower).
// A launch's fixed part is 7 to 15 us: its first slots 2.4, the epilogue 4 to 6, the burst
// of all CUs' outputs.  4096 x 28672 x 4096 369 to 380 us, 2530 to 2610 TOPS; 2048 x 6144 x
// 4096 43 to 46 us, 2300; 512 x 4096 x 14336 41 us (split, with its join 7).
#pragma once

#include "cek_int8.h"

namespace cek {

// RA slots of A, RB of B: a step's loads go out RA steps ahead, B's RB.
template <int BM_, int BN_, int WM_, int WN_, int RA_, int RB_, bool GLU_>
struct Int8Tile {
  static constexpr int BM = BM_, BN = BN_, BK = 128, WM = WM_, WN = WN_, RA = RA_, RB = RB_;
  static constexpr bool GLU = GLU_;
  static constexpr int BO = GLU ? BN / 2 : BN;              // output columns
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  static constexpr int ASLOT = BM * BK, BSLOT = BN * BK;
  static constexpr int LW = 4;                              // waves that load: 0 .. LW - 1
  static constexpr int AL = BM / 8 / LW, BL = BN / 8 / LW, L = AL + BL;  // 1 KB loads per such wave and step
  static constexpr int GROUPS = 2 * FM;                     // of FN MFMAs, in a step
  static constexpr int PB = GROUPS > 4 ? GROUPS - 4 : 1, NB = GROUPS - PB;  // the group before the step's barrier
  static constexpr int LB = RA == 2 ? L : (NB * L + GROUPS - 1) / GROUPS;  // loads in the groups from there on
  // in flight at the barrier: what was issued behind the A rows of the next step
  static constexpr int FLY = (RA - 2) * L + (RB > RA ? BL : 0);
  static constexpr int SA = (BM + 63) / 64 * 64, SO = (BO + 63) / 64 * 64;  // scale regions
  static constexpr int NSC = SA + (GLU ? 2 : 1) * SO;
  static constexpr int OUT = BM * BO * 2;
  static constexpr int RINGS = RA * ASLOT + RB * BSLOT, MAIN = RINGS > OUT ? RINGS : OUT;
  static constexpr int SMEM = MAIN + NSC * 4;
  static constexpr int SW = (BO / 4) % 16 == 0 ? 15 : 7;     // swizzle of the staged output's 8-byte units
  // first output column of block column j (lane group g = lane >> 4 holds four from 4 g on)
  static constexpr __device__ int col(int wn, int j) { return GLU ? wn * (TN / 2) + 8 * j : wn * TN + 16 * j; }
  static_assert(FM * 16 * WM == BM && FN * 16 * WN == BN && AL * 8 * LW == BM && BL * 8 * LW == BN, "tile");
  static_assert(GROUPS % 4 == 0 && (!GLU || FN % 2 == 0), "A fragments in a ring of four; gate and up in one wave");
  static_assert(RA >= 2 && (RB == RA || RB == RA + 1) && FLY + LB <= 63, "rings");
  static_assert((BO / 4) % 8 == 0 && SMEM <= 163840, "LDS");
};

template <int N>
__device__ __forceinline__ void tile_barrier() {  // all but the N latest loads have landed, LDS reads are done
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

__device__ inline __amdgpu_buffer_rsrc_t int8_rsrc(const void* p, uint32_t n) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)n, 0x00020000);
}

constexpr uint32_t kOutOfRange = 0x80000000u;  // an offset beyond every resource here: the load gives zeros

// Tile and part of workgroup b of n: runs of n / 8 consecutive ones per XCD (workgroup
// b is on XCD b % 8), in groups of GM tile rows.
template <int GM>
__device__ inline void int8_tile_of(int b, int n, int tiles_m, int tiles_n, int& tm, int& tn, int& part) {
  const int x = b & 7, lo = n >> 3, more = n & 7;
  const int t = x * lo + min(x, more) + (b >> 3), per = tiles_m * tiles_n;
  part = t / per;
  const int q = t - part * per, per_group = GM * tiles_n, group = q / per_group;
  const int first = group * GM, rows = min(tiles_m - first, GM), in = q - group * per_group;
  tm = first + in % rows;
  tn = in / rows;
}

struct Int8Args {
  const uint8_t* a;
  const float* sa;
  const uint8_t* b;
  const float* sb;
  uint16_t* y;
  int32_t* part;  // split K: int32 sums [parts][M][rows of b]
  int M, N, K;    // N: output columns
  int tiles_m, tiles_n, parts;
};

template <class C, class T, int ACT, bool SPLIT>
__global__ __launch_bounds__(C::NT, 1) void int8_tile_kernel(Int8Args p) {
  constexpr int FM = C::FM, FN = C::FN, L = C::L, RA = C::RA, RB = C::RB;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[C::SMEM];
  float* const sc = reinterpret_cast<float*>(smem + C::MAIN);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  int tm, tn, part;
  int8_tile_of<4>(blockIdx.x, gridDim.x, p.tiles_m, p.tiles_n, tm, tn, part);
  const int K = p.K, m0 = tm * C::BM, n0 = tn * C::BO;
  const int rows_m = min(C::BM, p.M - m0), rows_n = min(C::BO, p.N - n0);
  const __amdgpu_buffer_rsrc_t rA = int8_rsrc(p.a + (size_t)m0 * K, (uint32_t)rows_m * (uint32_t)K);
  // The gated block's tile holds sixteen gate rows of b, then the sixteen up rows of the same
  // outputs, and so on: loading waves 0 and 1 take the ones, 2 and 3 the others, and a
  // lane's accumulators hold both factors of its outputs.
  const int up_rows = C::GLU && (wave & 2) ? p.N : 0;
  const __amdgpu_buffer_rsrc_t rB = int8_rsrc(p.b + (size_t)(up_rows + n0) * K, (uint32_t)rows_n * (uint32_t)K);

  // scales to LDS: BM row scales, BO gate (or plain) and BO up scales, in runs of 64
#pragma unroll
  for (int q = 0; q < C::NSC / 64; ++q) {
    if (q % C::NW != wave) continue;
    const bool isA = q < C::SA / 64;
    const int base = isA ? q * 64 : (q * 64 - C::SA) % C::SO;
    const bool up = C::GLU && q * 64 >= C::SA + C::SO;
    const float* src = isA ? p.sa + m0 : p.sb + n0 + (up ? p.N : 0);
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(int8_rsrc(src, (uint32_t)(isA ? rows_m : rows_n) * 4u),
                                             (lds_ptr_t)(sc + 64 * q), 4, (uint32_t)(base + lane) * 4u, 0, 0, 0);
#endif
  }

  // Load i of this wave: rows 8 (wave + LW i) on of the slice, lane l row l >> 3 at position
  // l & 7.  A row's 16-byte chunk k lies at k ^ swz(row): the sixteen rows of a fragment
  // read then fall in all 64 banks.
  auto swz = [](int row) { return (row >> 1) & 7; };
  const int lrow = lane >> 3;
  const uint32_t cofs = (uint32_t)(((lane & 7) ^ swz(8 * (wave & 1) + lrow)) * 16);
  uint32_t va[C::AL], vb[C::BL];
#pragma unroll
  for (int i = 0; i < C::AL; ++i) va[i] = (uint32_t)min(8 * (wave + C::LW * i) + lrow, rows_m - 1) * (uint32_t)K + cofs;
#pragma unroll
  for (int i = 0; i < C::BL; ++i) {
    const int r = 8 * (wave + C::LW * i);
    vb[i] = (uint32_t)min((C::GLU ? (r >> 5) * 16 + (r & 15) : r) + lrow, rows_n - 1) * (uint32_t)K + cofs;
  }
  const int steps = (K + C::BK - 1) / C::BK;
  const int k0 = SPLIT ? (int)((int64_t)steps * part / p.parts) : 0;
  const int n = (SPLIT ? (int)((int64_t)steps * (part + 1) / p.parts) : steps) - k0;  // steps of this part

  uint8_t* const sB = smem + RA * C::ASLOT;
  auto load_a = [&](int i, int step, int slot) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
    // past the part: nothing (zeros); past the row's end: zeros, whatever b has there
    const uint32_t kb = step < n ? (uint32_t)(k0 + step) * C::BK : kOutOfRange, ka = kb + cofs >= (uint32_t)K ? kOutOfRange : kb;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rA, (lds_ptr_t)(smem + slot * C::ASLOT + 1024 * (wave + C::LW * i)), 16, va[i] + ka,
                                             0, 0, 0);
#endif
  };
  auto load_b = [&](int i, int step, int slot) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint32_t kb = step < n ? (uint32_t)(k0 + step) * C::BK : kOutOfRange;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rB, (lds_ptr_t)(sB + slot * C::BSLOT + 1024 * (wave + C::LW * i)), 16, vb[i] + kb,
                                             0, 0, 0);
#endif
  };
  // Load i of the group that step k's barrier lets go: A of step k + RA, then B of step k + RB.
  auto load = [&](int i, int k, int ca, int cb) __attribute__((always_inline)) {
    if (i < C::AL) load_a(i, k + RA, ca);
    else load_b(i - C::AL, k + RB, cb);
  };
  const bool loader = wave < C::LW;
  if (loader) {
#pragma unroll
    for (int s = 0; s < RB - RA; ++s)
#pragma unroll
      for (int i = 0; i < C::BL; ++i) load_b(i, s, s);
#pragma unroll
    for (int s = 0; s < RA; ++s)
#pragma unroll
      for (int i = 0; i < (s + 1 < RA ? L : C::LB); ++i) load(i, s - RA, s, s + RB - RA);
  }

  const int r16 = lane & 15, g = lane >> 4;
  const uint32_t la = (uint32_t)((wm * C::TM + r16) * C::BK), lb = (uint32_t)((wn * C::TN + r16) * C::BK);
  const uint32_t sw = (uint32_t)((g ^ swz(r16)) * 16);
  i4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = i4{0, 0, 0, 0};
  // A step is two halves of 64 K values, FM groups each: A fragment i of the half against
  // its FN B fragments.  A fragments pass through a ring of four: group q's place takes
  // group q + 4's, read as soon as group q's MFMAs are out.  B fragments are held in two
  // sets, the halves'.
  u4 fa[4], fb[2][FN];
  auto read_a = [&](int q, int slot) __attribute__((always_inline)) {  // of group q
    fa[q & 3] = *reinterpret_cast<const u4*>(smem + slot * C::ASLOT + (sw ^ (q < FM ? 0u : 64u)) + la + (q % FM) * 16 * C::BK);
  };
  auto read_b = [&](int j, int slot, int half) __attribute__((always_inline)) {
    fb[half][j] = *reinterpret_cast<const u4*>(sB + slot * C::BSLOT + (sw ^ (64u * half)) + lb + j * 16 * C::BK);
  };

  tile_barrier<C::FLY + C::LB>();
#pragma unroll
  for (int j = 0; j < FN; ++j) read_b(j, 0, 0);
#pragma unroll
  for (int q = 0; q < 4; ++q) read_a(q, 0);

  int ca = 0, cb = 0;
  for (int kt = 0; kt < n; ++kt) {
    const int na = ca + 1 == RA ? 0 : ca + 1, nb = cb + 1 == RB ? 0 : cb + 1;
    const int pa = ca == 0 ? RA - 1 : ca - 1, pb = cb == 0 ? RB - 1 : cb - 1;
#pragma unroll
    for (int q = 0; q < C::GROUPS; ++q) {
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[q % FM][j] = mfma_i8(fb[q / FM][j], fa[q & 3], acc[q % FM][j]);
      // The barrier, a group or more behind the last read of this step's slots: the next
      // step's have landed, this step's are fully read.  Behind the last step the reads
      // are of whatever the next slots hold, and unused.
      if (q == C::PB) tile_barrier<C::FLY>();
      constexpr int QB = FM - 1;                                 // the second half's B fragments: behind groups 0 ..
      if (q < QB) {
#pragma unroll
        for (int j = q * FN / QB; j < (q + 1) * FN / QB; ++j) read_b(j, cb, 1);
      }
      constexpr int Q0 = C::PB > QB ? C::PB : QB, NQ = C::GROUPS - 1 - Q0;  // the next first half's, once its set is free
      if (q >= Q0 && q < Q0 + NQ) {
#pragma unroll
        for (int j = (q - Q0) * FN / NQ; j < (q - Q0 + 1) * FN / NQ; ++j) read_b(j, nb, 0);
      }
      if (q + 4 < C::GROUPS) read_a(q + 4, ca);
      else if (q > C::PB) read_a(q + 4 - C::GROUPS, na);
      else if (q == C::PB) {
#pragma unroll
        for (int i = 0; i <= C::PB + 4 - C::GROUPS; ++i) read_a(i, na);
      }
      // the group of loads that this barrier lets go, then the rest of the one before's
      if (loader) {
        if (q >= C::PB) {
#pragma unroll
          for (int i = (q - C::PB) * C::LB / C::NB; i < (q - C::PB + 1) * C::LB / C::NB; ++i) load(i, kt, ca, cb);
        } else {
#pragma unroll
          for (int i = C::LB + q * (L - C::LB) / C::PB; i < C::LB + (q + 1) * (L - C::LB) / C::PB; ++i)
            load(i, kt - 1, pa, pb);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    ca = na;
    cb = nb;
  }
  tile_barrier<0>();

  // Lane l holds, of block (i, j), row m = l & 15 and columns 4 (l >> 4) + v.
  if constexpr (SPLIT) {
    const int NB = C::GLU ? 2 * p.N : p.N;
    int32_t* P = p.part + (size_t)part * p.M * NB;
    const bool vec = (p.N & 3) == 0;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = m0 + wm * C::TM + i * 16 + r16;
      if (m >= p.M) continue;
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const bool up = C::GLU && (j & 1);
        const int nn = n0 + C::col(wn, up ? j - 1 : j) + 4 * g;
        int32_t* dst = P + (size_t)m * NB + (up ? p.N : 0) + nn;
        if (vec && nn < p.N) *reinterpret_cast<i4*>(dst) = acc[i][j];
        else
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (nn + e < p.N) dst[e] = acc[i][j][e];
      }
    }
    return;
  }
  uint8_t* const out = smem;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = wm * C::TM + i * 16 + r16;
    const float s0 = sc[m];
#pragma unroll
    for (int j = 0; j < FN; j += C::GLU ? 2 : 1) {
      const int nn = C::col(wn, j) + 4 * g;
      const f4 sg = *reinterpret_cast<const f4*>(sc + C::SA + nn);
      float o[4];
      if constexpr (C::GLU) {
        const f4 su = *reinterpret_cast<const f4*>(sc + C::SA + C::SO + nn);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = int8_glu<ACT>(acc[i][j][e], acc[i][j + 1][e], s0, sg[e], su[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = int8_scaled(acc[i][j][e], s0, sg[e]);
      }
      *reinterpret_cast<uint2*>(out + (size_t)m * (C::BO * 2) + ((nn >> 2) ^ (m & C::SW)) * 8) =
          make_uint2(int8_pack2<T>(o[0], o[1]), int8_pack2<T>(o[2], o[3]));
    }
  }
  __syncthreads();
  uint16_t* const Y = p.y + (size_t)m0 * p.N + n0;
  if ((p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0) {
    for (int q = threadIdx.x; q < C::BM * C::BO / 8; q += C::NT) {
      const int r = q / (C::BO / 8), k = q % (C::BO / 8), s = r & C::SW;
      if (r >= rows_m || 8 * k >= rows_n) continue;
      u4 v = *reinterpret_cast<const u4*>(out + (size_t)r * (C::BO * 2) + (((2 * k) ^ s) & ~1) * 8);
      if (s & 1) v = u4{v[2], v[3], v[0], v[1]};
      __builtin_nontemporal_store(v, reinterpret_cast<u4*>(Y + (size_t)r * p.N + 8 * k));
    }
  } else {  // rows that start anywhere: consecutive lanes store consecutive values
    for (int q = threadIdx.x; q < C::BM * C::BO; q += C::NT) {
      const int r = q / C::BO, k = q % C::BO;
      if (r < rows_m && k < rows_n)
        Y[(size_t)r * p.N + k] =
            *reinterpret_cast<const uint16_t*>(out + (size_t)r * (C::BO * 2) + ((k >> 2) ^ (r & C::SW)) * 8 + (k & 3) * 2);
    }
  }
}

}  // namespace cek
