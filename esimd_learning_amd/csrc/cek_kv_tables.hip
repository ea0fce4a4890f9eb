// cek_kv_tables.hip -- block tables, slots and positions of a step's tokens
// from the requests' lengths, gfx950.
//
// Request r has len[r] cached tokens in ceil(len / bs) blocks of its table row;
// keep of them stay and q new ones follow, so it wants ceil((keep + q) / bs)
// blocks.  The free blocks are a ring (head, count): missing blocks are taken
// from the head on in request order, the ones no longer wanted are put behind
// the tail -- places that no block is taken from in the same call, so nothing
// is read after it was overwritten.  Offsets are prefix sums over the requests.
//
// All integer work on a few kilobytes: what it costs is latency, of the launch,
// two rounds of loads and four barriers (8 requests 3.5 us, a pass among others 6.0;
// 256 requests with prompts 8.5 and the second launch 3.9).  One workgroup, no larger than the
// requests and tokens need, holds up to four requests a thread, scans their
// counts by DPP, keeps the offsets in LDS and hands the moved blocks and the
// tokens out evenly, each finding its request by bisection there; a new token's
// block comes from the ring itself, so that nothing waits for the tables that are
// being written.  Above kTablesOneLaunch tokens a second launch fills the slots.
// With fixed_rows a request's rows lie where the wishes (q) of those before it put
// them, granted or not: cu_q follows the wishes, and rows that were not granted have
// no slot.  kv_lens_out and ring_state_out are written behind the barrier that follows the
// last read of kv_lens and ring_state, so that they may be the same memory.
#include <algorithm>

#include "cek_kv4.h"

namespace cek {

constexpr int kTablesThreads = 1024;
constexpr int kTablesMaxRequests = 4096;
constexpr int64_t kTablesOneLaunch = 4096;

struct KvTablesArgs {
  const int32_t *kv_lens, *keep_lens, *q_lens, *ring_state;
  int32_t *ring, *tables, *kv_lens_out, *ring_state_out, *cu_q, *status;
  int64_t *slots, *positions;
  int64_t table_stride, T;
  int R, cap, width, bs_log2;
  int fixed_rows;
};

__device__ inline int64_t wave_scan_incl(int64_t x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up((long long)x, off, 64);
    if (lane >= off) x += y;
  }
  return x;
}

// Inclusive scans of N values over the workgroup, in thread order; total: the sums.
template <typename I, int N>
__device__ inline void wg_scan(I (&x)[N], I (&total)[N], I (*sh)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = wave_scan_incl(x[i]);
    if (lane == 63) sh[wave][i] = x[i];
    total[i] = 0;
  }
  __syncthreads();
  for (int w = 0; w < waves; ++w)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (w < wave) x[i] += sh[w][i];
      total[i] += sh[w][i];
    }
  __syncthreads();
}

// The last i < n with at[i] <= x; at[0] <= x, at[n] > x.
__device__ inline int find_in(const int32_t* at, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// I: the type of the counts' sums -- 32 bits where they cannot overflow.
template <typename I>
__global__ __launch_bounds__(kTablesThreads) void kv_tables_kernel(KvTablesArgs a, int fill_slots) {
  constexpr int N = kTablesMaxRequests;
  __shared__ I sh2[kTablesThreads / 64][2], sh3[kTablesThreads / 64][3];
  // offsets of the requests' new tokens, taken and returned blocks; kept tokens (-1: refused), blocks held and wanted
  __shared__ int32_t at_q[N + 1], at_need[N + 1], at_gone[N + 1], keep_s[N], have_s[N], want_s[N];
  const int tid = threadIdx.x, nt = blockDim.x;
  const int per = (a.R + nt - 1) / nt;  // requests per thread, consecutive
  const int bs = 1 << a.bs_log2;
  const int64_t reach = (int64_t)a.width << a.bs_log2;  // tokens that a table row holds
  // the ring's state, kept in range whatever it holds
  const int count = min(max(a.ring_state[1], 0), a.cap);
  int head = a.ring_state[0];
  if (head < 0 || head >= a.cap) head = (head % a.cap + a.cap) % a.cap;
  auto place = [&](int64_t i) {  // of the ring, i < 3 cap from the head on
    i += head;
    i -= i >= a.cap ? a.cap : 0;
    i -= i >= a.cap ? a.cap : 0;
    return i - (i >= a.cap ? a.cap : 0);
  };

  int64_t q[4];
  I rows_of[4];  // rows that the request's new tokens take
  int len[4], keep[4], have[4], need[4], st[4];
  I sum[2] = {0, 0}, total2[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = tid * per + j;
    len[j] = keep[j] = have[j] = need[j] = st[j] = 0;
    q[j] = 0;
    rows_of[j] = 0;
    if (j < per && r < a.R) {
      len[j] = (int)min((int64_t)max(a.kv_lens[r], 0), reach);
      keep[j] = min(max(a.keep_lens[r], 0), len[j]);
      q[j] = max(a.q_lens[r], 0);
      rows_of[j] = (I)min(q[j], a.T + 1);
      if (keep[j] + q[j] > reach) st[j] = 2, q[j] = 0, rows_of[j] = a.fixed_rows ? rows_of[j] : 0;
      have[j] = (len[j] + bs - 1) >> a.bs_log2;
      need[j] = max((int)((keep[j] + q[j] + bs - 1) >> a.bs_log2) - have[j], 0);
      // (counts beyond what there is are as good as one more than that)
      sum[0] += (I)min(need[j], a.cap + 1);
      sum[1] += rows_of[j];
    }
  }
  const I own[2] = {sum[0], sum[1]};
  wg_scan<I, 2>(sum, total2, sh2);
  sum[0] -= own[0];
  sum[1] -= own[1];
  // requests whose blocks or rows the sums up to them leave no room for
  int want[4], gone[4];
  I at[3] = {0, 0, 0}, total[3];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sum[0] += (I)min(need[j], a.cap + 1);
    sum[1] += rows_of[j];
    if (st[j] == 0) st[j] = need[j] > 0 && sum[0] > (I)count ? 1 : (q[j] > 0 && sum[1] > (I)a.T ? 3 : 0);
    if (st[j]) need[j] = 0, q[j] = 0, rows_of[j] = a.fixed_rows ? rows_of[j] : 0;
    want[j] = (int)((keep[j] + q[j] + bs - 1) >> a.bs_log2);
    gone[j] = min(max(have[j] - want[j], 0), a.cap + 1);
    at[0] += (I)need[j];
    at[1] += rows_of[j];
    at[2] += (I)gone[j];
  }
  const I mine[3] = {at[0], at[1], at[2]};
  wg_scan<I, 3>(at, total, sh3);  // (the reads of kv_lens and ring_state are behind its barriers)
#pragma unroll
  for (int i = 0; i < 3; ++i) at[i] -= mine[i];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = tid * per + j;
    if (j < per && r < a.R) {
      at_need[r] = (int)at[0];
      a.cu_q[r] = at_q[r] = (int)min(at[1], (I)a.T);
      at_gone[r] = (int)at[2];
      keep_s[r] = st[j] ? -1 : keep[j];
      have_s[r] = have[j];
      want_s[r] = want[j];
      a.kv_lens_out[r] = keep[j] + (int)q[j];
      a.status[r] = st[j];
    }
    at[0] += (I)need[j];
    at[1] += rows_of[j];
    at[2] += (I)gone[j];
  }
  const int taken = (int)total[0], rows = (int)min(total[1], (I)a.T);
  // (lengths of more blocks than there are return no more than the ring has room for
  // beside all that was free: no place is read and written)
  const int given = (int)min((int64_t)total[2], (int64_t)a.cap - count);
  if (tid == 0) {
    at_need[a.R] = taken;
    a.cu_q[a.R] = at_q[a.R] = rows;
    at_gone[a.R] = (int)total[2];
    a.ring_state_out[0] = (int)place(taken);
    a.ring_state_out[1] = count - taken + given;
  }
  __syncthreads();
  // The blocks that are taken, and those that are returned: a row's entries beyond
  // the wanted ones are its own, and the ring's places behind the free blocks no one's.
  for (int i = tid; i < taken; i += nt) {
    const int r = find_in(at_need, a.R, i);
    a.tables[(int64_t)r * a.table_stride + have_s[r] + i - at_need[r]] = a.ring[place(i)];
  }
  for (int i = tid; i < given; i += nt) {
    const int r = find_in(at_gone, a.R, i);
    a.ring[place((int64_t)count + i)] = a.tables[(int64_t)r * a.table_stride + want_s[r] + i - at_gone[r]];
  }
  if (!fill_slots) return;
  for (int t = tid; t < (int)a.T; t += nt) {
    int64_t pos = 0, slot = -1;
    if (t < rows) {
      const int r = find_in(at_q, a.R, t);
      if (keep_s[r] >= 0) {
        pos = keep_s[r] + t - at_q[r];
        const int i = (int)(pos >> a.bs_log2);
        const int32_t blk = i < have_s[r] ? a.tables[(int64_t)r * a.table_stride + i]
                                          : a.ring[place((int64_t)at_need[r] + i - have_s[r])];
        slot = blk < 0 ? -1 : ((int64_t)blk << a.bs_log2) + (pos & (bs - 1));
      }
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
}

// Slots and positions of many tokens, behind kv_tables_kernel on the stream:
// what stays of a request is what it has now less its new tokens.
__global__ __launch_bounds__(256) void kv_slots_kernel(KvTablesArgs a) {
  __shared__ int32_t at_q[kTablesMaxRequests + 1];
  for (int i = threadIdx.x; i <= a.R; i += 256) at_q[i] = a.cu_q[i];
  __syncthreads();
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= a.T) return;
  int64_t pos = 0, slot = -1;
  if (t < at_q[a.R]) {
    const int r = find_in(at_q, a.R, (int)t);
    if (a.status[r] == 0) {
      pos = (int64_t)a.kv_lens_out[r] - at_q[r + 1] + t;
      const int32_t blk = a.tables[(int64_t)r * a.table_stride + (pos >> a.bs_log2)];
      slot = blk < 0 ? -1 : ((int64_t)blk << a.bs_log2) + (pos & ((1 << a.bs_log2) - 1));
    }
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

}  // namespace cek

using namespace cek;

static int block_tables_call(const int32_t* kv_lens, const int32_t* keep_lens, const int32_t* q_lens, int64_t R,
                             int64_t block_size, int32_t* free_ring, int64_t num_blocks, const int32_t* ring_state,
                             int32_t* block_tables, int64_t table_stride, int64_t max_blocks, int32_t* kv_lens_out,
                             int32_t* ring_state_out, int32_t* cu_q, int64_t* slot_mapping, int64_t* positions,
                             int64_t T, int32_t* status, int fixed_rows, void* stream) {
  if (R < 0 || T < 0 || T > INT32_MAX || num_blocks <= 0 || num_blocks > INT32_MAX || max_blocks <= 0 ||
      table_stride < max_blocks)
    return CEK_ERR_INVALID;
  if (block_size < 16 || block_size > 256 || (block_size & (block_size - 1))) return CEK_ERR_UNSUPPORTED;
  if (R > kTablesMaxRequests || max_blocks * block_size > INT32_MAX) return CEK_ERR_UNSUPPORTED;
  if (!ring_state || !free_ring || !ring_state_out || !cu_q || (T > 0 && (!slot_mapping || !positions)) ||
      (R > 0 && (!kv_lens || !keep_lens || !q_lens || !block_tables || !kv_lens_out || !status)))
    return CEK_ERR_INVALID;
  const KvTablesArgs a{kv_lens, keep_lens, q_lens, ring_state, free_ring, block_tables, kv_lens_out, ring_state_out, cu_q,
                       status, slot_mapping, positions, table_stride, T, (int)R, (int)num_blocks, (int)max_blocks,
                       __builtin_ctzll((unsigned long long)block_size), fixed_rows};
  hipStream_t st = (hipStream_t)stream;
  const int one = T <= kTablesOneLaunch;
  // a thread for each request and, where they are few, for each token
  const int64_t want = std::max<int64_t>(R, one ? T : 256);
  const int threads = (int)std::min<int64_t>(kTablesThreads, std::max<int64_t>(1, (want + 63) / 64) * 64);
  if (R * (std::max<int64_t>(T, num_blocks) + 1) < INT32_MAX) kv_tables_kernel<int><<<1, threads, 0, st>>>(a, one);
  else kv_tables_kernel<int64_t><<<1, threads, 0, st>>>(a, one);
  int rc = check_launch();
  if (rc != CEK_OK || one) return rc;
  kv_slots_kernel<<<(unsigned)((T + 255) / 256), 256, 0, st>>>(a);
  return check_launch();
}

extern "C" int cek_kv_block_tables(const int32_t* kv_lens, const int32_t* keep_lens, const int32_t* q_lens, int64_t R,
                                   int64_t block_size, int32_t* free_ring, int64_t num_blocks, const int32_t* ring_state,
                                   int32_t* block_tables, int64_t table_stride, int64_t max_blocks,
                                   int32_t* kv_lens_out, int32_t* ring_state_out, int32_t* cu_q, int64_t* slot_mapping,
                                   int64_t* positions, int64_t T, int32_t* status, void* stream) {
  return block_tables_call(kv_lens, keep_lens, q_lens, R, block_size, free_ring, num_blocks, ring_state, block_tables,
                           table_stride, max_blocks, kv_lens_out, ring_state_out, cu_q, slot_mapping, positions, T,
                           status, 0, stream);
}

extern "C" int cek_kv_block_tables_fixed_rows(const int32_t* kv_lens, const int32_t* keep_lens, const int32_t* q_lens,
                                              int64_t R, int64_t block_size, int32_t* free_ring, int64_t num_blocks,
                                              const int32_t* ring_state, int32_t* block_tables, int64_t table_stride,
                                              int64_t max_blocks, int32_t* kv_lens_out, int32_t* ring_state_out,
                                              int32_t* cu_q, int64_t* slot_mapping, int64_t* positions, int64_t T,
                                              int32_t* status, void* stream) {
  return block_tables_call(kv_lens, keep_lens, q_lens, R, block_size, free_ring, num_blocks, ring_state, block_tables,
                           table_stride, max_blocks, kv_lens_out, ring_state_out, cu_q, slot_mapping, positions, T,
                           status, 1, stream);
}
