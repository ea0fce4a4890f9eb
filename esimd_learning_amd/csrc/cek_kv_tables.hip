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
// All integer work on a few kilobytes: latency is what it costs.  One
// workgroup holds the requests (up to four a thread) and does the scans in
// LDS, the tables and the ring; kv_lens_out and ring_state_out are written
// after the barrier behind the last read of kv_lens and ring_state, so that
// they may be the same memory.
#include "cek_common.h"

namespace cek {

constexpr int kTablesThreads = 1024;
constexpr int kTablesMaxRequests = 4096;

struct KvTablesArgs {
  const int32_t *kv_lens, *keep_lens, *q_lens, *ring_state;
  int32_t *ring, *tables, *kv_lens_out, *ring_state_out, *cu_q, *status;
  int64_t *slots, *positions;
  int64_t table_stride, T;
  int R, cap, width, bs_log2;
};

// Inclusive scans of N values over the workgroup, in thread order.
template <int N>
__device__ inline void wg_scan(int64_t (&x)[N], int64_t (*sh)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t y = __shfl_up((long long)x[i], off, 64);
      if (lane >= off) x[i] += y;
    }
  }
  if (lane == 63)
    for (int i = 0; i < N; ++i) sh[wave][i] = x[i];
  __syncthreads();
  for (int w = 0; w < waves; ++w)
    if (w < wave)
      for (int i = 0; i < N; ++i) x[i] += sh[w][i];
  __syncthreads();
}

// The slot and position of token t: its request by bisection in cu[0 .. R].
template <typename CU, typename KEEP>
__device__ inline void token_slot(const KvTablesArgs& a, int64_t t, const CU& cu, const KEEP& keep_of) {
  int64_t pos = 0, slot = -1;
  if (t < cu(a.R)) {
    int lo = 0, hi = a.R;  // cu(lo) <= t < cu(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu(mid) <= t) lo = mid;
      else hi = mid;
    }
    pos = keep_of(lo) + (t - cu(lo));
    const int32_t blk = a.tables[(int64_t)lo * a.table_stride + (pos >> a.bs_log2)];
    slot = blk < 0 ? -1 : ((int64_t)blk << a.bs_log2) + (pos & ((1 << a.bs_log2) - 1));
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

__global__ __launch_bounds__(kTablesThreads) void kv_tables_kernel(KvTablesArgs a, int fill_slots) {
  __shared__ int64_t sh[kTablesThreads / 64][3];
  __shared__ int32_t cu_s[kTablesMaxRequests + 1], keep_s[kTablesMaxRequests];
  const int tid = threadIdx.x, nt = blockDim.x;
  const int per = (a.R + nt - 1) / nt;  // requests per thread, consecutive
  const int bs = 1 << a.bs_log2;
  const int64_t reach = (int64_t)a.width << a.bs_log2;  // tokens that a table row holds
  // the ring's state, kept in range whatever it holds
  int64_t head = a.ring_state[0], count = a.ring_state[1];
  count = count < 0 ? 0 : (count > a.cap ? a.cap : count);
  head %= a.cap;
  if (head < 0) head += a.cap;

  int64_t len[4], keep[4], q[4], need[4], sum[2] = {0, 0};
  int st[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = tid * per + j;
    len[j] = keep[j] = q[j] = need[j] = 0;
    st[j] = 0;
    if (j < per && r < a.R) {
      len[j] = min((int64_t)max(a.kv_lens[r], 0), reach);
      keep[j] = min((int64_t)max(a.keep_lens[r], 0), len[j]);
      q[j] = max(a.q_lens[r], 0);
      if (keep[j] + q[j] > reach) st[j] = 2;
      if (st[j]) q[j] = 0;
      need[j] = max(((keep[j] + q[j] + bs - 1) >> a.bs_log2) - ((len[j] + bs - 1) >> a.bs_log2), (int64_t)0);
      sum[0] += need[j];
      sum[1] += q[j];
    }
  }
  const int64_t own0 = sum[0], own1 = sum[1];
  wg_scan<2>(sum, reinterpret_cast<int64_t(*)[2]>(sh));
  sum[0] -= own0;
  sum[1] -= own1;
  // requests whose blocks or rows the sums up to them leave no room for
  int64_t gone[4], tot[3] = {0, 0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sum[0] += need[j];
    sum[1] += q[j];
    if (need[j] > 0 && sum[0] > count) st[j] = 1;
    else if (q[j] > 0 && sum[1] > a.T) st[j] = 3;
    if (st[j]) need[j] = q[j] = 0;
    gone[j] = max(((len[j] + bs - 1) >> a.bs_log2) - ((keep[j] + q[j] + bs - 1) >> a.bs_log2), (int64_t)0);
    tot[0] += need[j];
    tot[1] += q[j];
    tot[2] += gone[j];
  }
  int64_t at[3] = {tot[0], tot[1], tot[2]};
  wg_scan<3>(at, sh);
  const int64_t end0 = at[0], end1 = at[1], end2 = at[2];
#pragma unroll
  for (int i = 0; i < 3; ++i) at[i] -= tot[i];
  // every read of kv_lens, keep_lens and ring_state is behind the scans' barriers
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = tid * per + j;
    if (j < per && r < a.R) {
      const int64_t have = (len[j] + bs - 1) >> a.bs_log2, want = (keep[j] + q[j] + bs - 1) >> a.bs_log2;
      int32_t* row = a.tables + (int64_t)r * a.table_stride;
      for (int64_t i = 0; i < need[j]; ++i) {
        int64_t p = head + at[0] + i;
        if (p >= a.cap) p -= a.cap;
        row[have + i] = a.ring[p];
      }
      for (int64_t i = 0; i < gone[j]; ++i) {
        int64_t p = head + count + at[2] + i;
        p -= p >= a.cap ? a.cap : 0;
        p -= p >= a.cap ? a.cap : 0;
        a.ring[p] = row[want + i];
      }
      a.cu_q[r] = cu_s[r] = (int32_t)at[1];
      keep_s[r] = (int32_t)keep[j];
      a.kv_lens_out[r] = (int32_t)(keep[j] + q[j]);
      a.status[r] = st[j];
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) at[i] += i == 0 ? need[j] : (i == 1 ? q[j] : gone[j]);
  }
  if (tid == nt - 1) {
    a.cu_q[a.R] = cu_s[a.R] = (int32_t)end1;
    a.ring_state_out[0] = (int32_t)((head + end0) % a.cap);
    a.ring_state_out[1] = (int32_t)(count - end0 + end2);
  }
  if (!fill_slots) return;
  __syncthreads();  // tables and cu_s of the whole workgroup
  for (int64_t t = tid; t < a.T; t += nt)
    token_slot(a, t, [&](int r) { return (int64_t)cu_s[r]; }, [&](int r) { return (int64_t)keep_s[r]; });
}

// Slots and positions of many tokens, behind kv_tables_kernel on the stream:
// what stays of a request is what it has now less its new tokens.
__global__ __launch_bounds__(256) void kv_slots_kernel(KvTablesArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= a.T) return;
  token_slot(a, t, [&](int r) { return (int64_t)a.cu_q[r]; },
             [&](int r) { return (int64_t)a.kv_lens_out[r] - (a.cu_q[r + 1] - a.cu_q[r]); });
}

}  // namespace cek

using namespace cek;

// Tokens up to which the one workgroup fills the slots itself.
constexpr int64_t kTablesOneLaunch = 4096;

extern "C" int cek_kv_block_tables(const int32_t* kv_lens, const int32_t* keep_lens, const int32_t* q_lens, int64_t R,
                                   int64_t block_size, int32_t* free_ring, int64_t num_blocks, const int32_t* ring_state,
                                   int32_t* block_tables, int64_t table_stride, int64_t max_blocks,
                                   int32_t* kv_lens_out, int32_t* ring_state_out, int32_t* cu_q, int64_t* slot_mapping,
                                   int64_t* positions, int64_t T, int32_t* status, void* stream) {
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
                       __builtin_ctzll((unsigned long long)block_size)};
  hipStream_t st = (hipStream_t)stream;
  const int one = T <= kTablesOneLaunch;
  kv_tables_kernel<<<1, kTablesThreads, 0, st>>>(a, one);
  int rc = check_launch();
  if (rc != CEK_OK || one) return rc;
  kv_slots_kernel<<<(unsigned)((T + 255) / 256), 256, 0, st>>>(a);
  return check_launch();
}
