// esimd_kernel_kv.cpp -- torch shims of the 4-bit key/value cache's operators
// (no reference op): block tables and slots, cache writes and reads, attention.
//
// As in esimd_kernel.cpp: checks, a device guard, the current HIP stream of the
// first operand's device and one C-ABI call; nothing synchronises.
#include "torch_ops.h"

#include <algorithm>
#include <cmath>
#include <iterator>
#include <string>

#include "shim_common.h"

using namespace cek_shim;

namespace {

struct Cache {
  int64_t num_blocks, n_kv, block_size, hd, stride;
};

Cache check_cache(const at::Tensor& c, const at::Tensor& ref, const char* op) {
  TORCH_CHECK(c.scalar_type() == at::ScalarType::Byte, op, ": kv_cache must be uint8");
  check_device(c, ref, op, "kv_cache");
  TORCH_CHECK(c.dim() == 4 && c.numel() > 0 && c.size(3) > 8, op,
              ": kv_cache must be [num_blocks, n_kv, block_size, head_dim + 8]");
  Cache k{c.size(0), c.size(1), c.size(2), c.size(3) - 8, c.stride(0)};
  TORCH_CHECK(k.hd == 64 || k.hd == 128 || k.hd == 256, op, ": head_dim must be 64, 128 or 256, got ", k.hd);
  TORCH_CHECK(k.block_size >= 16 && k.block_size <= 256 && (k.block_size & (k.block_size - 1)) == 0, op,
              ": block_size must be a power of two from 16 to 256, got ", k.block_size);
  const int64_t head = k.block_size * (k.hd + 8);
  TORCH_CHECK(c.stride(3) == 1 && c.stride(2) == k.hd + 8 && (k.n_kv == 1 || c.stride(1) == head), op,
              ": a block of kv_cache must be contiguous");
  if (k.num_blocks == 1) k.stride = k.n_kv * head;
  TORCH_CHECK(k.stride % 16 == 0 && k.stride >= k.n_kv * head, op,
              ": blocks of kv_cache must be a multiple of 16 bytes apart and not overlap");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0, op, ": kv_cache must be 16-byte aligned");
  return k;
}

// Rows [T, heads, hd] or [T, heads * hd] with any row stride: that stride.
int64_t check_rows(const at::Tensor& t, const at::Tensor& ref, int64_t heads, int64_t hd, const char* op,
                   const char* name) {
  check_device(t, ref, op, name);
  TORCH_CHECK(is_io(t.scalar_type()), op, ": ", name, " must be fp16 or bf16");
  const bool flat = t.dim() == 2 && t.size(1) == heads * hd && t.stride(1) == 1;
  const bool split = t.dim() == 3 && t.size(1) == heads && t.size(2) == hd && t.stride(2) == 1 &&
                     (heads == 1 || t.stride(1) == hd);
  TORCH_CHECK(flat || split, op, ": ", name, " must be [T, ", heads, ", ", hd, "] or [T, ", heads * hd,
              "] with contiguous rows");
  const int64_t stride = t.size(0) <= 1 ? heads * hd : t.stride(0);
  TORCH_CHECK(stride >= heads * hd, op, ": rows of ", name, " must not overlap");
  return stride;
}

// Whether rows of a and b (n elements of one type, strides sa and sb) share
// bytes: by their extents, but for columns of one buffer side by side.
bool rows_overlap(const at::Tensor& a, int64_t sa, int64_t na, const at::Tensor& b, int64_t sb, int64_t nb) {
  if (a.size(0) == 0 || b.size(0) == 0) return false;
  const int64_t e = a.element_size();
  const auto pa = reinterpret_cast<intptr_t>(a.data_ptr()), pb = reinterpret_cast<intptr_t>(b.data_ptr());
  const intptr_t ea = pa + ((a.size(0) - 1) * sa + na) * e, eb = pb + ((b.size(0) - 1) * sb + nb) * e;
  if (pa >= eb || pb >= ea) return false;
  if (sa != sb || a.size(0) == 1 || b.size(0) == 1) return true;
  const int64_t row = sa * e;
  const int64_t off = (((int64_t)pb - (int64_t)pa) % row + row) % row;  // where b's columns start in a's rows
  return off < na * e || off + nb * e > row;
}

// Whether a tensor that is written (any strides) shares bytes with the rows.
bool extent_overlaps(const at::Tensor& a, int64_t sa, int64_t na, const at::Tensor& b) {
  if (a.size(0) == 0 || b.numel() == 0) return false;
  const auto pa = reinterpret_cast<intptr_t>(a.data_ptr()), pb = reinterpret_cast<intptr_t>(b.data_ptr());
  const intptr_t ea = pa + ((a.size(0) - 1) * sa + na) * a.element_size();
  int64_t last = 0;
  for (int64_t d = 0; d < b.dim(); ++d) last += (b.size(d) - 1) * b.stride(d);
  return pa < pb + (last + 1) * b.element_size() && pb < ea;
}

void check_ints(const at::Tensor& t, const at::Tensor& ref, int64_t n, at::ScalarType type, const char* op,
                const char* name) {
  check_device(t, ref, op, name);
  check_contig(t, op, name);
  TORCH_CHECK(t.scalar_type() == type && t.dim() == 1 && (n < 0 || t.numel() == n), op, ": ", name, " must be ",
              type == at::ScalarType::Int ? "int32" : "int64", n < 0 ? ", one-dimensional" : "", n < 0 ? "" : " [",
              n < 0 ? "" : std::to_string(n), n < 0 ? "" : "]");
}

int64_t check_tables(const at::Tensor& t, const at::Tensor& ref, int64_t R, const char* op) {
  check_device(t, ref, op, "block_tables");
  TORCH_CHECK(t.scalar_type() == at::ScalarType::Int && t.dim() == 2 && t.size(0) == R && t.size(1) > 0, op,
              ": block_tables must be int32 [requests, max_blocks]");
  const int64_t stride = R <= 1 ? t.size(1) : t.stride(0);
  TORCH_CHECK((t.size(1) == 1 || t.stride(1) == 1) && stride >= t.size(1), op, ": rows of block_tables must be contiguous");
  return stride;
}

}  // namespace

void esimd_kv_block_tables(at::Tensor kv_lens, at::Tensor keep_lens, at::Tensor q_lens, int64_t block_size,
                           at::Tensor free_ring, at::Tensor ring_state, at::Tensor block_tables, at::Tensor kv_lens_out,
                           at::Tensor ring_state_out, at::Tensor cu_q, at::Tensor slot_mapping, at::Tensor positions,
                           at::Tensor status, bool fixed_rows) {
  const char* op = "esimd_kv_block_tables";
  const auto i32 = at::ScalarType::Int, i64 = at::ScalarType::Long;
  TORCH_CHECK(kv_lens.dim() == 1, op, ": kv_lens must be int32, one-dimensional");
  const int64_t R = kv_lens.numel(), T = slot_mapping.numel();
  TORCH_CHECK(R <= 4096, op, ": at most 4096 requests");
  TORCH_CHECK(block_size >= 16 && block_size <= 256 && (block_size & (block_size - 1)) == 0, op,
              ": block_size must be a power of two from 16 to 256, got ", block_size);
  check_ints(kv_lens, kv_lens, R, i32, op, "kv_lens");
  check_ints(keep_lens, kv_lens, R, i32, op, "keep_lens");
  check_ints(q_lens, kv_lens, R, i32, op, "q_lens");
  check_ints(free_ring, kv_lens, -1, i32, op, "free_ring");
  TORCH_CHECK(free_ring.numel() > 0, op, ": free_ring must hold an element for each block");
  check_ints(ring_state, kv_lens, 2, i32, op, "ring_state");
  check_ints(kv_lens_out, kv_lens, R, i32, op, "kv_lens_out");
  check_ints(ring_state_out, kv_lens, 2, i32, op, "ring_state_out");
  check_ints(cu_q, kv_lens, R + 1, i32, op, "cu_q");
  check_ints(slot_mapping, kv_lens, T, i64, op, "slot_mapping");
  check_ints(positions, kv_lens, T, i64, op, "positions");
  check_ints(status, kv_lens, R, i32, op, "status");
  const int64_t stride = check_tables(block_tables, kv_lens, R, op);
  TORCH_CHECK(block_tables.size(1) * block_size <= INT32_MAX, op, ": a row of block_tables reaches beyond 2^31 tokens");
  // every output apart from the inputs and the other outputs, but for lengths
  // and ring state that are updated in place
  struct Range { uintptr_t at, end; };
  const auto range = [](const at::Tensor& t) {
    const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
    return Range{at, at + t.nbytes()};
  };
  const auto meet = [](const Range& x, const Range& y) { return x.at < x.end && y.at < y.end && x.at < y.end && y.at < x.end; };
  Range table = range(block_tables);
  if (R > 0) table.end = table.at + ((R - 1) * stride + block_tables.size(1)) * 4;
  const Range ins[] = {range(kv_lens), range(keep_lens), range(q_lens), range(ring_state)};
  const Range outs[] = {range(kv_lens_out), range(ring_state_out), range(free_ring), range(cu_q), range(slot_mapping),
                        range(positions), range(status), table};
  for (size_t i = 0; i < std::size(outs); ++i) {
    for (const auto& x : ins)
      TORCH_CHECK(!meet(outs[i], x) || (x.at == outs[i].at && ((i == 0 && x.at == ins[0].at) || (i == 1 && x.at == ins[3].at))),
                  op, ": an output overlaps an input (kv_lens_out may be kv_lens, ring_state_out ring_state)");
    for (size_t j = 0; j < i; ++j) TORCH_CHECK(!meet(outs[i], outs[j]), op, ": outputs overlap");
  }
  c10::OptionalDeviceGuard guard(kv_lens.device());
  const auto p = [](const at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
  const auto call = fixed_rows ? cek_kv_block_tables_fixed_rows : cek_kv_block_tables;
  check_rc(call(p(kv_lens), p(keep_lens), p(q_lens), R, block_size, p(free_ring), free_ring.numel(), p(ring_state),
                p(block_tables), stride, block_tables.size(1), p(kv_lens_out), p(ring_state_out), p(cu_q),
                static_cast<int64_t*>(slot_mapping.data_ptr()), static_cast<int64_t*>(positions.data_ptr()), T,
                p(status), current_stream(kv_lens)),
           op);
}

void esimd_kv4_cache_write(at::Tensor k, at::Tensor v, at::Tensor kv_cache, at::Tensor slot_mapping) {
  const char* op = "esimd_kv4_cache_write";
  const Cache c = check_cache(kv_cache, k, op);
  const int64_t ks = check_rows(k, k, c.n_kv, c.hd, op, "k"), vs = check_rows(v, k, c.n_kv, c.hd, op, "v");
  const int64_t T = k.size(0), n = c.n_kv * c.hd;
  TORCH_CHECK(v.scalar_type() == k.scalar_type(), op, ": k and v must have the same dtype");
  TORCH_CHECK(v.size(0) == T, op, ": k and v must have the same rows");
  check_ints(slot_mapping, k, T, at::ScalarType::Long, op, "slot_mapping");
  TORCH_CHECK(!extent_overlaps(k, ks, n, kv_cache) && !extent_overlaps(v, vs, n, kv_cache), op,
              ": kv_cache overlaps k or v");
  c10::OptionalDeviceGuard guard(k.device());
  check_rc(cek_kv4_cache_write(k.data_ptr(), v.data_ptr(), kv_cache.data_ptr(),
                               static_cast<const int64_t*>(slot_mapping.data_ptr()), T, c.n_kv, c.hd, c.block_size,
                               c.num_blocks, ks, vs, c.stride, io_code(k.scalar_type()), current_stream(k)),
           op);
}

void esimd_kv4_cache_read(at::Tensor kv_cache, at::Tensor slot_mapping, at::Tensor k, at::Tensor v) {
  const char* op = "esimd_kv4_cache_read";
  const Cache c = check_cache(kv_cache, kv_cache, op);
  const int64_t ks = check_rows(k, kv_cache, c.n_kv, c.hd, op, "k"), vs = check_rows(v, kv_cache, c.n_kv, c.hd, op, "v");
  const int64_t T = slot_mapping.numel(), n = c.n_kv * c.hd;
  TORCH_CHECK(v.scalar_type() == k.scalar_type(), op, ": k and v must have the same dtype");
  TORCH_CHECK(k.size(0) == T && v.size(0) == T, op, ": k and v must have a row for each slot");
  check_ints(slot_mapping, kv_cache, T, at::ScalarType::Long, op, "slot_mapping");
  TORCH_CHECK(!extent_overlaps(k, ks, n, kv_cache) && !extent_overlaps(v, vs, n, kv_cache) &&
                  !rows_overlap(k, ks, n, v, vs, n),
              op, ": k and v must not overlap each other or kv_cache");
  c10::OptionalDeviceGuard guard(kv_cache.device());
  check_rc(cek_kv4_cache_read(kv_cache.data_ptr(), static_cast<const int64_t*>(slot_mapping.data_ptr()), k.data_ptr(),
                              v.data_ptr(), T, c.n_kv, c.hd, c.block_size, c.num_blocks, ks, vs, c.stride,
                              io_code(k.scalar_type()), current_stream(kv_cache)),
           op);
}

void esimd_kv4_attention(at::Tensor q, at::Tensor kv_cache, at::Tensor block_tables, at::Tensor kv_lens, at::Tensor cu_q,
                         at::Tensor out, double scale, int64_t max_q_len, int64_t max_kv_len, int64_t window) {
  const char* op = "esimd_kv4_attention";
  const Cache c = check_cache(kv_cache, q, op);
  TORCH_CHECK(q.dim() == 2 || q.dim() == 3, op, ": q must be [T, n_q, head_dim] or [T, n_q * head_dim]");
  const int64_t width = q.dim() == 3 ? q.size(1) * q.size(2) : q.size(1), n_q = width / c.hd;
  TORCH_CHECK(n_q > 0 && width % c.hd == 0 && n_q % c.n_kv == 0, op, ": q's heads must be a multiple of the cache's ",
              c.n_kv, " heads of ", c.hd);
  const int64_t qs = check_rows(q, q, n_q, c.hd, op, "q"), os = check_rows(out, q, n_q, c.hd, op, "out");
  const int64_t T = q.size(0), R = kv_lens.numel();
  TORCH_CHECK(out.scalar_type() == q.scalar_type(), op, ": q and out must have the same dtype");
  TORCH_CHECK(out.size(0) == T, op, ": q and out must have the same rows");
  check_ints(kv_lens, q, R, at::ScalarType::Int, op, "kv_lens");
  check_ints(cu_q, q, R + 1, at::ScalarType::Int, op, "cu_q");
  const int64_t ts = check_tables(block_tables, q, R, op);
  TORCH_CHECK(block_tables.size(1) * c.block_size <= INT32_MAX, op,
              ": a row of block_tables reaches beyond 2^31 tokens");
  TORCH_CHECK(scale > 0 && std::isfinite((float)scale) && (float)scale > 0, op, ": scale must be positive and finite");
  TORCH_CHECK(max_q_len >= 0 && max_kv_len >= 0 && window >= 0 && window <= INT32_MAX, op,
              ": max_q_len, max_kv_len and window must not be negative");
  TORCH_CHECK(!rows_overlap(q, qs, width, out, os, width) && !extent_overlaps(out, os, width, kv_cache), op,
              ": out must not overlap q or kv_cache");
  c10::OptionalDeviceGuard guard(q.device());
  at::Tensor ws;
  const int64_t need = split_workspace(
      ws, cek_kv4_attention_workspace_size(T, R, n_q, c.n_kv, c.hd, max_q_len, max_kv_len), q);
  check_rc(cek_kv4_attention(q.data_ptr(), kv_cache.data_ptr(), static_cast<const int32_t*>(block_tables.data_ptr()),
                             static_cast<const int32_t*>(kv_lens.data_ptr()),
                             static_cast<const int32_t*>(cu_q.data_ptr()), out.data_ptr(), T, R, n_q, c.n_kv, c.hd,
                             c.block_size, c.num_blocks, qs, os, c.stride, ts, block_tables.size(1), (float)scale,
                             max_q_len, max_kv_len, window, io_code(q.scalar_type()),
                             need > 0 ? ws.data_ptr() : nullptr, need, current_stream(q)),
           op);
}
