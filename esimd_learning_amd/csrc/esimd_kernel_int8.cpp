// esimd_kernel_int8.cpp -- torch shims of the int8 ops: codes and scales of rows,
// alone or behind the add + RMS norm, the product and the gated block.
#include "torch_ops.h"

#include "shim_common.h"

using namespace cek_shim;

static void check_codes_out(const at::Tensor& ref, const at::Tensor& q, const at::Tensor& s, int64_t rows, const char* op) {
  TORCH_CHECK(q.scalar_type() == at::ScalarType::Char, op, ": out_q must be int8");
  TORCH_CHECK(s.scalar_type() == at::ScalarType::Float, op, ": out_scale must be fp32");
  check_device(q, ref, op, "out_q");
  check_device(s, ref, op, "out_scale");
  check_contig(q, op, "out_q");
  check_contig(s, op, "out_scale");
  TORCH_CHECK(q.numel() == ref.numel(), op, ": out_q must have as many elements as the input");
  TORCH_CHECK(s.numel() == rows, op, ": out_scale must have one element per row (", rows, ")");
  TORCH_CHECK(!overlaps(q, s), op, ": out_q and out_scale must not overlap");
}

void esimd_per_token_quant_int8(at::Tensor input, at::Tensor out_q, at::Tensor out_scale) {
  const char* op = "esimd_per_token_quant_int8";
  TORCH_CHECK(is_io(input.scalar_type()), op, ": input must be fp16 or bf16");
  TORCH_CHECK(input.is_cuda(), op, ": input must be a GPU tensor");
  check_contig(input, op, "input");
  TORCH_CHECK(input.dim() >= 1 && input.size(-1) > 0, op, ": input must have a non-empty last dimension");
  const int64_t H = input.size(-1), rows = input.numel() / H;
  check_codes_out(input, out_q, out_scale, rows, op);
  TORCH_CHECK(!overlaps(out_q, input) && !overlaps(out_scale, input), op, ": outputs must not overlap the input");
  c10::OptionalDeviceGuard guard(input.device());
  check_rc(cek_per_token_quant_int8(input.data_ptr(), rows, H, io_code(input.scalar_type()),
                                    static_cast<int8_t*>(out_q.data_ptr()), static_cast<float*>(out_scale.data_ptr()),
                                    current_stream(input)),
           op);
}

void esimd_fused_add_rms_norm_quant_int8(at::Tensor hidden_states, at::Tensor residual, at::Tensor weight, double eps,
                                         at::Tensor out_q, at::Tensor out_scale) {
  const char* op = "esimd_fused_add_rms_norm_quant_int8";
  const auto& h = hidden_states;
  TORCH_CHECK(is_io(h.scalar_type()), op, ": hidden_states must be fp16 or bf16");
  TORCH_CHECK(residual.scalar_type() == h.scalar_type() && weight.scalar_type() == h.scalar_type(), op,
              ": residual and weight must have the dtype of hidden_states");
  TORCH_CHECK(h.is_cuda(), op, ": hidden_states must be a GPU tensor");
  check_device(residual, h, op, "residual");
  check_device(weight, h, op, "weight");
  check_contig(h, op, "hidden_states");
  check_contig(residual, op, "residual");
  check_contig(weight, op, "weight");
  TORCH_CHECK(h.dim() >= 1 && h.size(-1) > 0, op, ": hidden_states must have a non-empty last dimension");
  TORCH_CHECK(residual.numel() == h.numel(), op, ": residual must match hidden_states");
  TORCH_CHECK(weight.numel() == h.size(-1), op, ": weight must have hidden_states.size(-1) elements");
  const int64_t H = h.size(-1), rows = h.numel() / H;
  check_codes_out(h, out_q, out_scale, rows, op);
  for (auto* t : {&h, &static_cast<const at::Tensor&>(weight)}) {
    TORCH_CHECK(!overlaps(out_q, *t) && !overlaps(out_scale, *t) && !overlaps(residual, *t), op,
                ": outputs must not overlap inputs");
  }
  TORCH_CHECK(!overlaps(out_q, residual) && !overlaps(out_scale, residual), op, ": outputs must not overlap");
  c10::OptionalDeviceGuard guard(h.device());
  check_rc(cek_fused_add_rms_norm_quant_int8(h.data_ptr(), residual.data_ptr(), weight.data_ptr(), rows, H, (float)eps,
                                             io_code(h.scalar_type()), static_cast<int8_t*>(out_q.data_ptr()),
                                             static_cast<float*>(out_scale.data_ptr()), current_stream(h)),
           op);
}

// The checks that both products share; N: columns of the output.
static void check_product(const at::Tensor& a, const at::Tensor& sa, const at::Tensor& b, const at::Tensor& sb,
                          const at::Tensor& y, int64_t N, const char* op) {
  TORCH_CHECK(a.scalar_type() == at::ScalarType::Char && b.scalar_type() == at::ScalarType::Char, op,
              ": a and b must be int8");
  TORCH_CHECK(sa.scalar_type() == at::ScalarType::Float && sb.scalar_type() == at::ScalarType::Float, op,
              ": scales must be fp32");
  TORCH_CHECK(is_io(y.scalar_type()), op, ": output must be fp16 or bf16");
  TORCH_CHECK(a.is_cuda(), op, ": a must be a GPU tensor");
  TORCH_CHECK(a.size(1) == b.size(1), op, ": a and b must have the same K");
  for (auto* t : {&sa, &b, &sb, &y}) check_device(*t, a, op, "operand");
  check_contig(a, op, "a");
  check_contig(b, op, "b");
  check_contig(sa, op, "a_scale");
  check_contig(sb, op, "b_scale");
  check_contig(y, op, "output");
  TORCH_CHECK(a.size(1) > 0 && a.size(1) % 16 == 0, op, ": K must be a positive multiple of 16");
  TORCH_CHECK(a.size(1) <= 131071, op, ": K must be at most 131071 (the sums are held in 32 bits)");
  TORCH_CHECK(a.size(0) <= (1 << 24) && b.size(0) <= (1 << 24), op, ": a and b must have at most 2^24 rows");
  TORCH_CHECK(sa.numel() == a.size(0) && sb.numel() == b.size(0), op, ": a_scale [M] and b_scale [rows of b] required");
  TORCH_CHECK(y.numel() == a.size(0) * N, op, ": output must be [M, ", N, "]");
  for (auto* t : {&a, &sa, &b, &sb})
    TORCH_CHECK(!overlaps(y, *t), op, ": output must not overlap the operands");
}

at::Tensor esimd_gemm_int8_a8w8(at::Tensor a, at::Tensor a_scale, at::Tensor b, at::Tensor b_scale, at::Tensor output) {
  const char* op = "esimd_gemm_int8_a8w8";
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2, op, ": a [M, K] and b [N, K] required");
  const int64_t M = a.size(0), K = a.size(1), N = b.size(0);
  check_product(a, a_scale, b, b_scale, output, N, op);
  c10::OptionalDeviceGuard guard(a.device());
  // shapes with too few tiles split K: int32 partial sums in a workspace from the
  // caching allocator (no kernel runs to allocate or clear it)
  at::Tensor ws;
  const int64_t need = split_workspace(ws, cek_gemm_int8_a8w8_workspace_size(M, N, K), a_scale);
  check_rc(cek_gemm_int8_a8w8(static_cast<const int8_t*>(a.data_ptr()), static_cast<const float*>(a_scale.data_ptr()),
                              static_cast<const int8_t*>(b.data_ptr()), static_cast<const float*>(b_scale.data_ptr()),
                              output.data_ptr(), M, N, K, io_code(output.scalar_type()),
                              need > 0 ? ws.data_ptr() : nullptr, need, current_stream(a)),
           op);
  return output;
}

void esimd_gemm_int8_a8w8_glu(at::Tensor a, at::Tensor a_scale, at::Tensor b, at::Tensor b_scale, at::Tensor output,
                              c10::string_view activation) {
  const char* op = "esimd_gemm_int8_a8w8_glu";
  TORCH_CHECK(activation == "gelu_tanh" || activation == "silu", op, ": activation must be \"gelu_tanh\" or \"silu\"");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2, op, ": a [M, K] and b [2d, K] required");
  TORCH_CHECK(b.size(0) % 2 == 0, op, ": b must have an even number of rows (gate rows, then up rows)");
  const int64_t M = a.size(0), K = a.size(1), d = b.size(0) / 2;
  check_product(a, a_scale, b, b_scale, output, d, op);
  c10::OptionalDeviceGuard guard(a.device());
  at::Tensor ws;
  const int64_t need = split_workspace(ws, cek_gemm_int8_a8w8_glu_workspace_size(M, d, K), a_scale);
  check_rc(cek_gemm_int8_a8w8_glu(static_cast<const int8_t*>(a.data_ptr()), static_cast<const float*>(a_scale.data_ptr()),
                                  static_cast<const int8_t*>(b.data_ptr()), static_cast<const float*>(b_scale.data_ptr()),
                                  output.data_ptr(), M, d, K, activation == "silu" ? CEK_SILU : CEK_GELU_TANH,
                                  io_code(output.scalar_type()), need > 0 ? ws.data_ptr() : nullptr, need,
                                  current_stream(a)),
           op);
}
