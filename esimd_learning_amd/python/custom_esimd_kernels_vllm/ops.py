"""Python wrappers of the ``torch.ops.custom_esimd_kernels_vllm`` ops.

The first four keep the reference's names, signatures and forwarding
(reference python/custom_esimd_kernels_vllm/ops.py:7-67); the docstrings
state this build's contract.  The rest wrap the new ops of the same
namespace.
"""

import torch

_ops = torch.ops.custom_esimd_kernels_vllm


def esimd_gemv_fp8_pern(
    input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
    output: torch.Tensor,
    N: int, K: int,
) -> torch.Tensor:
    """fp8-weight GEMV with a per-output-channel scale, fp32 accumulation.

    input/output: [M, K]/[M, N] fp16 or bf16 of one dtype (every row is
    computed; the reference computes row 0); weight: [N, K] float8_e4m3fn or
    float8_e5m2; weight_scale: [N] fp16, bf16 or fp32.  Returns ``output``.
    """
    return _ops.esimd_gemv_fp8_pern(input, weight, weight_scale, output, N, K)


def esimd_gemv_fp8_pert(
    input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
    output: torch.Tensor,
) -> torch.Tensor:
    """fp8-weight GEMV with a per-tensor fp32 scale (read on the device).

    N and K are taken from weight's shape.  Returns ``output``.
    """
    return _ops.esimd_gemv_fp8_pert(input, weight, weight_scale, output)


def esimd_fused_add_rms_norm_batched(
    hidden_states: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
) -> torch.Tensor:
    """Batched fused residual add + RMSNorm (Gemma-style), in place.

    residual = hidden_states + residual; hidden_states = rmsnorm(residual) *
    weight, with weight already shifted (w + 1.0).  Any number of rows.
    Returns ``hidden_states``.
    """
    return _ops.esimd_fused_add_rms_norm_batched(hidden_states, residual, weight, eps)


def esimd_gemm_fp8_pert(
    input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
    output: torch.Tensor,
) -> torch.Tensor:
    """fp8-weight GEMM with a per-tensor fp32 scale, any M.

    input/output: [M, K]/[M, N] fp16 or bf16 of one dtype; weight [N, K] fp8.
    M <= 16 runs the decode GEMV kernels, larger M the MFMA GEMM.
    """
    return _ops.esimd_gemm_fp8_pert(input, weight, weight_scale, output)


# ---- new ops -------------------------------------------------------------

def esimd_gemv_fp8_pern_fused(input, weights, weight_scales, outputs) -> None:
    """Several per-channel-scale fp8 GEMVs sharing ``input`` in one launch.

    weights[i]: [N_i, K] fp8; weight_scales[i]: [N_i]; outputs[i]: [M, N_i].
    Each output equals esimd_gemv_fp8_pern on its own matrix.
    """
    _ops.esimd_gemv_fp8_pern_fused(input, list(weights), list(weight_scales), list(outputs))


def esimd_gemv_fp8_pert_fused(input, weights, weight_scales, outputs) -> None:
    """Several per-tensor-scale fp8 GEMVs sharing ``input`` in one launch."""
    _ops.esimd_gemv_fp8_pert_fused(input, list(weights), list(weight_scales), list(outputs))


def esimd_fused_add_rms_norm_quant_fp8(
    hidden_states: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float,
    out_q: torch.Tensor, out_scale: torch.Tensor,
) -> None:
    """residual += hidden_states (in place); per-token e4m3 codes of
    rmsnorm(residual) * weight into out_q [T, H] and fp32 scales into
    out_scale [T].  hidden_states is only read."""
    _ops.esimd_fused_add_rms_norm_quant_fp8(hidden_states, residual, weight, eps, out_q, out_scale)


def esimd_per_token_quant_fp8(input: torch.Tensor, out_q: torch.Tensor, out_scale: torch.Tensor) -> None:
    """Per-token e4m3 quantisation: out_scale[t] = max(amax_t / 448, 1/(448*512))."""
    _ops.esimd_per_token_quant_fp8(input, out_q, out_scale)


def esimd_gelu_and_mul(out: torch.Tensor, input: torch.Tensor) -> None:
    """out = gelu_tanh(input[..., :d]) * input[..., d:]."""
    _ops.esimd_gelu_and_mul(out, input)


def esimd_gemv_fp8_gelu_and_mul(
    input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, output: torch.Tensor,
) -> None:
    """Gate/up GEMV over a merged fp8 weight with gelu_and_mul fused.

    input [M, K] fp16/bf16; weight [2d, K] fp8 (gate rows, then up rows);
    weight_scale [2d] fp16/bf16/fp32; output [M, d] of input's dtype.
    output equals esimd_gemv_fp8_pern into [M, 2d] followed by
    esimd_gelu_and_mul, in one launch for decode batches.
    """
    _ops.esimd_gemv_fp8_gelu_and_mul(input, weight, weight_scale, output)


def esimd_fused_add_rms_norm_gemv_fp8(
    hidden_states: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float,
    residual_out: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, output: torch.Tensor,
    gelu_and_mul: bool = False,
) -> None:
    """residual_out = hidden_states + residual; output = the fp8 GEMV of
    rmsnorm(residual_out) * weight (with ``gelu_and_mul``: w holds gate then up
    rows and output [M, d] is gelu_tanh(gate) * up).  One launch for up to
    four rows; the values equal esimd_fused_add_rms_norm_batched followed by
    the GEMV.  hidden_states and residual are only read."""
    _ops.esimd_fused_add_rms_norm_gemv_fp8(hidden_states, residual, weight, eps, residual_out, w, w_scale, output,
                                           gelu_and_mul)


def esimd_fused_add_rms_norm_quant_gemv_fp8(
    hidden_states: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float,
    residual_out: torch.Tensor, out_q: torch.Tensor, out_scale: torch.Tensor,
    b: torch.Tensor, b_scale: torch.Tensor, output: torch.Tensor, gelu_and_mul: bool = False,
) -> None:
    """esimd_fused_add_rms_norm_quant_fp8 (into residual_out, out_q, out_scale)
    followed by esimd_gemm_fp8_a8w8 (or its gelu_and_mul form), one launch
    for up to four rows."""
    _ops.esimd_fused_add_rms_norm_quant_gemv_fp8(hidden_states, residual, weight, eps, residual_out, out_q,
                                                 out_scale, b, b_scale, output, gelu_and_mul)


def esimd_qk_norm_rope(
    q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
    positions: torch.Tensor, eps: float, theta: float = 10000.0, is_neox: bool = True,
) -> None:
    """Per-head RMSNorm then rotary embedding of q and k, in place."""
    _ops.esimd_qk_norm_rope(q, k, q_weight, k_weight, positions, eps, theta, is_neox)


def gemv_tail_counters(n_q, n_k, device) -> torch.Tensor:
    """Zeroed arrival counters for esimd_gemv_fp8_qk_norm_rope (64 per head)."""
    return torch.zeros(64 * (n_q + n_k), dtype=torch.int32, device=device)


def esimd_gemv_fp8_qk_norm_rope(
    input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, output: torch.Tensor,
    q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor, n_q: int, n_k: int,
    eps: float, theta: float, is_neox: bool, counters: torch.Tensor,
    q_out: torch.Tensor = None,
) -> None:
    """The QKV GEMV (esimd_gemv_fp8_pern into output [M, N]) followed by
    esimd_qk_norm_rope on its q columns [0, n_q hd) and k columns
    [n_q hd, (n_q + n_k) hd), in one launch for decode batches.  counters:
    int32 device tensor of >= 64 * (n_q + n_k) elements
    (``gemv_tail_counters``, allocated once by the caller, not per call, so
    that the call can be captured in a graph), zero before the first call and
    left zero by each.  q_out (optional, [M, n_q hd]) also receives the rotated q heads,
    as a copy of output's q columns would."""
    _ops.esimd_gemv_fp8_qk_norm_rope(input, weight, weight_scale, output, q_weight, k_weight, positions, n_q, n_k,
                                     eps, theta, is_neox, counters, q_out)


def esimd_gemv_fp8_add_rms_norm_defer_groups(N: int) -> int:
    """G, the number of partial sums of squares per row that
    esimd_gemv_fp8_add_rms_norm_defer writes for N output columns (N / 16,
    or N / 12 where that fills more CUs: N = 3072 -> 256); 0 if N is not a
    multiple of 16."""
    return _ops.esimd_gemv_fp8_add_rms_norm_defer_groups(N)


def esimd_defer_norm_shift(norm_weight: torch.Tensor) -> int:
    """The norm_shift E for esimd_gemv_fp8_add_rms_norm_defer with this norm
    weight: the smallest E with 2^E >= max|norm_weight| (so that the
    producer's output cannot overflow whatever the residual holds).  Reads
    the weight's maximum back to the host: call it once per weight, not per
    step."""
    return _ops.esimd_defer_norm_shift(float(norm_weight.float().abs().max()))


def esimd_gemv_fp8_add_rms_norm_defer(
    input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, residual: torch.Tensor,
    norm_weight: torch.Tensor, output: torch.Tensor, row_ss: torch.Tensor, norm_shift: int = 0,
) -> None:
    """The producer half of an add + RMSNorm deferred into the next GEMV
    (up to four rows, e4m3 weights): o = the GEMV's rounded output; residual
    += o in place; output = residual * norm_weight * 2^-norm_shift (rounded;
    the norm without its 1 / rms); row_ss [M, G] fp32, G =
    ``esimd_gemv_fp8_add_rms_norm_defer_groups(N)``, = the sums of squares of
    the unrounded (o + residual) * 2^-norm_shift over G equal runs of
    columns.  Feed output and row_ss to a ``*_rs`` op with eps *
    4^-norm_shift, which then applies 2^norm_shift / rms.  With norm_shift =
    ``esimd_defer_norm_shift(norm_weight)`` the output cannot overflow; with
    0 an fp16 output overflows where |residual * norm_weight| > 65504."""
    _ops.esimd_gemv_fp8_add_rms_norm_defer(input, weight, weight_scale, residual, norm_weight, output, row_ss,
                                           norm_shift)


def esimd_gemv_fp8_pern_rs(
    input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, output: torch.Tensor,
    row_ss: torch.Tensor, eps: float,
) -> None:
    """esimd_gemv_fp8_pern with each output row m scaled by
    rsqrt(sum(row_ss[m]) / K + eps) (the deferred norm's consumer)."""
    _ops.esimd_gemv_fp8_pern_rs(input, weight, weight_scale, output, row_ss, eps)


def esimd_gemv_fp8_gelu_and_mul_rs(
    input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, output: torch.Tensor,
    row_ss: torch.Tensor, eps: float,
) -> None:
    """esimd_gemv_fp8_gelu_and_mul with the gate and up rows scaled by the
    deferred norm's rsqrt(sum(row_ss[m]) / K + eps) before gelu_and_mul."""
    _ops.esimd_gemv_fp8_gelu_and_mul_rs(input, weight, weight_scale, output, row_ss, eps)


def esimd_gemv_fp8_qk_norm_rope_rs(
    input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, output: torch.Tensor,
    q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor, n_q: int, n_k: int,
    eps: float, theta: float, is_neox: bool, counters: torch.Tensor, row_ss: torch.Tensor, row_eps: float,
    q_out: torch.Tensor = None,
) -> None:
    """esimd_gemv_fp8_qk_norm_rope with the GEMV's rows scaled by the
    deferred norm's rsqrt(sum(row_ss[m]) / K + row_eps) before QK-norm and
    RoPE."""
    _ops.esimd_gemv_fp8_qk_norm_rope_rs(input, weight, weight_scale, output, q_weight, k_weight, positions, n_q,
                                        n_k, eps, theta, is_neox, counters, row_ss, row_eps, q_out)


def kv4_cache(num_blocks, n_kv, block_size, head_dim, device) -> torch.Tensor:
    """A 4-bit key/value cache, uint8 [num_blocks, n_kv, block_size, head_dim + 8].

    One (block, kv head) of bs tokens holds, in this order, the K codes
    [bs, head_dim / 2] (value d: nibble d % 2 of byte d / 2), the V codes
    [bs / 4, head_dim / 4, 4] in 16-bit words (values 4u .. 4u + 3 of token
    4t + i are the nibbles of word [t, u, i]), and the K and the V parameters
    [bs], a bf16 step s and a bf16 centre m each; a value is m + s (c - 7.5).
    block_size: a power of two from 16 to 256; head_dim 64, 128 or 256.  Not
    initialised: what lies behind a request's length is never used."""
    return torch.empty(num_blocks, n_kv, block_size, head_dim + 8, dtype=torch.uint8, device=device)


def kv_free_ring(num_blocks, device):
    """(free_ring, ring_state) with all blocks free, in ascending order."""
    ring = torch.arange(num_blocks, dtype=torch.int32, device=device)
    return ring, torch.tensor([0, num_blocks], dtype=torch.int32, device=device)


def esimd_kv_block_tables(
    kv_lens: torch.Tensor, keep_lens: torch.Tensor, q_lens: torch.Tensor, block_size: int,
    free_ring: torch.Tensor, ring_state: torch.Tensor, block_tables: torch.Tensor,
    kv_lens_out: torch.Tensor, ring_state_out: torch.Tensor, cu_q: torch.Tensor,
    slot_mapping: torch.Tensor, positions: torch.Tensor, status: torch.Tensor, fixed_rows: bool = False,
) -> None:
    """Block tables, slots and positions of one step, from the lengths alone.

    Request r holds kv_lens[r] cached tokens in the first ceil(kv_lens /
    block_size) entries of block_tables[r].  keep_lens[r] of them stay (fewer
    after rejected drafts, 0 for a request that ended or starts over) and
    q_lens[r] new ones follow.  Blocks it lacks are taken from the free ring,
    blocks it no longer needs are returned to it, both in request order and
    ascending in the table; a block returned by a call can be taken from the
    next call on.  free_ring int32 [num_blocks] with ring_state int32 [2] =
    (place of the first free block, how many are free): ``kv_free_ring``.

    Written: block_tables and free_ring (the changed entries), kv_lens_out =
    keep + q, ring_state_out, cu_q int32 [R + 1] (offsets of the requests' new
    tokens), slot_mapping and positions int64 [T] of the new tokens in order
    (behind the last one: -1 and 0), and status int32 [R]: 0; 1 the blocks up
    to and with this request's are more than are free; 2 block_tables is too
    narrow for it; 3 the new tokens up to and with its own are more than T.  A
    request with status != 0 gets no new token (its q counts as 0) and takes
    no block, but returns what lies behind keep_lens.  Status 1 and 3 count the
    wishes of all requests before, refused ones too; a request that needs no
    new block is never refused for one.

    A refused request closes up the rows: those behind it begin where cu_q says,
    earlier than q_lens alone would put them, so that a caller lays out its rows
    by cu_q, or sees from status that nobody was refused.  With ``fixed_rows``
    the rows do not depend on who was refused (a captured step, whose rows are
    laid out before it runs): cu_q are the offsets of q_lens (negative ones as 0,
    no further than T), and a refused request's rows are padding, slot -1 and
    position 0.  Status 3 then counts the wishes of requests with status 2 too.

    kv_lens_out may be kv_lens and ring_state_out ring_state (a captured step
    replayed); no other output may share memory with another argument.  A block
    is free or one request's: what several requests read is not shared here.
    Lengths are taken within 0 .. the table's reach, keep_lens within 0 ..
    kv_lens (2^31 - 1 keeps all).  At most 4096 requests."""
    _ops.esimd_kv_block_tables(kv_lens, keep_lens, q_lens, block_size, free_ring, ring_state, block_tables, kv_lens_out,
                               ring_state_out, cu_q, slot_mapping, positions, status, fixed_rows)


def esimd_kv4_cache_write(
    k: torch.Tensor, v: torch.Tensor, kv_cache: torch.Tensor, slot_mapping: torch.Tensor,
) -> None:
    """Quantise k and v rows to 4 bits into kv_cache at their slots.

    k, v [T, n_kv, head_dim] or [T, n_kv * head_dim], fp16 or bf16, any row
    stride; slot_mapping int64 [T], block * block_size + token.  Rows whose slot
    lies outside the cache (-1: padding) are skipped.  A slot may occur once.
    Per row and head: m = bf16((min + max) / 2), s = bf16(max(max - m, m - min)
    / 7.5), c = clamp(rint((x - m) / s + 7.5), 0, 15); a row with a value that
    is not finite reads back as NaN throughout."""
    _ops.esimd_kv4_cache_write(k, v, kv_cache, slot_mapping)


def esimd_kv4_cache_read(
    kv_cache: torch.Tensor, slot_mapping: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
) -> None:
    """The cached rows of slot_mapping [T] into k and v [T, n_kv, head_dim] (or
    [T, n_kv * head_dim]), fp16 or bf16: m + s (c - 7.5), rounded once.  Rows
    whose slot lies outside the cache are zero."""
    _ops.esimd_kv4_cache_read(kv_cache, slot_mapping, k, v)


def esimd_kv4_attention(
    q: torch.Tensor, kv_cache: torch.Tensor, block_tables: torch.Tensor, kv_lens: torch.Tensor,
    cu_q: torch.Tensor, out: torch.Tensor, scale: float, max_q_len: int = 0, max_kv_len: int = 0,
    window: int = 0,
) -> None:
    """Causal attention of new tokens over the cache, which holds theirs too.

    q, out [T, n_q, head_dim] or [T, n_q * head_dim] (any row strides); rows
    cu_q[r] .. cu_q[r + 1] - 1 are the last tokens of request r, whose kv_lens[r]
    keys and values lie in the blocks of block_tables[r].  Row at position p
    sees keys 0 .. p, with window > 0 keys p - window + 1 .. p; query head h
    reads kv head h / (n_q / n_kv).  out = sum softmax(scale q k) v; rows without
    a key (kv_lens 0) are zero; rows of out before cu_q[0] or behind cu_q[R] are
    left as they were.  Tokens whose table entry lies outside the cache count
    as absent.  cu_q ascends.  |q| and |v| up to 2^100, and V steps up to 2^9
    where scores pass 2^22; weights times V steps are rounded to 2^-12 of
    themselves, or 2^-34 of the largest that the row sees.  Other rows, finite or
    not, and tokens that a row does not see leave it as it is.  max_q_len and
    max_kv_len, the longest of the batch (0: not known), choose the kernels;
    wrong ones cost time, and change results by that rounding and the order of
    sums alone."""
    _ops.esimd_kv4_attention(q, kv_cache, block_tables, kv_lens, cu_q, out, scale, max_q_len, max_kv_len, window)


def esimd_gemm_fp8_a8w8(
    a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
    output: torch.Tensor,
) -> torch.Tensor:
    """output[m, n] = a_scale[m] * b_scale[n] * sum_k a[m, k] * b[n, k] (e4m3 x e4m3)."""
    return _ops.esimd_gemm_fp8_a8w8(a, a_scale, b, b_scale, output)


def esimd_gemm_fp8_a8w8_gelu_and_mul(
    a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
    output: torch.Tensor,
) -> None:
    """esimd_gemm_fp8_a8w8 over a merged [2d, K] gate/up weight, then
    gelu_and_mul, fused for M <= 16: output [M, d]."""
    _ops.esimd_gemm_fp8_a8w8_gelu_and_mul(a, a_scale, b, b_scale, output)


# ---- the int8 path ---------------------------------------------------------

def esimd_per_token_quant_int8(input: torch.Tensor, out_q: torch.Tensor, out_scale: torch.Tensor) -> None:
    """int8 codes and one fp32 scale of each row of input [..., H] (fp16 or bf16).

    out_scale[t] = max(amax_t / 127, 2^-126); out_q = input / out_scale[t] to the
    nearest integer, ties to even.  Takes activations (a row per token) and, when a
    model is loaded, an [N, K] weight (a row per output channel).  A row with a
    value that is not finite gets scale NaN and codes 0: its products are NaN."""
    _ops.esimd_per_token_quant_int8(input, out_q, out_scale)


def esimd_fused_add_rms_norm_quant_int8(
    hidden_states: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float,
    out_q: torch.Tensor, out_scale: torch.Tensor,
) -> None:
    """residual += hidden_states (in place); int8 codes and scales of
    rmsnorm(residual) * weight into out_q [T, H] and out_scale [T], as
    esimd_per_token_quant_int8 of the normed rows before any rounding to 16
    bits.  hidden_states is only read.

    The normed values are fp32: a code whose exact quotient lies next to a half may be
    one off (some ten of a million; the same every time for the same call)."""
    _ops.esimd_fused_add_rms_norm_quant_int8(hidden_states, residual, weight, eps, out_q, out_scale)


def esimd_gemm_int8_a8w8(
    a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
    output: torch.Tensor,
) -> torch.Tensor:
    """output[m, n] = (sum_k a[m, k] * b[n, k]) * b_scale[n] * a_scale[m], the sum exact.

    a [M, K], b [N, K] int8, scales fp32 [M] and [N], output [M, N] fp16 or bf16.
    M and N up to 2^24 (decode steps stream the weights, prompts run MFMA tiles), K a
    multiple of 16 up to 131071.  A row of the output does not depend on the others,
    on M or on the kernel that served the call.  Returns ``output``."""
    return _ops.esimd_gemm_int8_a8w8(a, a_scale, b, b_scale, output)


def esimd_gemm_int8_a8w8_glu(
    a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
    output: torch.Tensor, activation: str = "gelu_tanh",
) -> None:
    """The gated block in one call: output[m, i] = act(g) * u, g and u the fp32
    values that esimd_gemm_int8_a8w8 has for rows i and d + i of b [2d, K] (gate rows, then
    up rows), not rounded before the product.  activation: "gelu_tanh" or
    "silu"; output [M, d] fp16 or bf16."""
    _ops.esimd_gemm_int8_a8w8_glu(a, a_scale, b, b_scale, output, activation)
