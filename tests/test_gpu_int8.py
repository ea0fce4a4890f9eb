"""GPU parity of the int8 path against its 64-bit oracle.

Products and quantised codes are equal bit for bit: sums are integers, and what follows is a fixed
sequence of fp32 operations.  The gated block lies within the bound that the oracle derives, plus
half a step of the output's type; codes behind the norm may be one off where the fp32 norm lies next
to a border.
"""

import math

import pytest
import torch

from esimd_learning_amd import synthetic
from oracle import int8 as oint8

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def _codes(rows, k, seed, lo=-127, hi=128):
    g = synthetic.gen(seed)
    return torch.randint(lo, hi, (rows, k), generator=g, dtype=torch.int8), torch.rand(rows, generator=g) * 0.02 + 1e-3


def _rows(t, h, seed, dtype):
    x = torch.randn(t, h, generator=synthetic.gen(seed))
    x[:, 3 % h::17] *= 20
    return x.to(dtype)


# ---- codes ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,h", [(1, 1), (3, 7), (1, 8), (5, 64), (2, 129), (9, 136), (4, 512), (1, 1000), (3, 2048), (2, 2056),
                                 (7, 4096), (2, 5120), (1, 14336), (600, 520), (513, 4104), (2, 16384), (2, 16392), (1, 33001),
                                 (2, 40960), (5, 9), (3, 15), (1025, 1001), (1030, 4099), (2, 8195), (1024, 8190), (1, 65536), (1, 65537),
                                 (1, 70000)])
def test_quant(ops, dev, t, h, dtype):
    x = _rows(t, h, t * 1000 + h, dtype)
    q = torch.full((t, h), 77, dtype=torch.int8, device=dev)
    s = torch.empty(t, device=dev)
    ops.esimd_per_token_quant_int8(x.to(dev), q, s)
    want_q, want_s = oint8.quant(x)
    assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu(), want_q)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_ties_and_borders(ops, dev, dtype):
    """Rows whose quotients are ties (scales of few bits) or lie as near to one as 16-bit values can."""
    rows = []
    for amax in (127.0, 254.0, 381.0, 63.5, 0.49609375, 1.0, 3.0, 100.0):   # scales 1, 2, 3, 0.5, 2^-8, and inexact ones
        s = torch.tensor(amax, dtype=dtype).double().div(127).float().double()
        k = torch.arange(0, 127, dtype=torch.float64) + 0.5
        near = (k * s).float().to(dtype)
        bits = near.view(torch.int16)
        row = torch.cat([near, (bits + 1).view(dtype), (bits - 1).view(dtype), -near])
        row[row.abs() > amax] = 0
        rows.append(torch.cat([row, torch.tensor([amax], dtype=dtype), torch.zeros(3, dtype=dtype)]))
    x = torch.stack(rows)
    for cut in (x.shape[1], 511):                                     # the vector and the element form
        y = x[:, -cut:].contiguous()
        q, s = torch.empty(y.shape, dtype=torch.int8, device=dev), torch.empty(len(y), device=dev)
        ops.esimd_per_token_quant_int8(y.to(dev), q, s)
        want_q, want_s = oint8.quant(y)
        assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu(), want_q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [40, 1031, 4096])
def test_quant_ends_of_the_range(ops, dev, h, dtype):
    """Rows of zeros, of the smallest and the largest values, and rows that hold inf or NaN."""
    x = _rows(9, h, 5, dtype)
    fi = torch.finfo(dtype)
    x[0] = 0
    x[1] = 0
    x[1, 2] = fi.smallest_normal * fi.eps            # the smallest subnormal
    x[2] = -fi.smallest_normal
    x[3] = fi.max
    x[3, 1::2] = fi.min
    x[4, h - 1] = math.inf
    x[5, 0] = -math.inf
    x[6, h // 2] = math.nan
    x[7] = math.nan
    q, s = torch.empty(9, h, dtype=torch.int8, device=dev), torch.empty(9, device=dev)
    ops.esimd_per_token_quant_int8(x.to(dev), q, s)
    want_q, want_s = oint8.quant(x)
    assert torch.isnan(want_s).tolist() == [False] * 4 + [True] * 4 + [False]
    assert torch.equal(s.cpu().view(torch.int32)[:4], want_s.view(torch.int32)[:4]) and torch.isnan(s[4:8]).all()
    assert torch.equal(q.cpu(), want_q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,h", [(1, 1), (3, 7), (4, 64), (2, 136), (5, 1000), (4, 5120), (1, 4096), (513, 2048), (3, 8192), (2, 16384),
                                 (2, 16400), (2, 4099), (5, 9), (3, 15), (1030, 1001), (1025, 4099), (1024, 5121), (1027, 8190), (2, 8195), (3, 30001),
                                 (1, 32768), (1, 32769)])
def test_norm_quant(ops, dev, t, h, dtype):
    """The residual and the scale are the oracle's (the scale within fp32's roundings), codes at most one off and
    only next to a border."""
    hid, res, w = _rows(t, h, 1, dtype), _rows(t, h, 2, dtype), synthetic.norm_weight(h, 3, dtype)
    r = res.to(dev)
    q, s = torch.empty(t, h, dtype=torch.int8, device=dev), torch.empty(t, device=dev)
    h_dev = hid.to(dev)
    ops.esimd_fused_add_rms_norm_quant_int8(h_dev, r, w.to(dev), 1e-6, q, s)
    kept, x = oint8.add_rms_norm(hid, res, w, 1e-6)
    assert torch.equal(r.cpu(), kept) and torch.equal(h_dev.cpu(), hid)
    # x in fp32: the mean of squares (its sum in any order: h additions of like sign, h u at most, half of it under
    # the root, and in practice some u sqrt(h)), rsqrt 2 u, two products 2 u; the scale one division more
    u = 2.0 ** -24
    rel = (h / 2 + 8) * u
    want_q, want_s = oint8.quant(x)
    assert ((s.cpu().double() - want_s.double()).abs() <= want_s.double() * rel).all()
    exact = x / want_s.double()[:, None]
    off = q.cpu().double() - exact
    assert (off.abs() <= 0.5 + 127 * 2 * rel).all()
    assert (q.cpu() != want_q).double().mean() <= 4 * 127 * rel + 1.0 / (t * h)


@pytest.mark.parametrize("h", [4096, 4093, 520, 77])
def test_rows_that_start_anywhere(ops, dev, h):
    """Tensors whose storage is not aligned: the same codes, and nothing outside them written."""
    t = 3
    x, res, w = _rows(t, h, 1, torch.float16), _rows(t, h, 2, torch.float16), synthetic.norm_weight(h, 3)
    want_q, want_s = oint8.quant(x)
    for off in (1, 3, 8):
        put = lambda v: torch.cat([torch.zeros(off, dtype=v.dtype), v.reshape(-1)]).to(dev)[off:].view(v.shape)  # noqa: E731
        buf = torch.full((off + t * h + 16,), 99, dtype=torch.int8, device=dev)
        q, s = buf[off:off + t * h].view(t, h), torch.empty(t, device=dev)
        ops.esimd_per_token_quant_int8(put(x), q, s)
        assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
        a, b = torch.empty(t, h, dtype=torch.int8, device=dev), torch.empty(t, device=dev)
        r, r0 = put(res), res.to(dev)
        ops.esimd_fused_add_rms_norm_quant_int8(put(x), r, put(w), 1e-6, q, s)
        ops.esimd_fused_add_rms_norm_quant_int8(x.to(dev), r0, w.to(dev), 1e-6, a, b)
        assert torch.equal(r, r0)
        assert (q - a).abs().max() <= 1 and ((s - b).abs() <= b * 2.0 ** -20).all()
        assert (buf[:off] == 99).all() and (buf[off + t * h:] == 99).all()


def test_norm_quant_not_finite(ops, dev):
    hid, res, w = _rows(4, 264, 1, torch.float16), _rows(4, 264, 2, torch.float16), synthetic.norm_weight(264, 3)
    hid[1, 5], res[2, 9] = math.nan, math.inf
    r = res.to(dev)
    q, s = torch.empty(4, 264, dtype=torch.int8, device=dev), torch.empty(4, device=dev)
    ops.esimd_fused_add_rms_norm_quant_int8(hid.to(dev), r, w.to(dev), 1e-6, q, s)
    assert torch.isnan(s).tolist() == [False, True, True, False] and q[1:3].abs().max() == 0
    zero = torch.zeros(2, 264, dtype=torch.float16, device=dev)
    ops.esimd_fused_add_rms_norm_quant_int8(zero, zero.clone(), w.to(dev), 1e-6, q[:2], s[:2])
    assert (q[:2] == 0).all() and (s[:2] == 2.0 ** -126).all()


# ---- products ------------------------------------------------------------------------

SIZES = [(1, 1, 16), (1, 7, 64), (1, 100, 48), (2, 33, 80), (3, 64, 128), (4, 130, 4096), (5, 1000, 1040), (8, 257, 2576), (13, 24, 144),
         (16, 96, 14336), (17, 100, 512), (31, 260, 2064), (33, 48, 192), (37, 300, 2576), (48, 512, 64), (63, 77, 272), (64, 640, 1024),
         (65, 130, 128), (100, 1, 4096), (127, 255, 336), (128, 256, 128), (129, 257, 1024), (200, 384, 5120), (256, 512, 256),
         (300, 770, 400), (333, 1030, 2560), (512, 600, 4112), (1000, 129, 640), (1025, 520, 896)]


def _product(ops, dev, a, sa, b, sb, dtype, act=None):
    y = torch.full((len(a), len(b) // (2 if act else 1)), math.nan, dtype=dtype, device=dev)
    args = (a.to(dev), sa.to(dev), b.to(dev), sb.to(dev), y)
    ops.esimd_gemm_int8_a8w8_glu(*args, act) if act else ops.esimd_gemm_int8_a8w8(*args)
    return y.cpu()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(ops, dev, m, n, k, dtype):
    (a, sa), (b, sb) = _codes(m, k, m + k, lo=-128), _codes(n, k, n + k + 1, lo=-128)
    got = _product(ops, dev, a, sa, b, sb, dtype)
    assert torch.equal(got, oint8.product(a, sa, b, sb, dtype))


@pytest.mark.parametrize("m", [1, 2, 4, 9, 40, 64, 70, 150])
def test_product_longest_sums(ops, dev, m):
    """K at its limit with codes of one sign: the sums reach 2^31 - 2^18."""
    k, n = 131056, 40
    a, b = torch.full((m, k), -128, dtype=torch.int8), torch.full((n, k), -128, dtype=torch.int8)
    b[1::2] = 127
    b[5, ::2] = 3
    sa, sb = torch.rand(m, generator=synthetic.gen(1)) * 1e-4, torch.rand(n, generator=synthetic.gen(2)) * 1e-4
    assert torch.equal(_product(ops, dev, a, sa, b, sb, torch.float16), oint8.product(a, sa, b, sb, torch.float16))


def _check_gated(got, a, sa, b, sb, act, dtype):
    want, bound = oint8.gated(a, sa, b, sb, act)
    fi = torch.finfo(dtype)
    limit = bound + want.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
    over = want.abs() + bound >= fi.max
    err = (got.double() - want).abs()
    assert (err <= limit)[~over].all(), float((err / limit)[~over].max())
    assert (got[over].double().abs() >= fi.max * (1 - fi.eps)).all()


@pytest.mark.parametrize("dtype,act", [(torch.float16, "gelu_tanh"), (torch.bfloat16, "silu"), (torch.float16, "silu"),
                                       (torch.bfloat16, "gelu_tanh")])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gated(ops, dev, m, n, k, dtype, act):
    (a, sa), (b, sb) = _codes(m, k, m + k), _codes(2 * n, k, n + k + 1)
    sb[:n] /= math.sqrt(k)                # gates of some units
    sb[n:] /= 10 * math.sqrt(k)
    _check_gated(_product(ops, dev, a, sa, b, sb, dtype, act), a, sa, b, sb, act, dtype)


@pytest.mark.parametrize("act", ["gelu_tanh", "silu"])
@pytest.mark.parametrize("m", [1, 30, 130])
def test_gated_far_gates(ops, dev, m, act):
    """Gates from where sigmoid underflows to where it is 1."""
    (a, sa), (b, sb) = _codes(m, 64, 1), _codes(512, 64, 2)
    sb[:256] = torch.logspace(-4, 1, 256)
    sb[256:] = 1e-3
    _check_gated(_product(ops, dev, a, sa, b, sb, torch.bfloat16, act), a, sa, b, sb, act, torch.bfloat16)


@pytest.mark.parametrize("m", [1, 3, 40, 140])
@pytest.mark.parametrize("act", [None, "silu"])
def test_rows_that_are_not_finite_stay_apart(ops, dev, m, act):
    """A NaN scale makes its own row NaN, an infinite one its own values; the others are as without."""
    (a, sa), (b, sb) = _codes(m, 192, 7), _codes(64, 192, 8)
    clean = _product(ops, dev, a, sa, b, sb, torch.float16, act)
    bad = sa.clone()
    bad[m // 2] = math.nan
    got = _product(ops, dev, a, bad, b, sb, torch.float16, act)
    rest = torch.arange(m) != m // 2
    assert torch.isnan(got[m // 2]).all() and torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_rows_do_not_depend_on_the_batch(ops, dev, act):
    """Every kernel gives a row the same bits."""
    (a, sa), (b, sb) = _codes(700, 1088, 11), _codes(520, 1088, 12)
    whole = _product(ops, dev, a, sa, b, sb, torch.bfloat16, act)
    for m in (1, 2, 4, 7, 16, 20, 33, 64, 65, 130, 260, 513):
        assert torch.equal(_product(ops, dev, a[:m], sa[:m], b, sb, torch.bfloat16, act), whole[:m]), m


def test_no_rows_and_refusals(ops, dev):
    a, s, y = torch.zeros(4, 64, dtype=torch.int8, device=dev), torch.ones(4, device=dev), torch.ones(4, 4, dtype=torch.float16, device=dev)
    ops.esimd_gemm_int8_a8w8(a[:0], s[:0], a, s, y[:0])
    ops.esimd_gemm_int8_a8w8(a, s, a[:0].clone(), s[:0], y[:, :0].contiguous())
    ops.esimd_gemm_int8_a8w8_glu(a[:0], s[:0], a, s, y[:0, :2])
    x = torch.ones(0, 64, dtype=torch.float16, device=dev)
    ops.esimd_per_token_quant_int8(x, a[:0], s[:0])
    b = a.clone()
    wide = torch.zeros(4, 80, dtype=torch.int8, device=dev)
    flat = torch.zeros(4 * 64 + 8, dtype=torch.int8, device=dev)
    f16 = torch.zeros(4, 64, dtype=torch.float16, device=dev)
    bad = [lambda: ops.esimd_gemm_int8_a8w8(a.float(), s, b, s, y), lambda: ops.esimd_gemm_int8_a8w8(a, s, b.view(torch.uint8), s, y),
           lambda: ops.esimd_gemm_int8_a8w8(a, s.double(), b, s, y), lambda: ops.esimd_gemm_int8_a8w8(a, s[:3], b, s, y),
           lambda: ops.esimd_gemm_int8_a8w8(a, s, b, s[:2], y), lambda: ops.esimd_gemm_int8_a8w8(a, s, b, s, y.float()),
           lambda: ops.esimd_gemm_int8_a8w8(a, s, b, s, y[:, :3].contiguous()), lambda: ops.esimd_gemm_int8_a8w8(wide[:, :64], s, b, s, y),
           lambda: ops.esimd_gemm_int8_a8w8(a, s, wide, s, y), lambda: ops.esimd_gemm_int8_a8w8(a[:, :24].contiguous(), s, b[:, :24].contiguous(), s, y),
           lambda: ops.esimd_gemm_int8_a8w8(flat[8:].view(4, 64), s, b, s, y), lambda: ops.esimd_gemm_int8_a8w8(a, s, b.cpu(), s, y),
           lambda: ops.esimd_gemm_int8_a8w8(a, s, b, s, a.view(torch.float16)[:, :4].contiguous().t()),
           lambda: ops.esimd_gemm_int8_a8w8(a, s, b, s, a.view(-1)[:32].view(torch.float16).view(4, 4)),
           lambda: ops.esimd_gemm_int8_a8w8_glu(a, s, b, s, y[:, :2].contiguous(), "relu"),
           lambda: ops.esimd_gemm_int8_a8w8_glu(a, s, b[:3], s[:3], y[:, :1].contiguous()),
           lambda: ops.esimd_gemm_int8_a8w8_glu(a, s, b, s, y),
           lambda: ops.esimd_per_token_quant_int8(f16.float(), a, s), lambda: ops.esimd_per_token_quant_int8(f16, a.view(torch.uint8), s),
           lambda: ops.esimd_per_token_quant_int8(f16, a, s[:3]), lambda: ops.esimd_per_token_quant_int8(f16, a[:3], s),
           lambda: ops.esimd_per_token_quant_int8(f16[:, ::2], a, s),
           lambda: ops.esimd_per_token_quant_int8(f16, f16.view(torch.int8)[:2].view(4, 64), s),
           lambda: ops.esimd_fused_add_rms_norm_quant_int8(f16, f16, f16[0], 1e-6, a, s),
           lambda: ops.esimd_fused_add_rms_norm_quant_int8(f16, f16.bfloat16(), f16[0], 1e-6, a, s),
           lambda: ops.esimd_fused_add_rms_norm_quant_int8(f16, f16.clone(), f16[0, :32].clone(), 1e-6, a, s)]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            print("not refused:", i)
    assert (y == 1).all()


# Sizes of no tile: each tile's own, then tiles that split K, in two to eight parts.
TILED = [(771, 12299, 464), (513, 13092, 464), (386, 11726, 464), (513, 9821, 464), (257, 10890, 464), (129, 10885, 464),
         (66, 68, 464)]
SPLIT = [(500, 4090, 14320), (3000, 700, 12000), (66, 5442, 4944), (71, 65, 3056), (65, 70, 4032), (1030, 1030, 16384),
         (68, 5414, 4832), (384, 5122, 13824), (1030, 4098, 14336)]
# Few rows of a wide matrix with short rows, which the tiles take too.
WIDE = [(4, 16390, 496), (16, 21506, 512), (17, 16390, 2032), (32, 28674, 1040), (33, 16402, 240)]


def test_every_tile_is_tested():
    from esimd_learning_amd import cabi
    plan = cabi.load().cek_gemm_int8_plan
    for gated in (0, 1):
        plans = [plan(m, n // (1 + gated), k, gated, 1 << 40) for m, n, k in TILED]
        assert sorted(p // 16 for p in plans) == list(range(7)) and all(p % 16 == 1 for p in plans)
        plans = [plan(m, n // (1 + gated), k, gated, 1 << 40) for m, n, k in SPLIT]
        assert all(p % 16 > 1 for p in plans) and {p // 16 for p in plans} >= {0, 2, 5, 6}
        assert all(plan(m, n // (1 + gated), k, gated, 1 << 40) % 16 == 1 for m, n, k in WIDE if not (gated and m == 4))


@pytest.mark.parametrize("m,n,k", TILED + SPLIT + WIDE)
def test_tiles(ops, dev, m, n, k):
    """Both forms of every tile, whole and split, and without the workspace that the split takes."""
    from esimd_learning_amd import cabi
    lib = cabi.load()
    n -= n % 2
    g = torch.Generator(device=dev).manual_seed(m + n + k)
    a, b = (torch.randint(-128, 128, (rows, k), generator=g, dtype=torch.int8, device=dev) for rows in (m, n))
    sa, sb = torch.rand(m, generator=g, device=dev) * 0.01, torch.rand(n, generator=g, device=dev) * 0.01
    acc = a.double() @ b.double().t()                 # integers below 2^53: exact in any order
    want = (acc.float() * sb * sa[:, None]).bfloat16()
    y = torch.full((m, n), math.nan, dtype=torch.bfloat16, device=dev)
    ops.esimd_gemm_int8_a8w8(a, sa, b, sb, y)
    assert torch.equal(y, want)
    y.fill_(math.nan)
    cabi.check(lib.cek_gemm_int8_a8w8(cabi.ptr(a), cabi.ptr(sa), cabi.ptr(b), cabi.ptr(sb), cabi.ptr(y), m, n, k, cabi.CEK_BF16,
                                      None, 0, cabi.stream_ptr()))
    assert torch.equal(y, want)
    sb /= 127 * math.sqrt(k)                          # gates of some units
    z, z0 = (torch.full((m, n // 2), math.nan, dtype=torch.float16, device=dev) for _ in range(2))
    ops.esimd_gemm_int8_a8w8_glu(a, sa, b, sb, z, "silu")
    cabi.check(lib.cek_gemm_int8_a8w8_glu(cabi.ptr(a), cabi.ptr(sa), cabi.ptr(b), cabi.ptr(sb), cabi.ptr(z0), m, n // 2, k,
                                          cabi.CEK_SILU, cabi.CEK_F16, None, 0, cabi.stream_ptr()))
    assert torch.equal(z, z0)
    gu = acc * sb.double() * sa.double()[:, None]
    gate, up = gu[:, : n // 2], gu[:, n // 2:]
    f = gate * torch.sigmoid(gate) * up
    rel = (16 + 16 * gate.abs() * torch.sigmoid(-gate)) * 2.0 ** -24      # the bound of oracle.int8.gated
    limit = f.abs() * (rel + 2.0 ** -11) + gate.abs() * up.abs() * 2.0 ** -126 + 2.0 ** -25
    assert ((z.double() - f).abs() <= limit).all()


# ---- offsets beyond 32 bits ----------------------------------------------------------

@pytest.mark.parametrize("h", [16, 9])
def test_more_rows_than_a_launch_takes(ops, dev, h):
    t = (1 << 21) + 5
    x = torch.randn(t, h, generator=torch.Generator(device=dev).manual_seed(h), device=dev).half()
    q, s = torch.full((t, h), 77, dtype=torch.int8, device=dev), torch.full((t,), math.nan, device=dev)
    ops.esimd_per_token_quant_int8(x, q, s)
    r = torch.zeros_like(x)
    qn, sn = torch.full_like(q, 77), torch.full_like(s, math.nan)
    ops.esimd_fused_add_rms_norm_quant_int8(x, r, torch.ones(h, dtype=torch.float16, device=dev), 1e-6, qn, sn)
    assert torch.equal(r, x)
    for lo in (0, (1 << 20) - 300, (1 << 21) - 300):                 # 600 rows about each launch's end
        part = x[lo:lo + 600]
        want_q, want_s = oint8.quant(part.cpu())
        assert torch.equal(s[lo:lo + 600].cpu(), want_s) and torch.equal(q[lo:lo + 600].cpu(), want_q)
        pq, ps, pr = torch.empty_like(q[:len(part)]), torch.empty(len(part), device=dev), torch.zeros_like(part)
        ops.esimd_fused_add_rms_norm_quant_int8(part, pr, torch.ones(h, dtype=torch.float16, device=dev), 1e-6, pq, ps)
        assert torch.equal(qn[lo:lo + 600], pq) and torch.equal(sn[lo:lo + 600], ps)
    assert not torch.isnan(s).any() and not torch.isnan(sn).any()


@pytest.mark.parametrize("t,h", [(40001, 131072), (80001, 65536)])
def test_more_values_than_32_bits_count(ops, dev, t, h):
    x = torch.zeros(t, h, dtype=torch.float16, device=dev)
    ends = [0, 2 ** 31 // h, 2 ** 32 // h, 2 ** 32 // h + 1, t - 1]
    rows = torch.randn(len(ends), h, generator=synthetic.gen(1)).half()
    x[ends] = rows.to(dev)
    q, s = torch.full((t, h), 77, dtype=torch.int8, device=dev), torch.empty(t, device=dev)
    ops.esimd_per_token_quant_int8(x, q, s)
    want_q, want_s = oint8.quant(rows)
    assert torch.equal(q[ends].cpu(), want_q) and torch.equal(s[ends].cpu(), want_s)
    assert s.numel() - (s == 2.0 ** -126).sum().item() == len(ends)  # the rest are rows of zeros
    assert sum(int(part.count_nonzero()) for part in q.split(4000)) == int(want_q.count_nonzero())


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m", [1, 16, 64, 300])
def test_weights_beyond_32_bits(ops, dev, m, gated):
    """b of 4.6 GB: every kernel reaches its last rows."""
    n, k = 140000, 32768
    b = torch.empty(n, k, dtype=torch.int8, device=dev)
    for i in range(0, n, 20000):
        b[i:i + 20000] = torch.randint(-128, 128, (20000, k), generator=torch.Generator(device=dev).manual_seed(i), dtype=torch.int8,
                                       device=dev)
    a, sa = _codes(m, k, 5)
    a, sa, sb = a.to(dev), sa.to(dev), torch.rand(n, device=dev) * 0.01
    cols = torch.tensor([0, 1, 65535, 65536, 65537, 69999, 70000, 131071, 131072, 131073, n - 2, n - 1], device=dev)

    def sums(c):
        return a.double() @ b[c].double().t()                        # integers below 2^53: exact in any order
    if gated:
        cols = cols[cols < n // 2]
        y = torch.full((m, n // 2), math.nan, dtype=torch.bfloat16, device=dev)
        ops.esimd_gemm_int8_a8w8_glu(a, sa, b, sb, y)
        few = torch.cat([cols, cols + n // 2])                       # the same rows alone give the same bits
        want = torch.empty(m, len(cols), dtype=torch.bfloat16, device=dev)
        ops.esimd_gemm_int8_a8w8_glu(a, sa, b[few].contiguous(), sb[few].contiguous(), want)
    else:
        y = torch.full((m, n), math.nan, dtype=torch.bfloat16, device=dev)
        ops.esimd_gemm_int8_a8w8(a, sa, b, sb, y)
        want = (sums(cols).float() * sb[cols] * sa[:, None]).bfloat16()
    assert torch.equal(y[:, cols], want) and not torch.isnan(y).any()


@pytest.mark.parametrize("m,n,k", [(20001, 120002, 32), (140000, 130, 32768)])
def test_outputs_and_activations_beyond_32_bits(ops, dev, m, n, k):
    g = torch.Generator(device=dev).manual_seed(m)
    a, b = (torch.empty(rows, k, dtype=torch.int8, device=dev) for rows in (m, n))
    for t in (a, b):
        for part in t.split(20000):
            part.copy_(torch.randint(-128, 128, part.shape, generator=g, dtype=torch.int8, device=dev))
    sa, sb = torch.rand(m, device=dev) * 0.01, torch.rand(n, device=dev) * 0.01
    y = torch.full((m, n), math.nan, dtype=torch.bfloat16, device=dev)
    ops.esimd_gemm_int8_a8w8(a, sa, b, sb, y)
    rows = torch.tensor([0, 8947, 8948, 17895, 17896, 65535, 65536, 131071, 131072, m - 2, m - 1], device=dev)
    rows = rows[rows < m]
    want = ((a[rows].double() @ b.double().t()).float() * sb * sa[rows, None]).bfloat16()
    assert torch.equal(y[rows], want) and not any(torch.isnan(part).any() for part in y.split(4000))


def test_more_rows_than_a_grid_takes(ops, dev):
    long, one = torch.zeros((1 << 24) + 1, 16, dtype=torch.int8, device=dev), torch.zeros(2, 16, dtype=torch.int8, device=dev)
    s, y = torch.ones(len(long), device=dev), torch.empty(2 * len(long), dtype=torch.float16, device=dev)
    for a, b in ((long, one), (one, long)):
        with pytest.raises(RuntimeError, match="2\\^24 rows"):
            ops.esimd_gemm_int8_a8w8(a, s[:len(a)], b, s[:len(b)], y.view(len(a), len(b)))
    with pytest.raises(RuntimeError, match="2\\^24 rows"):
        ops.esimd_gemm_int8_a8w8_glu(long, s, one, s[:2], y[:len(long)].view(-1, 1))
    a, b = long[:-1], one                                            # the most that it takes
    a[-3:] = 7
    b += 1
    ops.esimd_gemm_int8_a8w8(a, s[:-1], b, s[:2], y[:2 * len(a)].view(-1, 2))
    assert (y[:2 * len(a)].view(-1, 2)[-4:].cpu() == torch.tensor([[0.], [112.], [112.], [112.]])).all()
    y.zero_()
    ops.esimd_gemm_int8_a8w8(b, s[:2], a, s[:-1], y[:2 * len(a)].view(2, -1))
    assert (y[:2 * len(a)].view(2, -1)[:, -4:].cpu() == torch.tensor([0., 112., 112., 112.])).all()
