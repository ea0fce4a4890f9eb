"""CPU: pins of the int8 oracle, and the refusals of the int8 entry points before any GPU work."""

import ctypes as C
from fractions import Fraction

import pytest
import torch

import esimd_learning_amd
from esimd_learning_amd import cabi, synthetic
from oracle import int8 as oint8

P, ODD, N = C.c_void_p(16), C.c_void_p(8), None     # never dereferenced: every call below fails its checks first
INVALID, OK = cabi.CEK_ERR_INVALID, cabi.CEK_OK


# ---- the oracle ------------------------------------------------------------------

def _nearest_even(v):
    """The integer nearest to a fraction, ties to even, by integer arithmetic."""
    n, d = v.numerator, v.denominator
    f, r = divmod(n, d)
    return f + (2 * r > d or (2 * r == d and f % 2 == 1))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_quant_by_fractions(dtype):
    x = torch.randn(6, 40, generator=synthetic.gen(3)).to(dtype)
    x[1] *= 1e-3
    x[2] = torch.arange(40) - 20 + 0.5
    x[2, 0] = 127.0                        # scale 1: every value a tie
    x[3] = 0
    x[4] = 0
    x[4, 7] = torch.finfo(dtype).tiny
    q, s = oint8.quant(x)
    for t in range(6):
        assert s[t] == max(torch.tensor(float(x[t].abs().max()), dtype=torch.float64).div(127).float().item(), 2.0 ** -126)
        step = Fraction(float(s[t]))
        assert q[t].tolist() == [_nearest_even(Fraction(float(v)) / step) for v in x[t]]
    assert q[2, 1:5].tolist() == [-18, -18, -16, -16] and q[3].abs().max() == 0


def test_quant_not_finite():
    x = torch.randn(4, 16, generator=synthetic.gen(4))
    x[1, 3], x[2, 5] = float("inf"), float("nan")
    q, s = oint8.quant(x)
    assert torch.isnan(s).tolist() == [False, True, True, False] and q[1:3].abs().max() == 0


def test_product_by_integers():
    a = torch.randint(-128, 128, (3, 64), generator=synthetic.gen(5), dtype=torch.int8)
    b = torch.randint(-128, 128, (4, 64), generator=synthetic.gen(6), dtype=torch.int8)
    acc = oint8.sums(a, b)
    for m in range(3):
        for n in range(4):
            assert acc[m, n] == sum(int(u) * int(v) for u, v in zip(a[m], b[n]))
    top = torch.full((1, 131056), -128, dtype=torch.int8)
    assert oint8.sums(top, top) == 131056 * 16384 < 2 ** 31


def test_norm_and_activations_against_torch():
    h, r = (synthetic.activations(5, 96, seed=i) for i in (7, 8))
    w = synthetic.norm_weight(96, seed=9)
    kept, x = oint8.add_rms_norm(h, r, w, 1e-6)
    assert torch.equal(kept, h + r)
    t = h.double() + r.double()
    ref = torch.nn.functional.rms_norm(t, (96,), w.double(), 1e-6)
    assert ((x - ref).abs() <= ref.abs() * 2.0 ** -11 + 1e-9).all()       # r' is rounded, t is not
    g = torch.linspace(-12, 12, 1001, dtype=torch.float64)
    assert torch.allclose(oint8.act(g, "silu")[0], torch.nn.functional.silu(g), rtol=1e-12, atol=1e-15)
    assert torch.allclose(oint8.act(g, "gelu_tanh")[0], torch.nn.functional.gelu(g, approximate="tanh"), rtol=1e-9, atol=1e-14)


# ---- refusals ----------------------------------------------------------------------

def _call(fn, base, change):
    assert set(change) <= set(base), change
    return fn(*[change.get(n, base[n]) for n in base])


GEMM = dict(a=P, sa=P, b=P, sb=P, y=P, M=4, N=8, K=64, out=0, ws=N, ws_bytes=0, stream=N)
BAD = [*[({n: N}, INVALID) for n in ("a", "sa", "b", "sb", "y")], (dict(a=ODD), INVALID), (dict(b=ODD), INVALID),
       (dict(M=-1), INVALID), (dict(M=2 ** 31), INVALID), (dict(M=2 ** 24 + 1), INVALID), (dict(N=2 ** 24 + 1), INVALID), (dict(N=-1), INVALID), (dict(N=2 ** 31), INVALID),
       (dict(K=0), INVALID), (dict(K=-16), INVALID), (dict(K=72), INVALID), (dict(K=131072), INVALID),
       (dict(out=2), INVALID), (dict(out=-1), INVALID), (dict(ws=ODD, ws_bytes=64), INVALID), (dict(ws_bytes=-1), INVALID),
       (dict(M=0, a=N, y=N), OK), (dict(N=0, b=N), OK)]


@pytest.mark.parametrize("change,rc", BAD)
def test_product(change, rc):
    lib = cabi.load()
    assert _call(lib.cek_gemm_int8_a8w8, GEMM, change) == rc
    glu = {k: v for kv in GEMM.items() for k, v in ([kv] if kv[0] != "out" else [("act", 0), kv])}
    assert _call(lib.cek_gemm_int8_a8w8_glu, glu, change) == rc
    for act in (-1, 2):
        assert _call(lib.cek_gemm_int8_a8w8_glu, glu, dict(act=act)) == INVALID


QUANT = dict(x=P, rows=2, H=64, io=0, q=P, scale=P, stream=N)
NORM = dict(hidden=P, residual=P, weight=P, rows=2, H=64, eps=1e-6, io=0, q=P, scale=P, stream=N)


@pytest.mark.parametrize("change,rc", [(dict(q=N), INVALID), (dict(scale=N), INVALID), (dict(rows=-1), INVALID),
                                       (dict(rows=2 ** 31), INVALID), (dict(H=0), INVALID), (dict(H=2 ** 30), INVALID),
                                       (dict(io=2), INVALID), (dict(rows=0, q=N), OK)])
def test_rows(change, rc):
    lib = cabi.load()
    assert _call(lib.cek_per_token_quant_int8, QUANT, change) == rc
    assert _call(lib.cek_fused_add_rms_norm_quant_int8, NORM, change) == rc
    assert _call(lib.cek_per_token_quant_int8, QUANT, dict(x=N)) == INVALID
    for n in ("hidden", "residual", "weight"):
        assert _call(lib.cek_fused_add_rms_norm_quant_int8, NORM, {n: N}) == INVALID


def test_workspace_sizes():
    """Nonsense needs none; what is asked for is bounded and 16-byte granular."""
    lib = cabi.load()
    for size in (lib.cek_gemm_int8_a8w8_workspace_size, lib.cek_gemm_int8_a8w8_glu_workspace_size):
        for bad in ((0, 8, 64), (-3, 8, 64), (8, 0, 64), (8, -1, 64), (8, 8, 0), (8, 8, 72), (8, 8, 131072), (2 ** 40, 8, 64)):
            assert size(*bad) == 0, bad
        for m in (1, 64, 65, 300, 512, 2048, 8192):
            for n, k in ((4096, 14336), (14336, 4096), (100, 131056)):
                assert 0 <= size(m, n, k) <= 2 ** 28 and size(m, n, k) % 16 == 0


def test_torch_ops():
    """Registered, with the written tensors marked, and loud about CPU tensors."""
    ops = esimd_learning_amd.ops()
    for name, written in (("esimd_per_token_quant_int8", 2), ("esimd_fused_add_rms_norm_quant_int8", 3),
                          ("esimd_gemm_int8_a8w8", 1), ("esimd_gemm_int8_a8w8_glu", 1)):
        schema = str(getattr(torch.ops.custom_esimd_kernels_vllm, name).default._schema)
        assert len({x.split("!")[0][-1] for x in schema.split("Tensor(")[1:]}) == written, schema
    x, q, s = torch.zeros(2, 64, dtype=torch.float16), torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2)
    y = torch.zeros(2, 2, dtype=torch.float16)
    for call in (lambda: ops.esimd_per_token_quant_int8(x, q, s),
                 lambda: ops.esimd_fused_add_rms_norm_quant_int8(x, x.clone(), x[0], 1e-6, q, s),
                 lambda: ops.esimd_gemm_int8_a8w8(q, s, q.clone(), s, y),
                 lambda: ops.esimd_gemm_int8_a8w8_glu(q, s, q.clone(), s, y[:, :1].contiguous())):
        with pytest.raises(NotImplementedError):
            call()
