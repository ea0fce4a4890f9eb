"""GPU: scales that are not finite, of a token and of a channel, in every kind of kernel of the int8 products."""

import math

import pytest
import torch

from esimd_learning_amd import synthetic
from oracle import int8 as oint8

pytestmark = pytest.mark.gpu

# v_dot4, rings of each height, a tile, a split tile
SIZES = [(1, 64, 192), (3, 64, 192), (8, 64, 192), (16, 70, 1040), (30, 64, 192), (40, 66, 592), (64, 64, 192), (140, 64, 192), (66, 70, 4112)]


@pytest.mark.parametrize("act", [None, "silu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_scales_that_are_not_finite(ops, dev, m, n, k, act):
    """Rows and columns of an infinite or NaN scale hold what fp32 gives for them; all others keep their bits."""
    g = synthetic.gen(m + n + k)
    a, b = (torch.randint(-127, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, n))
    sa, sb = torch.rand(m, generator=g) * 0.02 + 1e-3, torch.rand(n, generator=g) * 1e-4 + 1e-6
    a[m // 2, ::2] = 0
    b[5] = 0                                             # sums of zero, times infinity

    def run(sa, sb):
        y = torch.zeros(m, n // (2 if act else 1), dtype=torch.float16, device=dev)
        args = [t.to(dev) for t in (a, sa, b, sb)] + [y]
        ops.esimd_gemm_int8_a8w8_glu(*args, act) if act else ops.esimd_gemm_int8_a8w8(*args)
        return y.cpu()

    clean = run(sa, sb)
    for where, bad in ((m // 2, math.inf), (m - 1, math.nan)):
        s = sa.clone()
        s[where] = bad
        got, rest = run(s, sb), torch.arange(m) != where
        assert torch.equal(got[rest], clean[rest])
        if act is None:
            want = oint8.product(a, s, b, sb, torch.float16)
            assert ((got == want) | (torch.isnan(got) & torch.isnan(want))).all()
            assert torch.isnan(got[where, 5])            # 0 * inf, or the NaN
        elif math.isnan(bad):
            assert torch.isnan(got[where]).all()
    half = n // 2
    for where, bad in ((7, math.inf), (n - 2, math.nan), (5, math.inf)):
        s = sb.clone()
        s[where] = bad
        got, col = run(sa, s), where % half if act else where
        rest = torch.arange(got.shape[1]) != col
        assert torch.equal(got[:, rest], clean[:, rest])
        if act is None:
            want = oint8.product(a, sa, b, s, torch.float16)
            assert ((got == want) | (torch.isnan(got) & torch.isnan(want))).all()
        if math.isnan(bad) or where == 5:
            assert torch.isnan(got[:, col]).all()
