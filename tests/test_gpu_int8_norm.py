"""GPU: add + RMS norm + int8 codes against 64 bits, within the bound of the kernels' own reductions.

u = 2^-24.  h + r is rounded once (2 u in its square).  A thread adds its squares one after another (`serial`
of them, one rounding each: up to four units of eight in the register kernels, H / 256 in the element kernel), a
wave's lanes add in 4 + 3 steps and up to sixteen waves in one each; none of the terms is negative, so the sum is off by
at most (2 + serial + 23) u.  The mean and the sum with eps round once each, the root halves all of this, and
rsqrt is within 2 u.  A value takes two products more (2 u), its scale a division (u).  Where the sum of squares passes fp32,
1 / rms may lie below fp32's normal range, down to 2^-128: 4 u more.
"""

import math

import pytest
import torch

from esimd_learning_amd import synthetic
from oracle import int8 as oint8

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _rel(h, far=False):
    serial = 32 if 8 <= h <= 32768 else math.ceil(h / 256)
    return ((2 + serial + 23 + 2) / 2 + 2 + 2 + 1 + (4 if far else 0)) * U


def _run(ops, dev, hid, res, w, eps):
    t, h = hid.shape
    r, q, s = res.to(dev), torch.full((t, h), 77, dtype=torch.int8, device=dev), torch.full((t,), -1.0, device=dev)
    ops.esimd_fused_add_rms_norm_quant_int8(hid.to(dev), r, w.to(dev), eps, q, s)
    return r.cpu(), q.cpu(), s.cpu()


def _check(got, hid, res, w, eps, rel):
    r, q, s = got
    kept, x = oint8.add_rms_norm(hid, res, w, eps)
    assert torch.equal(r, kept)
    want_s = oint8.quant(x)[1].double()
    off = (s.double() - want_s).abs() / want_s
    assert (off <= rel).all(), float(off.max() / U)
    assert ((q.double() - x / want_s[:, None]).abs() <= 0.5 + 127 * 2 * rel).all()


FAR = [(12, 8), (12, 40), (12, 264), (12, 1001), (12, 1031), (12, 2048), (12, 4096), (12, 6144), (12, 8195), (12, 16384), (12, 30001),
       (12, 7), (12, 32769), (1030, 1031), (1030, 4096), (1030, 4099), (1030, 6144), (1030, 8192)]


@pytest.mark.parametrize("t,h", FAR)
def test_rows_whose_squares_pass_fp32(ops, dev, t, h):
    """bf16 rows up to the type's largest values get the codes of the definition; beside them an ordinary row keeps its
    bits, and rows that are not finite, before or after the sum, their NaN scale."""
    g = synthetic.gen(t + h)
    hid, res = torch.randn(t, h, generator=g), torch.randn(t, h, generator=g)
    w = synthetic.norm_weight(h, 3, torch.bfloat16)
    most = torch.finfo(torch.bfloat16).max
    for i, scale in enumerate((1e16, 1e18, 3e19, 1e25, 1e30, 1e37)):
        hid[i] *= scale
        res[i] *= scale
    hid[6], res[6] = most, 0
    hid[7] = torch.where(torch.arange(h) % 3 == 0, most, -most)
    res[7] = -hid[7] / 2
    hid[9, h // 2] = math.inf
    hid[10], res[10] = most, most                     # finite, but their sum is not
    hid[11, -1] = most                                # one value far above its row
    hid, res = hid.bfloat16(), res.bfloat16()
    got = _run(ops, dev, hid, res, w, 1e-6)
    good = torch.tensor([i for i in range(t) if i not in (9, 10)])
    _check([x[good] for x in got], hid[good], res[good], w, 1e-6, _rel(h, far=True))
    assert torch.isnan(got[2][9:11]).all() and (got[1][9:11] == 0).all()
    if t == 12:
        alone = _run(ops, dev, hid[8:9], res[8:9], w, 1e-6)
        assert all(torch.equal(x[8:9], y) for x, y in zip(got, alone))


FORMS = [(4, 1), (4, 7), (5, 8), (5, 9), (6, 15), (7, 64), (4, 136), (9, 505), (5, 520), (6, 1000), (5, 1031), (4, 2048), (3, 2056), (4, 4093),
         (5, 4096), (4, 4099), (3, 5120), (4, 8192), (3, 8195), (4, 16384), (3, 16390), (4, 30001), (3, 32768), (3, 32769), (3, 40000),
         (1025, 1001), (1026, 4096), (1025, 4099), (1027, 5121), (1024, 6144), (1025, 8185)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,h", FORMS)
def test_within_the_reduction(ops, dev, t, h, dtype):
    """Ordinary rows; one whose sums all round down, so that a mean of the rounded residual is off; one whose last eight
    values, the last unit of an odd length, outweigh the rest, so that a value counted twice shows."""
    g = synthetic.gen(t + h)
    hid, res = torch.randn(t, h, generator=g), torch.randn(t, h, generator=g)
    hid[:, 3 % h::17] *= 20
    step, sign = torch.finfo(dtype).eps, torch.randint(0, 2, (h,), generator=g) * 2.0 - 1
    res[1 % t] = sign * (1 + step * torch.randint(0, int(1 / step), (h,), generator=g))
    hid[1 % t] = sign * step * 0.375
    hid[2 % t, -8:] *= 30
    hid, res, w = hid.to(dtype), res.to(dtype), synthetic.norm_weight(h, 3, dtype)
    _check(_run(ops, dev, hid, res, w, 1e-6), hid, res, w, 1e-6, _rel(h))
