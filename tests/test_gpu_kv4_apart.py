"""GPU: a row of the attention over the 4-bit cache beside others that are far larger or smaller, or not finite.  The
batch and the tolerance are tests/test_gpu_kv4.py's; where nothing that a row may see has changed, its bits have not."""

import math

import pytest
import torch

from test_gpu_kv4 import Batch, _say

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 64), (8, 2, 128), (8, 2, 256), (4, 4, 128), (7, 1, 64)]
# hints: true ones, none (keys shared by the workgroups), and two that name the kernel for few and for many rows
HINTS = [dict(mq=45, mk=160), dict(mq=0, mk=0), dict(mq=1, mk=160), dict(mq=45, mk=5000), dict(mq=1, mk=5000)]
LENS, QLENS = [160, 45, 90, 7], [45, 45, 3, 1]


def _set_q(b, q):
    b.q = q
    b.qd = q.to(b.tables.device)


@pytest.mark.parametrize("nq,nk,hd", HEADS)
@pytest.mark.parametrize("far", [2.0 ** 12, -2.0 ** 40, 2.0 ** 100])
def test_far_larger_rows(ops, dev, nq, nk, hd, far):
    """Heads and tokens of a tile times 2^12 .. 2^100: every other row's bits stay."""
    _say("far larger", nq, nk, hd, far)
    b = Batch(LENS, QLENS, nq, nk, hd, 16, torch.bfloat16, dev, seed=nq + hd)
    refs = [b.run(ops, **h) for h in HINTS]
    for out in refs:
        b.check(out)
    t, h = torch.arange(b.cu[-1])[:, None], torch.arange(nq)[None]
    large = (t + 2 * h) % 5 == 1
    _set_q(b, torch.where(large[..., None], b.q.float() * far, b.q.float()).bfloat16())
    for h, ref in zip(HINTS, refs):
        same = (b.run(ops, **h) == ref).all(-1).cpu()
        assert same[~large].all(), (h, (~same & ~large).nonzero()[:8].tolist())


@pytest.mark.parametrize("nq,nk,hd", HEADS)
@pytest.mark.parametrize("hints", HINTS)
def test_rows_of_many_sizes(ops, dev, nq, nk, hd, hints):
    """bf16 rows of a tile up to 2^60 apart: each as if it were alone."""
    _say("many sizes", nq, nk, hd, hints)
    b = Batch(LENS, QLENS, nq, nk, hd, 16, torch.bfloat16, dev, seed=nq + hd)
    size = torch.tensor([0, 3, -30, -60, -12, 1])
    t, h = torch.arange(b.cu[-1])[:, None], torch.arange(nq)[None]
    _set_q(b, (b.q.float() * torch.exp2(size[(t + 2 * h) % 6].float())[..., None]).bfloat16())
    b.check(b.run(ops, **hints))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,nk,hd", HEADS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_one_row_that_is_not_finite(ops, dev, nq, nk, hd, bad, dtype):
    """One element of one head of a token: every other row's bits stay."""
    _say("not finite", nq, nk, hd, bad, dtype)
    for window in (0, 50):
        b = Batch(LENS, QLENS, nq, nk, hd, 16, dtype, dev, seed=nq + hd)
        refs = [b.run(ops, window=window, **h) for h in HINTS]
        for out in refs:
            b.check(out, window)
        spoilt = [(20, 1), (44, 0), (50, nq - 1), (91, 2), (93, 0)]
        q = b.q.clone()
        for t, h in spoilt:
            q[t, h, 5] = bad
        _set_q(b, q)
        for h, ref in zip(HINTS, refs):
            out = b.run(ops, window=window, **h)
            same = (out == ref).all(-1).cpu()
            same[tuple(zip(*spoilt))] = True
            assert same.all(), (h, (~same).nonzero()[:8].tolist())
