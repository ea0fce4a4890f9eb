"""GPU: long keys dealt out over all workgroups -- tiles that begin, continue and end in the middle of a workgroup's
share, shares of the different layers, requests that hold little beside others that hold much.  The batch and the
tolerance are tests/test_gpu_kv4.py's."""

import pytest
import torch

from test_gpu_kv4 import Batch, _say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,nk,hd,lens,qlens,window", [
    (32, 32, 128, [4000, 700, 9000, 1], [1, 1, 1, 1], 0),
    (20, 20, 128, [7001, 13000], [3, 1], 0),                    # 256 workgroups are no whole number a head
    (16, 16, 64, [20000, 15000], [1, 1], 0),
    (16, 16, 256, [6000, 9000, 2], [1, 5, 2], 0),
    (64, 32, 128, [9000, 0, 8000], [8, 0, 9], 0),               # tiles of 32 rows
    (16, 16, 256, [9000, 9000, 9000], [1, 2, 1], 7000),
    (32, 32, 128, [300] * 40 + [5000], [1] * 41, 0),
])
def test_shares(ops, dev, nq, nk, hd, lens, qlens, window, dtype):
    _say("shares", nq, nk, hd, len(lens), window, dtype)
    b = Batch(lens, qlens, nq, nk, hd, 64, dtype, dev, seed=nq + hd)
    out = b.run(ops, window=window)
    b.check(out, window)
    assert torch.equal(b.run(ops, window=window), out)
    b.check(b.run(ops, window=window, hints=False), window)
