"""CPU: the synthetic int8 weights are what the quantisation operator makes of the same rows."""

import math

import pytest
import torch

from esimd_learning_amd import synthetic
from oracle import int8 as oint8


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rows_as_the_operator_has_them(dtype):
    W = (torch.randn(9, 300, generator=synthetic.gen(1)) * 0.02).to(dtype)
    W[1] = 0
    W[2] = 0
    W[2, 7] = torch.finfo(dtype).smallest_normal
    W[3] = torch.arange(300) % 127 + 0.5
    W[3, 0] = 127                                        # scale 1: every other value a tie
    W[4, 5], W[5, 6], W[6, 7] = math.inf, -math.inf, math.nan
    q, s = synthetic.quantize_rows(W, torch.int8)
    want_q, want_s = oint8.quant(W)
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    assert torch.equal(q, want_q) and torch.equal(torch.isnan(s), torch.isnan(want_s))
    assert torch.equal(s[~torch.isnan(s)], want_s[~torch.isnan(s)]) and torch.isnan(s).tolist() == [False] * 4 + [True] * 3 + [False] * 2
    assert s[1] == 2.0 ** -126 and (q[1] == 0).all()


def test_layer_weights():
    """Ordinary weights: the nearest integers of the quotient by the row's scale."""
    p = synthetic.gemma_layer(seed=10, hidden=128, n_q=2, n_kv=1, head_dim=32, mlp=256, fmt=torch.int8)
    for w, s in (("Wqkv", "sqkv"), ("Wo", "so"), ("Wgu", "sgu"), ("Wd", "sd")):
        assert p[w].dtype == torch.int8 and p[s].dtype == torch.float32 and (p[w].abs().amax(1) == 127).all()
