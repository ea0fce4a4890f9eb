"""CPU: what a layer of int8 weights holds for its rows."""

import pytest
import torch

from esimd_learning_amd import synthetic
from esimd_learning_amd.layer import GemmaDecodeLayer

DIMS = dict(hidden=128, n_q=4, n_kv=2, head_dim=32, mlp=272)


def _row_bytes(layer, M):
    return sum(t.nbytes for t in vars(layer).values() if isinstance(t, torch.Tensor) and t.shape[:1] == (M,)) // M


@pytest.mark.parametrize("fuse_glu", [True, False])
def test_only_buffers_that_a_step_touches(fuse_glu):
    M = 1009                                             # no weight has as many rows
    p = synthetic.gemma_layer(seed=10, fmt=torch.int8, **DIMS)
    layer = GemmaDecodeLayer(p, M, "cpu", fuse_glu=fuse_glu)
    hidden, heads, kv, mlp = 128, 128, 64, 272
    # 16 bits: qkv, attention, o, gated block, out (and both halves unfused); codes of norms, attention, block; a scale
    want = 2 * (heads + 2 * kv + heads + 2 * hidden + mlp + (0 if fuse_glu else 2 * mlp)) + hidden + heads + mlp + 4
    assert _row_bytes(layer, M) == want


def test_fp8_layers_keep_theirs():
    p = synthetic.gemma_layer(seed=10, **DIMS)
    layer = GemmaDecodeLayer(p, 3, "cpu")
    assert layer.gu.shape == (3, 544) and layer.r_mid.shape == (3, 128)
