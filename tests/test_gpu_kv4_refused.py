"""GPU: requests that get no room in a step -- at their longest, or with the free blocks gone -- beside requests that do.
The others' rows, outputs and cached bytes are what they are where nobody is refused, bit for bit: their keys are short
enough to stay whole, so that a row's sums do not depend on the batch."""

import sys

import pytest
import torch

from esimd_learning_amd import synthetic
from esimd_learning_amd.kv4 import KV4Cache
from esimd_learning_amd.layer import GemmaDecodeLayer, capture_forward, forward

pytestmark = pytest.mark.gpu

DIMS = dict(hidden=512, n_q=4, n_kv=2, head_dim=64, mlp=1024)
M = 8
# new tokens of four requests with five blocks of 16 between them and 32 tokens each at most: the first one is refused
# for its length from step 6 on, the second one for a block from step 9 on and the third one from step 11 on
STEPS = [[5, 1, 0, 1], [6, 0, 2, 0], [6, 1, 0, 1], [7, 0, 1, 0], [6, 1, 1, 0]] + [[2, 3, 2, 1]] * 7
REFUSED = {0: {6, 7, 8, 9, 10, 11}, 1: {9, 10, 11}, 2: {11}, 3: set()}


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _inputs(step, dev):
    return (synthetic.activations(M, DIMS["hidden"], seed=400 + step).to(dev),
            synthetic.activations(M, DIMS["hidden"], seed=500 + step).to(dev))


def _roomy(stack, dev, refused):
    """What each step's rows give where there is room for all: steps in which a request was refused bring it no token."""
    kv, res = KV4Cache(2, 40, 2, 64, 4, M, max_len=200, block_size=16, device=dev), []
    for i, q in enumerate(STEPS):
        h, r = _inputs(i, dev)
        real = [0 if i in refused[j] else n for j, n in enumerate(q)]
        # the granted requests' rows, closed up
        at, rows = 0, []
        for n, m in zip(q, real):
            rows += list(range(at, at + m))
            at += n
        rows = torch.tensor(rows + [M - 1] * (M - len(rows)), device=dev)
        h, r = h[rows].contiguous(), r[rows].contiguous()
        kv.advance(_i32(real, dev), None, M, 100)
        out = forward(stack, h, r, kv.positions, kv)
        assert kv.status.tolist() == [0] * 4
        res.append((rows[: sum(real)], out[: sum(real)].clone(), r[: sum(real)].clone()))
    return kv, res


def _compare(kv, steps, stack, dev):
    far, ref = _roomy(stack, dev, REFUSED)
    for i, (status, out, r) in enumerate(steps):
        assert [s != 0 for s in status] == [i in REFUSED[j] for j in range(4)], (i, status)
        rows, o, rr = ref[i]
        assert torch.equal(out[rows], o), f"step {i}"
        assert torch.equal(r[rows], rr), f"step {i}"
    assert kv.lens.tolist() == far.lens.tolist()
    for j, n in enumerate(kv.lens.tolist()):
        for a, b in zip(kv.layers, far.layers):
            for x, y in zip(a.read(kv.slots(j, 0, n)), b.read(far.slots(j, 0, n))):
                assert torch.equal(x, y), f"request {j}"


def _stack(dev):
    return [GemmaDecodeLayer(synthetic.gemma_layer(seed=70 + i, **DIMS), M, dev) for i in range(2)]


def test_captured_steps_with_refused_requests(ops, dev):
    """The caller lays its rows out by q_lens before each replay: a refused request's rows shift no one else's."""
    stack = _stack(dev)
    kv = KV4Cache(2, 5, 2, 64, 4, M, max_len=32, block_size=16, device=dev)
    q, (h, r) = _i32([0] * 4, dev), _inputs(0, dev)
    g = capture_forward(stack, h, r, kv.positions, kv=kv, q_lens=q, max_q_len=M, max_kv_len=100)
    steps = []
    for i, n in enumerate(STEPS):
        print("step", i, n, flush=True)
        sys.stdout.flush()
        q.copy_(_i32(n, dev))
        for to, x in zip((h, r), _inputs(i, dev)):
            to.copy_(x)
        g.replay()
        steps.append((kv.status.tolist(), stack[-1].out.clone(), r.clone()))
    _compare(kv, steps, stack, dev)


def test_eager_steps_with_refused_requests(ops, dev):
    """The same without a graph, status never read before a step's rows are laid out."""
    stack = _stack(dev)
    kv = KV4Cache(2, 5, 2, 64, 4, M, max_len=32, block_size=16, device=dev)
    steps = []
    for i, n in enumerate(STEPS):
        h, r = _inputs(i, dev)
        kv.advance(_i32(n, dev), None, M, 100, fixed_rows=True)
        out = forward(stack, h, r, kv.positions, kv).clone()
        steps.append((kv.status.tolist(), out, r))
    _compare(kv, steps, stack, dev)
