"""GPU: calls of the attention over the 4-bit cache that its documentation allows and no model makes every day.  The batch
and the tolerance are tests/test_gpu_kv4.py's."""

import pytest
import torch

from oracle import kv4
from test_gpu_kv4 import Batch, _say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,nk,hd", [(128, 1, 128), (71, 1, 64), (96, 1, 256), (130, 2, 64)])
def test_many_heads_of_one(ops, dev, nq, nk, hd, dtype):
    """Single tokens with more heads a kv head than the kernel for few rows takes."""
    _say("heads", nq, nk, hd, dtype)
    b = Batch([1, 33, 700, 1500], [1, 1, 1, 1], nq, nk, hd, 16, dtype, dev, seed=nq)
    b.check(b.run(ops))
    b.check(b.run(ops, hints=False))


@pytest.mark.parametrize("mq,mk", [(1, 1), (1, 5000), (10 ** 6, 10 ** 9), (3, 0), (0, 16), (70, 100)])
@pytest.mark.parametrize("nq,nk,hd,window", [(8, 2, 128, 0), (4, 4, 64, 100), (16, 2, 256, 0)])
def test_wrong_hints(ops, dev, nq, nk, hd, window, mq, mk):
    _say("hints", nq, nk, hd, mq, mk)
    b = Batch([900, 60, 1300, 4], [50, 1, 7, 4], nq, nk, hd, 32, torch.float16, dev, seed=hd)
    b.check(b.run(ops, window=window, mq=mq, mk=mk), window)


@pytest.mark.parametrize("nq,nk,hd,chunk", [(8, 2, 64, 1), (4, 4, 128, 1), (8, 2, 64, 40), (2, 1, 256, 33)])
def test_many_requests(ops, dev, nq, nk, hd, chunk):
    """More requests than a wave has lanes, most of them short or empty, a few long; some with rows for the other kernel."""
    _say("requests", nq, nk, hd, chunk)
    lens = [(7 * i) % 50 for i in range(700)]
    qlens = [min(n, 1) for n in lens]
    for i, n in ((3, 2000), (64, 1500), (65, 900), (333, 3000), (699, 700)):
        lens[i], qlens[i] = n, chunk if i % 2 else 1
    b = Batch(lens, qlens, nq, nk, hd, 16, torch.bfloat16, dev, seed=chunk)
    b.check(b.run(ops))
    b.check(b.run(ops, hints=False))
    b.check(b.run(ops, window=30), 30)


@pytest.mark.parametrize("nq,nk,hd,rows", [(2, 2, 128, 1), (4, 2, 64, 1), (2, 1, 256, 1), (8, 2, 128, 20), (8, 1, 64, 20)])
def test_flat_weights_over_many_keys(ops, dev, nq, nk, hd, rows):
    """The mean of 40000 values is a two hundredth of each: what sums lose must be small against it, not against them.

    Of the outputs' norm: the output's rounding is at most 2^-11 of a value, uniformly distributed 2^-11 / sqrt(3); the
    weights' rounding the same, independently for each key, on values whose sum is what the output is made of: the
    root of both squares is 2^-11 sqrt(2 / 3) = 0.0004.  Half as much again is left for the sample."""
    _say("flat", nq, nk, hd, rows)
    b = Batch([40000], [rows], nq, nk, hd, 64, torch.float16, dev, seed=hd + rows)
    b.q = b.q * 0.01
    b.qd = b.q.to(dev)
    ref = kv4.attention(b.q, b.keys[0], b.vals[0], b.scale)
    for hints in (dict(mq=rows, mk=1), dict(mq=rows, mk=40000), dict(mq=0, mk=0)):
        err = b.run(ops, **hints).cpu().double() - ref
        assert float(err.norm() / ref.norm()) <= 6e-4, hints


def test_two_streams_at_once(ops, dev):
    """Calls of two batches in flight together, each on its stream, give what they give alone."""
    pair = [Batch([3000, 20, 5000], [1, 40, 2], 16, 4, 128, 32, torch.bfloat16, dev, seed=s) for s in (1, 2)]
    refs = [b.run(ops) for b in pair]
    for b, ref in zip(pair, refs):
        b.check(ref)
    streams = [torch.cuda.Stream() for _ in pair]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(pair[i].run(ops))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, refs[i]) for o in outs[i])


def test_tables_inside_a_larger_one_and_shared_blocks(ops, dev):
    """Rows of block_tables apart from each other; two requests that read the same blocks; one of them shorter."""
    b = Batch([200, 90], [1, 1], 8, 2, 128, 16, torch.float16, dev, seed=3)
    big = torch.full((2, b.width + 9), 10 ** 6, dtype=torch.int32, device=dev)
    big[:, 5:5 + b.width] = b.tables
    b.tables = big[:, 5:5 + b.width]
    b.check(b.run(ops))
    big[1] = big[0]
    b.keys[1], b.vals[1], b.spread[1] = (x[0][:90] for x in (b.keys, b.vals, b.spread))
    b.check(b.run(ops))


def test_write_read_and_tables_on_a_side_stream(ops, dev):
    hd, nk, bs = 128, 2, 16
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(40, nk, hd, generator=g).half().to(dev) for _ in range(2))
    res = []
    for side in (False, True):
        cache = torch.zeros(4, nk, bs, hd + 8, dtype=torch.uint8, device=dev)
        ring, state = ops.kv_free_ring(4, dev)
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
        lens, tables, cu, status = i32(1), i32(1, 4), i32(2), i32(1)
        slots, pos = (torch.zeros(40, dtype=torch.int64, device=dev) for _ in range(2))
        q = torch.full((1,), 37, dtype=torch.int32, device=dev)
        a, b = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
        s = torch.cuda.Stream() if side else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.esimd_kv_block_tables(lens, lens, q, bs, ring, state, tables, lens, state, cu, slots, pos, status)
            ops.esimd_kv4_cache_write(k, v, cache, slots)
            ops.esimd_kv4_cache_read(cache, slots, a, b)
        s.synchronize()
        assert slots.tolist() == list(range(37)) + [-1] * 3 and lens.tolist() == [37] and state.tolist() == [3, 1]
        assert (a[37:] == 0).all() and (b[37:] == 0).all()
        res.append((cache, a, b))
    for x, y in zip(*res):
        assert torch.equal(x, y)
