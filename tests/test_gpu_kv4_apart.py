"""GPU: a row of the attention over the 4-bit cache beside others that are far larger or smaller, or not finite, and
before tokens that it must not see.  The batch and the tolerance are tests/test_gpu_kv4.py's; where nothing that a row
may see has changed, its bits have not."""

import math

import pytest
import torch

from oracle import kv4
from test_gpu_kv4 import EPS, Batch, _say

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 64), (8, 2, 128), (8, 2, 256), (4, 4, 128), (7, 1, 64)]
# hints: true ones, none (keys shared by the workgroups), and two that name the kernel for few and for many rows
HINTS = [dict(mq=45, mk=160), dict(mq=0, mk=0), dict(mq=1, mk=160), dict(mq=45, mk=5000), dict(mq=1, mk=5000)]
LENS, QLENS = [160, 45, 90, 7], [45, 45, 3, 1]


def _slots(b, r, first, n):
    t = torch.arange(first, first + n)
    return (b.host_tables[r].long()[t // b.bs] * b.bs + t % b.bs).to(b.tables.device)


def _store(b, ops, r, first, k=None, v=None):
    """Tokens first .. of request r take the rows k, v [n, nk, hd] (None: as they are)."""
    n = len(v if k is None else k)
    slots = _slots(b, r, first, n)
    old = [torch.empty(n, *b.heads[1:], dtype=b.dtype, device=b.tables.device) for _ in range(2)]
    keep = b.cache.clone()
    ops.esimd_kv4_cache_read(b.cache, slots, *old)
    new = [o if x is None else x.to(o) for o, x in zip(old, (k, v))]
    ops.esimd_kv4_cache_write(*new, b.cache, slots)
    nk, bs, hd = b.heads[1], b.bs, b.heads[2]
    for x, a, z, vals in ((k, 0, bs * hd // 2, b.keys), (v, bs * hd // 2, bs * hd, b.vals)):
        p = bs * hd + (0 if vals is b.keys else 4 * bs)
        if x is None:       # the bytes as they were
            now, was = b.cache.flatten(2), keep.flatten(2)
            now[..., a:z], now[..., p:p + 4 * bs] = was[..., a:z], was[..., p:p + 4 * bs]
            continue
        c, s, m = kv4.quantise(x)
        vals[r][first:first + n] = kv4.values(c, s, m)
        if vals is b.vals:
            b.spread[r][first:first + n] = 7.5 * s.double()[..., None]


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


@pytest.mark.parametrize("nq,nk,hd", HEADS)
@pytest.mark.parametrize("far", [1.0, 2.0 ** 20, 2.0 ** 60, -2.0 ** 90])
def test_tokens_behind_a_row_change_nothing(ops, dev, nq, nk, hd, far):
    """One token of a chunk with another key, and a value far larger: the rows before it keep their bits, the others are right."""
    _say("behind", nq, nk, hd, far)
    b = Batch(LENS, QLENS, nq, nk, hd, 16, torch.bfloat16, dev, seed=nq + hd)
    refs = [b.run(ops, **h) for h in HINTS]
    g = torch.Generator().manual_seed(1)
    # position 140 of request 0 is its row 25, position 30 of request 1 its row 30, 88 of request 2 its row 1
    for r, at in ((0, 140), (1, 30), (2, 88)):
        _store(b, ops, r, at, k=torch.randn(1, nk, hd, generator=g).bfloat16(),
               v=(torch.randn(1, nk, hd, generator=g) * far).bfloat16())
    for h, ref in zip(HINTS, refs):
        out = b.run(ops, **h)
        assert torch.equal(out[:25], ref[:25]), h
        assert torch.equal(out[45:75], ref[45:75]), h
        assert torch.equal(out[90], ref[90]) and torch.equal(out[93], ref[93]), h
        b.check(out)


@pytest.mark.parametrize("hints", HINTS)
@pytest.mark.parametrize("nq,nk,hd", HEADS)
@pytest.mark.parametrize("size", [2.0 ** 40, -2.0 ** 100, 2.0 ** -60, 0.0])
def test_values_without_spread(ops, dev, nq, nk, hd, hints, size):
    """V rows that are one value throughout (step 0), large and small."""
    _say("no spread", nq, nk, hd, hints, size)
    b = Batch(LENS, QLENS, nq, nk, hd, 16, torch.bfloat16, dev, seed=nq + hd)
    g = torch.Generator().manual_seed(2)
    for r, n in enumerate(LENS):
        _store(b, ops, r, 0, v=(torch.rand(n, nk, 1, generator=g) + 0.5).mul(size).expand(-1, -1, hd).bfloat16())
        assert (b.spread[r] == 0).all()
    b.check(b.run(ops, **hints))


@pytest.mark.parametrize("nq,nk,hd", HEADS)
@pytest.mark.parametrize("hints", HINTS)
def test_rows_of_all_sizes(ops, dev, nq, nk, hd, hints):
    """bf16 rows of a tile 2^130 apart, tokens and heads: each as if it were alone.  (Rows of 2^24 and more have one key
    left: what fp32 loses of a score of 2^26, some 2^4, is a 2^22th of the distance between two.)"""
    _say("sizes", nq, nk, hd, hints)
    b = Batch(LENS, QLENS, nq, nk, hd, 16, torch.bfloat16, dev, seed=nq + hd)
    size = torch.tensor([0, 40, -30, 100, 24, -3])
    t, h = torch.arange(b.cu[-1])[:, None], torch.arange(nq)[None]
    _set_q(b, (b.q.float() * torch.exp2(size[(t + 2 * h) % 6].float())[..., None]).bfloat16())
    b.check(b.run(ops, **hints))


@pytest.mark.parametrize("hints", HINTS)
@pytest.mark.parametrize("nq,nk,hd", HEADS)
def test_scores_far_below_zero(ops, dev, nq, nk, hd, hints):
    """q of 2^100 against the only key there is, its negative: the key's value, however small the score."""
    _say("far below", nq, nk, hd, hints)
    b = Batch([1, 1, 45], [1, 1, 45], nq, nk, hd, 16, torch.bfloat16, dev, seed=nq + hd)
    k = torch.ones(1, nk, hd).bfloat16()
    for r in (0, 1):
        _store(b, ops, r, 0, k=k)
    _store(b, ops, 2, 0, k=k.expand(45, -1, -1))
    _set_q(b, torch.full_like(b.q, -2.0 ** 100))
    b.check(b.run(ops, **hints))


def test_parts_whose_keys_are_all_nan(ops, dev):
    """Keys split over workgroups: NaN keys that fill a workgroup's share reach the rows like any others, whichever of
    the joins has them."""
    nq, nk, hd, n = 8, 8, 128, 20000
    for rows in (1, 70):
        _say("nan parts", rows)
        b = Batch([n], [rows], nq, nk, hd, 64, torch.float16, dev, seed=3)
        nan = torch.full((128, nk, hd), math.nan, dtype=torch.float16, device=dev)
        one = torch.ones_like(nan)
        for first in range(0, 6400, 128):
            ops.esimd_kv4_cache_write(nan, one, b.cache, _slots(b, 0, first, 128))
            for h in (dict(mq=rows), dict(mq=0, mk=0), dict(mq=1)):
                assert b.run(ops, **h).isnan().all(), (first, h)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 30, 1])
@pytest.mark.parametrize("nq,nk,hd", HEADS)
def test_windows_beyond_everything(ops, dev, nq, nk, hd, window):
    """Requests with fewer keys than new rows: the rows that have keys see them, up to the largest window there is."""
    _say("windows", nq, nk, hd, window)
    b = Batch([3, 40, 0, 1, 17], [10, 45, 4, 2, 17], nq, nk, hd, 16, torch.float16, dev, seed=nq + hd)
    for h in HINTS:
        out = b.run(ops, window=window, **h)
        b.check(out, window)
        assert (out[:7] == 0).all() and (out[55:60] == 0).all()
        if window > 40:
            assert torch.equal(out, b.run(ops, **h))


@pytest.mark.parametrize("hints", HINTS)
@pytest.mark.parametrize("nq,nk,hd", HEADS)
@pytest.mark.parametrize("far", [2.0 ** 14, 2.0 ** 24, 2.0 ** 80])
def test_large_values_of_no_weight(ops, dev, nq, nk, hd, far, hints):
    """Tokens with far larger values that a row sees, but hardly weighs: a weight times its step is rounded to 2^-34 of
    the largest weight times the largest step at worst, which is beside tests/test_gpu_kv4.py's bound

        n 2^-34 max_j p_j 2 max_j s_j 8

    of n keys (the power of two above a step is at most twice it, and a code at most 8 from the products' zero)."""
    _say("no weight", nq, nk, hd, far, hints)
    b = Batch(LENS, QLENS, nq, nk, hd, 16, torch.bfloat16, dev, seed=nq + hd)
    g = torch.Generator().manual_seed(3)
    _set_q(b, (torch.ones_like(b.q.float()) + 0.1 * b.q.float()).bfloat16())
    at = {0: (1, 60, 118), 1: (0, 20), 2: (50,), 3: (2,)}
    for r, tokens in at.items():
        for t in tokens:
            _store(b, ops, r, t, k=torch.full((1, nk, hd), -60 / hd ** 0.5).bfloat16(),
                   v=(torch.randn(1, nk, hd, generator=g) * far).bfloat16())
    out = b.run(ops, **hints).cpu().double()
    for r, n in enumerate(LENS):
        a, z = b.cu[r], b.cu[r + 1]
        one = torch.eye(n, dtype=torch.float64)[:, None].expand(-1, nk, -1)
        ref, (spread, size, p) = kv4.attention(b.q[a:z], b.keys[r], b.vals[r], b.scale, weigh=(b.spread[r], b.vals[r].abs(), one))
        step = b.spread[r].amax() / 7.5
        tol = EPS[b.dtype] / 2 * ref.abs() + 2.0 ** -11 * spread + 2.0 ** -13 * size
        tol = tol + n * 2.0 ** -34 * p.amax(-1, keepdim=True) * 2 * step * 8
        assert ((out[a:z] - ref).abs() <= tol).all(), f"request {r}: {float(((out[a:z] - ref).abs() / tol).max()):.3g} tolerances"
