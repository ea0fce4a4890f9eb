"""GPU: the 4-bit key/value cache -- writes, reads and attention against the fp64 oracle.

Tolerances are bounds, not fits.  Cache writes follow the format's definition one
rounding at a time, so the bytes are equal.  Reads: one fp32 and one output
rounding.  Attention, per output element,

    eps_out / 2 |out|  +  2^-11 sum_j p_j 7.5 s_j  +  2^-13 sum_j p_j |v_j|

the output's rounding; the weights p_j times the V step s_j, which the kernels may
round once to fp16 (half a step, 2^-12 of the value, and twice that allows for
weights in fp16's subnormal range), against codes at most 7.5 from the centre; and
what fp32 leaves of the scores: an exponent |x| <= 64 is off by at most a few
2^-24 |x| after its product, its centre term and its scaling, 2^-15 in all, and a
weight by as much, once in the numerator and once in the denominator.
"""

import math
import sys

import pytest
import torch

from oracle import kv4

pytestmark = pytest.mark.gpu

EPS = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def _say(*what):
    print(*what, flush=True)
    sys.stdout.flush()


def _rand(*shape, seed, dtype, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _same_bytes(cache, ref):
    """Equal bytes, or which differ."""
    at = (cache.cpu() != ref).flatten(2).nonzero()
    if len(at):
        a, b = cache.cpu().flatten(2), ref.flatten(2)
        what = [(i, int(a[tuple(i)]), int(b[tuple(i)])) for i in at[:6].tolist()]
        pytest.fail(f"{len(at)} bytes of (block, head, byte) differ: {what}")


# ---- write and read -----------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd,nk,bs,T", [(64, 1, 16, 1), (64, 3, 16, 37), (128, 8, 32, 5), (128, 2, 64, 70),
                                        (256, 16, 16, 2), (256, 1, 256, 33)])
def test_write_bytes_equal_the_definition(ops, dev, dtype, hd, nk, bs, T):
    _say("write", dtype, hd, nk, bs, T)
    blocks = T // bs + 4
    g = torch.Generator().manual_seed(T)
    slots = torch.randperm(blocks * bs, generator=g)[:T]
    if T > 8:
        slots[:8] = torch.arange(8) + bs - 4         # a run over a block's end, tokens 4-aligned in part
        rest = torch.randperm((blocks - 2) * bs, generator=g)[:T - 8] + 2 * bs
        slots[8:] = rest
        slots[T // 2] = -1                           # padding in the middle
        slots[T - 1] = blocks * bs                   # one past the cache
    k, v = _rand(T, nk, hd, seed=1, dtype=dtype), _rand(T, nk, hd, seed=2, dtype=dtype, scale=0.01)
    if T > 4:
        k[1, 0] = 2.5                                # a row without spread
        v[2, 0, 3] = math.inf
        k[3, 0, hd - 1] = math.nan
        v[4, 0] = v[4, 0] + 100
    ref = kv4.empty(blocks, nk, bs, hd)
    for t in range(T):
        if 0 <= slots[t] < blocks * bs:
            kv4.put(ref, int(slots[t]), k[t], v[t])
    cache = kv4.empty(blocks, nk, bs, hd).to(dev)
    ops.esimd_kv4_cache_write(k.to(dev), v.to(dev), cache, slots.to(dev))
    torch.cuda.synchronize()
    _same_bytes(cache, ref)


def test_write_extreme_rows(ops, dev):
    """Spreads from bf16's largest to its subnormals."""
    hd, nk, bs = 128, 1, 16
    rows = []
    for e in (-133, -126, -101, -100, -99, -96, -60, 0, 60, 100, 126):
        x = torch.randn(hd, generator=torch.Generator().manual_seed(e + 200)).clamp(-1, 1)
        rows.append((x * 2.0 ** min(e, 100) * 2.0 ** max(0, e - 100)).bfloat16())
    rows.append(torch.tensor([3.38e38, -3.38e38] * 64).bfloat16())
    k = torch.stack(rows)[:, None]
    T = k.shape[0]
    ref = kv4.empty(2, nk, bs, hd)
    for t in range(T):
        kv4.put(ref, t, k[t], -k[t])
    cache = kv4.empty(2, nk, bs, hd).to(dev)
    ops.esimd_kv4_cache_write(k.to(dev), -k.to(dev), cache, torch.arange(T, device=dev))
    _same_bytes(cache, ref)


@pytest.mark.parametrize("flat", [False, True])
def test_write_from_projection_columns(ops, dev, flat):
    """k and v as column views of a fused projection, also with rows that are not 16-byte aligned."""
    nk, hd, bs, T = 2, 128, 16, 21
    for extra in (0, 3):
        qkv = _rand(T, 6 * hd + extra, seed=5, dtype=torch.bfloat16)
        k, v = qkv[:, 2 * hd:4 * hd], qkv[:, 4 * hd:6 * hd]
        if not flat:
            k, v = k.unflatten(1, (nk, hd)), v.unflatten(1, (nk, hd))
        d = qkv.to(dev)
        kd, vd = d[:, 2 * hd:4 * hd], d[:, 4 * hd:6 * hd]
        if not flat:
            kd, vd = kd.unflatten(1, (nk, hd)), vd.unflatten(1, (nk, hd))
        a, b = (kv4.empty(4, nk, bs, hd, fill=7).to(dev) for _ in range(2))
        slots = torch.arange(T, device=dev) + 3
        ops.esimd_kv4_cache_write(kd, vd, a, slots)
        ops.esimd_kv4_cache_write(k.contiguous().to(dev), v.contiguous().to(dev), b, slots)
        assert torch.equal(a, b) and not torch.equal(a, torch.full_like(a, 7))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd,nk,bs,T", [(64, 2, 16, 1), (64, 4, 16, 50), (128, 8, 32, 9), (256, 3, 256, 301)])
def test_read(ops, dev, dtype, hd, nk, bs, T):
    _say("read", dtype, hd, nk, bs, T)
    g = torch.Generator().manual_seed(hd)
    blocks = 5
    cache = torch.randint(0, 256, (blocks, nk, bs, hd + 8), generator=g, dtype=torch.uint8)
    par = cache.view(blocks, nk, -1)[..., bs * hd:].view(torch.bfloat16)   # finite parameters
    par.copy_(torch.randn(par.shape, generator=g).bfloat16())
    slots = torch.randint(-2, blocks * bs + 2, (T,), generator=g)
    slots[: min(T, 9)] = torch.arange(min(T, 9)) + bs - 3
    k, v = (torch.full((T, nk, hd), 7.0, dtype=dtype, device=dev) for _ in range(2))
    ops.esimd_kv4_cache_read(cache.to(dev), slots.to(dev), k, v)
    for t in range(T):
        in_cache = 0 <= slots[t] < blocks * bs
        for got, ref in zip((k[t], v[t]), kv4.get(cache, int(slots[t])) if in_cache else (torch.zeros(nk, hd),) * 2):
            ref = ref.double()
            # values are one fp32 rounding off, which may carry a 16-bit rounding over its half
            tol = ref.abs() * (EPS[dtype] / 2 + 2.0 ** -23) + TINY[dtype]
            assert ((got.cpu().double() - ref).abs() <= tol).all()


def test_read_into_strided_rows_leaves_the_rest(ops, dev):
    hd, nk, bs, T = 128, 2, 16, 6
    cache = kv4.empty(1, nk, bs, hd, fill=0)
    for t in range(T):
        kv4.put(cache, t, _rand(nk, hd, seed=t, dtype=torch.float16), _rand(nk, hd, seed=50 + t, dtype=torch.float16))
    for pad in (8, 5):
        buf = torch.full((T, 2 * nk * hd + pad), 9.0, dtype=torch.float16, device=dev)
        k, v = buf[:, :nk * hd], buf[:, nk * hd:2 * nk * hd]
        ops.esimd_kv4_cache_read(cache.to(dev), torch.arange(T, device=dev), k, v)
        a, b = (torch.empty(T, nk, hd, dtype=torch.float16, device=dev) for _ in range(2))
        ops.esimd_kv4_cache_read(cache.to(dev), torch.arange(T, device=dev), a, b)
        assert torch.equal(k, a.flatten(1)) and torch.equal(v, b.flatten(1))
        assert (buf[:, 2 * nk * hd:] == 9).all()


# ---- attention ------------------------------------------------------------------

class Batch:
    """Requests with cached keys and values: a cache on the GPU whose unused bytes are NaN parameters, and the fp64
    values of the used ones."""

    def __init__(self, lens, qlens, nq, nk, hd, bs, dtype, dev, seed=0, spare=3, width=None, kscale=1.0, vscale=1.0,
                 vmean=0.0, block_gap=0):
        self.lens, self.qlens, self.dtype, self.bs, self.heads = lens, qlens, dtype, bs, (nq, nk, hd)
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // bs) for n in lens]
        blocks = sum(need) + spare
        order = torch.randperm(blocks, generator=g).tolist()
        self.width = width or max(need + [1]) + 1
        tables = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        host = kv4.empty(blocks, nk, bs, hd)
        flat = host.view(blocks, nk, -1)
        self.keys, self.vals, self.spread = [], [], []
        at = 0
        for r, n in enumerate(lens):
            mine = order[at:at + need[r]]
            at += need[r]
            tables[r, :need[r]] = torch.tensor(mine, dtype=torch.int32)
            k = (torch.randn(n, nk, hd, generator=g) * kscale).to(dtype)
            v = (torch.randn(n, nk, hd, generator=g) * vscale + vmean).to(dtype)
            got = []
            for part, x in ((0, k), (1, v)):
                c, s, m = kv4.quantise(x)
                got.append((c, s, m))
                by = c[..., 0::2] | (c[..., 1::2] << 4)
                par = torch.stack([s, m], -1).bfloat16().view(torch.uint8)     # [n, nk, 4]
                for i, b in enumerate(mine):
                    t0, t1 = i * bs, min(n, i * bs + bs)
                    to = flat[b, :, bs * hd + part * 4 * bs:bs * hd + part * 4 * bs + 4 * bs].view(nk, bs, 4)
                    to[:, :t1 - t0] = par[t0:t1].transpose(0, 1)
                    rows = by[t0:t1].transpose(0, 1)
                    if part == 0:
                        flat[b, :, :bs * hd // 2].view(nk, bs, hd // 2)[:, :t1 - t0] = rows
                    else:
                        w = flat[b, :, bs * hd // 2:bs * hd].view(nk, bs // 4, hd // 4, 4, 2)
                        full = torch.full((nk, bs, hd // 2), 0xFF, dtype=torch.uint8)
                        full[:, :t1 - t0] = rows
                        w.copy_(full.view(nk, bs // 4, 4, hd // 4, 2).transpose(2, 3))
            self.keys.append(kv4.values(*got[0]))
            self.vals.append(kv4.values(*got[1]))
            self.spread.append(7.5 * got[1][1].double()[..., None])
        if block_gap:
            buf = torch.full((blocks, flat.shape[-1] * nk + block_gap), 0xFF, dtype=torch.uint8, device=dev)
            self.cache = buf.as_strided((blocks, nk, bs, hd + 8), (buf.shape[1], bs * (hd + 8), hd + 8, 1))
            self.cache.copy_(host)
        else:
            self.cache = host.to(dev)
        self.host_tables = tables
        self.tables = tables.to(dev)
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        cu = [0]
        for n in qlens:
            cu.append(cu[-1] + n)
        self.cu = cu
        self.cu_q = torch.tensor(cu, dtype=torch.int32, device=dev)
        self.q = _rand(cu[-1], nq, hd, seed=seed + 1, dtype=dtype, scale=2.0)
        self.qd = self.q.to(dev)
        self.scale = hd ** -0.5

    def run(self, ops, q=None, out=None, window=0, hints=True, **kw):
        q = self.qd if q is None else q
        out = torch.full_like(q, 7.0) if out is None else out
        mq, mk = (max(self.qlens + [0]), max(self.lens + [0])) if hints else (0, 0)
        ops.esimd_kv4_attention(q, self.cache, self.tables, self.kv_lens, self.cu_q, out, kw.get("scale", self.scale),
                                kw.get("mq", mq), kw.get("mk", mk), window)
        return out

    def check(self, out, window=0, scale=None):
        out = out.detach().cpu().double().view(-1, *self.heads[::2])
        eps = EPS[self.dtype]
        for r, n in enumerate(self.lens):
            a, b = self.cu[r], self.cu[r + 1]
            if a == b:
                continue
            ref, (spread, size) = kv4.attention(self.q[a:b], self.keys[r], self.vals[r], scale or self.scale, window,
                                                weigh=(self.spread[r], self.vals[r].abs()))
            tol = eps / 2 * ref.abs() + 2.0 ** -11 * spread + 2.0 ** -13 * size + TINY[self.dtype]
            bad = (out[a:b] - ref).abs() > tol
            assert torch.isfinite(out[a:b]).all(), f"request {r}: not finite"
            assert not bad.any(), (f"request {r} of {n} keys, {b - a} rows: {int(bad.sum())} elements, worst "
                                   f"{float(((out[a:b] - ref).abs() / tol).max()):.3g} tolerances")


HEADS = [(1, 1, 64), (8, 8, 64), (16, 4, 64), (8, 8, 128), (32, 8, 128), (28, 1, 128), (4, 4, 256), (16, 2, 256)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("nq,nk,hd", HEADS)
def test_decode(ops, dev, nq, nk, hd, bs, dtype):
    """One token a request: no key, one, and lengths around every tile's end."""
    _say("decode", nq, nk, hd, bs, dtype)
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 1021]
    b = Batch(lens, [1] * len(lens), nq, nk, hd, bs, dtype, dev, seed=hd + nq)
    out = b.run(ops)
    b.check(out)
    assert (out[0] == 0).all()
    b.check(b.run(ops, hints=False))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,nk,hd,lens", [(32, 8, 128, [5000]), (2, 1, 64, [9001]), (4, 4, 256, [4097, 3, 2500]),
                                           (32, 32, 128, [2049, 1000])])
def test_decode_long(ops, dev, nq, nk, hd, lens, dtype):
    _say("decode long", nq, nk, hd, lens, dtype)
    b = Batch(lens, [1] * len(lens), nq, nk, hd, 32, dtype, dev, seed=7)
    b.check(b.run(ops))


@pytest.mark.parametrize("window", [0, 1, 37, 128])
@pytest.mark.parametrize("nq,nk,hd", [(8, 8, 128), (16, 2, 64), (4, 1, 256), (28, 4, 128)])
def test_few_rows(ops, dev, nq, nk, hd, window):
    """Drafted tokens: a few rows a request, none for some, windows that end inside tiles."""
    _say("few rows", nq, nk, hd, window)
    lens, ql = [5, 40, 33, 0, 130, 257, 600], [5, 3, 0, 0, 8, 2, 7]
    b = Batch(lens, ql, nq, nk, hd, 16, torch.bfloat16, dev, seed=window + nq)
    b.check(b.run(ops, window=window), window)
    b.check(b.run(ops, window=window, mq=0, mk=1), window)   # a wrong hint: the same results


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("nq,nk,hd,lens,ql", [
    (8, 2, 128, [129, 300], [129, 77]), (4, 4, 64, [65, 513, 200], [65, 1, 200]), (2, 1, 256, [333], [333]),
    (32, 8, 128, [70, 1, 90], [33, 1, 90]), (7, 1, 128, [200, 31], [150, 31])])
def test_prompt_chunks(ops, dev, nq, nk, hd, lens, ql, window, dtype):
    _say("chunks", nq, nk, hd, lens, ql, window, dtype)
    b = Batch(lens, ql, nq, nk, hd, 32, dtype, dev, seed=sum(lens))
    b.check(b.run(ops, window=window), window)


@pytest.mark.parametrize("window", [0, 300])
def test_mixed_batch(ops, dev, window):
    """Decodes, drafts and prompt chunks in one call, with and without the lengths known."""
    lens, ql = [1500, 7, 400, 2100, 64, 0, 900], [1, 7, 260, 1, 5, 0, 1]
    b = Batch(lens, ql, 8, 2, 64, 16, torch.float16, dev, seed=11)
    for hints in (True, False):
        b.check(b.run(ops, window=window, hints=hints), window)


def test_chunk_on_a_long_prefix(ops, dev):
    b = Batch([6100], [70], 4, 1, 128, 64, torch.bfloat16, dev, seed=12)
    b.check(b.run(ops))


def test_rows_outside_the_sequences_stay(ops, dev):
    """Rows before cu_q[0] and behind cu_q[R], and a request without rows between others."""
    b = Batch([20, 50, 9], [2, 0, 1], 8, 2, 128, 16, torch.bfloat16, dev, seed=13)
    pad = torch.cat([b.qd[:1], b.qd, b.qd[:2]])
    out = torch.full_like(pad, 7.0)
    ops.esimd_kv4_attention(pad, b.cache, b.tables, b.kv_lens, b.cu_q + 1, out, b.scale)
    b.check(out[1:4])
    assert (out[0] == 7).all() and (out[4:] == 7).all()


def test_rows_without_positions_are_zero(ops, dev):
    """More new rows than cached tokens: the rows before the first key are zero, the others as usual."""
    b = Batch([2], [2], 4, 4, 64, 16, torch.float16, dev, seed=14)
    q = torch.cat([b.qd, b.qd])
    out = torch.full_like(q, 7.0)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    ops.esimd_kv4_attention(q, b.cache, b.tables, b.kv_lens, cu, out, b.scale)
    assert (out[:2] == 0).all()
    b.check(out[2:])


@pytest.mark.parametrize("nq,nk,hd", [(8, 2, 128), (4, 4, 64), (2, 1, 256)])
def test_views_and_block_gaps(ops, dev, nq, nk, hd):
    """q as columns of a wider row (aligned or not), out likewise, blocks apart from each other."""
    b = Batch([100, 40], [3, 60], nq, nk, hd, 16, torch.float16, dev, seed=15, block_gap=48)
    ref = b.run(ops)
    b.check(ref)
    for extra in (0, 3):
        buf = torch.full((63, 2 * nq * hd + extra), 7.0, dtype=torch.float16, device=dev)
        q, out = buf[:, :nq * hd], buf[:, nq * hd:2 * nq * hd]
        q.copy_(b.qd.flatten(1))
        b.run(ops, q=q, out=out)
        assert torch.equal(out, ref.flatten(1)) and torch.equal(q, b.qd.flatten(1))
        assert (buf[:, 2 * nq * hd:] == 7).all()
    wide = torch.full((2, b.width + 5), -1, dtype=torch.int32, device=dev)
    wide[:, :b.width] = b.tables
    b.tables = wide[:, :b.width]
    assert torch.equal(b.run(ops), ref)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kscale,vscale,vmean", [(6.0, 1.0, 0.0), (1.0, 1e-4, 0.0), (1.0, 300.0, 0.0), (0.01, 1.0, 50.0)])
def test_scales(ops, dev, kscale, vscale, vmean, dtype):
    """Sharp softmaxes, tiny and large values, values far from zero."""
    lens, ql = [700, 90, 260], [1, 4, 100]
    b = Batch(lens, ql, 8, 2, 128, 32, dtype, dev, seed=16, kscale=kscale, vscale=vscale, vmean=vmean)
    b.check(b.run(ops))


def test_bf16_range(ops, dev):
    """q and k far outside fp16's range, in both directions; values up to 1e30."""
    b = Batch([300, 50], [1, 40], 4, 2, 128, 16, torch.bfloat16, dev, seed=17, kscale=1e-9, vscale=1e30)
    for f in (1e9, 1e-3):
        b.q = (b.q.float() * f).bfloat16()
        b.qd = b.q.to(dev)
        b.check(b.run(ops))


def test_growing_scores(ops, dev):
    """Scores that rise along the keys, so that the running maximum moves all the way, and fall."""
    for sign in (1, -1):
        b = Batch([900], [1], 4, 4, 64, 16, torch.float16, dev, seed=18)
        n = 900
        ramp = torch.linspace(-1, 1, n)[:, None, None] * sign
        k = (ramp * torch.ones(1, 4, 64) * 2 + 0.01 * torch.randn(n, 4, 64, generator=torch.Generator().manual_seed(1)))
        c, s, m = kv4.quantise(k.half())
        b.keys[0] = kv4.values(c, s, m)
        cache = torch.empty_like(b.cache)
        cache.copy_(b.cache)
        slots = torch.tensor([int(b.host_tables[0, i // 16]) * 16 + i % 16 for i in range(n)], device=dev)
        v = torch.empty(n, 4, 64, dtype=torch.float16, device=dev)
        kk = torch.empty_like(v)
        ops.esimd_kv4_cache_read(cache, slots, kk, v)
        ops.esimd_kv4_cache_write(k.half().to(dev), v, cache, slots)
        b.cache = cache
        c, s, m = kv4.quantise(v.cpu())
        b.vals[0], b.spread[0] = kv4.values(c, s, m), 7.5 * s.double()[..., None]
        b.q = torch.ones(1, 4, 64, dtype=torch.float16)
        b.qd = b.q.to(dev)
        b.check(b.run(ops))


def test_nan_and_inf_in_the_cache(ops, dev):
    """NaN parameters behind a request's length or outside its window change nothing; inside, they reach exactly the
    rows that see them."""
    b = Batch([100, 64], [1, 64], 4, 2, 128, 16, torch.float16, dev, seed=19)
    ref = b.run(ops)
    b.check(ref)
    nan = torch.full((1, 2, 128), math.nan, dtype=torch.float16, device=dev)
    one = torch.ones_like(nan)
    slot = lambda r, t: torch.tensor([int(b.host_tables[r, t // 16]) * 16 + t % 16], device=dev)  # noqa: E731
    ops.esimd_kv4_cache_write(one, nan, b.cache, slot(1, 40))
    ops.esimd_kv4_cache_write(nan, one, b.cache, slot(0, 3))
    out = b.run(ops)
    assert out[0].isnan().all()
    assert torch.equal(out[1:41], ref[1:41]) and out[41:].isnan().all()
    out = b.run(ops, window=20)
    assert not out[0].isnan().any()                       # key 3 lies outside the window of row 99
    assert out[41:61].isnan().all() and not out[61:].isnan().any() and not out[1:41].isnan().any()


def test_bad_table_entries_are_absent_tokens(ops, dev):
    """Entries below 0 and at or above num_blocks: their tokens do not exist."""
    nk, hd, bs = 2, 64, 16
    b = Batch([100, 100], [1, 50], 4, nk, hd, bs, torch.bfloat16, dev, seed=20)
    t = b.tables.clone()
    t[0, 2], t[1, 1], t[1, 4] = -5, b.cache.shape[0], 2 ** 31 - 1
    b.tables = t
    out = b.run(ops)
    assert torch.isfinite(out).all()
    keep = torch.ones(100, dtype=torch.bool)
    keep[32:48] = False
    ref = kv4.attention(b.q[:1], b.keys[0][keep], b.vals[0][keep], b.scale)
    assert (out[:1].cpu().double() - ref).abs().max() < 2.0 ** -6
    # row 0 of request 1 stands at position 50
    keep = torch.ones(51, dtype=torch.bool)
    keep[16:32] = False
    ref = kv4.attention(b.q[1:2], b.keys[1][:51][keep], b.vals[1][:51][keep], b.scale)
    assert (out[1:2].cpu().double() - ref).abs().max() < 2.0 ** -6
    b.tables = torch.full_like(t, -1)
    assert (b.run(ops) == 0).all()


def test_lengths_beyond_the_table(ops, dev):
    """kv_lens larger than the table's reach is taken as the reach."""
    b = Batch([64], [1], 4, 2, 64, 16, torch.float16, dev, seed=21, width=4)
    ref = b.run(ops)
    b.kv_lens = torch.tensor([10 ** 6], dtype=torch.int32, device=dev)
    assert torch.equal(b.run(ops), ref)


def test_empty_calls(ops, dev):
    b = Batch([10], [1], 4, 2, 64, 16, torch.float16, dev, seed=22)
    e = torch.empty(0, 4, 64, dtype=torch.float16, device=dev)
    ops.esimd_kv4_attention(e, b.cache, b.tables, b.kv_lens, b.cu_q, e.clone(), 1.0)
    out = torch.full_like(b.qd, 7.0)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    ops.esimd_kv4_attention(b.qd, b.cache, b.tables[:0], none, b.cu_q[:1], out, 1.0)
    assert (out == 7).all()
    kv = torch.empty(0, 2, 64, dtype=torch.float16, device=dev)
    before = b.cache.clone()
    ops.esimd_kv4_cache_write(kv, kv, b.cache, torch.empty(0, dtype=torch.int64, device=dev))
    ops.esimd_kv4_cache_read(b.cache, torch.empty(0, dtype=torch.int64, device=dev), kv.clone(), kv.clone())
    assert torch.equal(before, b.cache)


def test_blocks_beyond_4_gib(ops, dev):
    """Offsets of a cache above 2^32 bytes: the same answer as from a small cache."""
    b = Batch([200, 90], [1, 30], 8, 8, 128, 256, torch.float16, dev, seed=23)
    ref = b.run(ops)
    b.check(ref)
    nb, per = b.cache.shape[0], b.cache[0].numel()
    far = (2 ** 32 + 2 ** 30) // per
    big = torch.empty(far + nb, *b.cache.shape[1:], dtype=torch.uint8, device=dev)
    big[far:] = b.cache
    small, b.cache = b.cache, big
    b.tables = torch.where(b.tables >= 0, b.tables + far, b.tables)
    assert torch.equal(b.run(ops), ref)
    k, v = (torch.empty(200, 8, 128, dtype=torch.float16, device=dev) for _ in range(2))
    k2, v2 = torch.empty_like(k), torch.empty_like(v)
    t = torch.arange(200, device=dev)
    slots = b.tables[0, 0].long() * 256 + t
    ops.esimd_kv4_cache_read(big, slots, k, v)
    ops.esimd_kv4_cache_read(small, slots - far * 256, k2, v2)
    assert torch.equal(k, k2) and torch.equal(v, v2)
    ops.esimd_kv4_cache_write(v2, k2, big, slots)
    ops.esimd_kv4_cache_write(v2, k2, small, slots - far * 256)
    assert torch.equal(big[far:], small)


def test_streams_and_graph_replays(ops, dev):
    """Write and attend on a side stream, captured; two graphs of one shape replayed in turn, with eager work between,
    against the eager results; the same call twice gives the same bits."""
    mk = lambda seed: Batch([2000, 33, 500, 1], [1, 1, 1, 1], 16, 4, 128, 32, torch.bfloat16, dev, seed=seed)  # noqa: E731
    pair = [mk(24), mk(25)]
    graphs, outs, refs = [], [], []
    for b in pair:
        refs.append(b.run(ops))
        b.check(refs[-1])
        assert torch.equal(b.run(ops), refs[-1])
        out = torch.zeros_like(b.qd)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            b.run(ops, out=out)
        graphs.append(g)
        outs.append(out)
    for i in (0, 1, 1, 0, 1):
        outs[i].zero_()
        graphs[i].replay()
        torch.randn(1000, device=dev).sum().item()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], refs[i])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = pair[0].run(ops)
    s.synchronize()
    assert torch.equal(out, refs[0])


def test_lengths_change_between_replays(ops, dev):
    """A captured call reads the lengths on the device: replayed after they changed, it answers for the new ones."""
    b = Batch([1200, 700], [1, 1], 8, 2, 128, 16, torch.float16, dev, seed=26)
    out = torch.zeros_like(b.qd)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.run(ops, out=out)
    full = (b.lens, list(b.keys), list(b.vals), list(b.spread))
    for lens in ([1200, 700], [3, 650], [1, 0], [1111, 64]):
        b.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        b.lens = lens
        b.keys, b.vals, b.spread = ([x[:n] for x, n in zip(full[i], lens)] for i in (1, 2, 3))
        b.check(out)


# ---- refusals --------------------------------------------------------------------

def test_refusals(ops, dev):
    b = Batch([20], [1], 4, 2, 64, 16, torch.float16, dev, seed=27)
    out = torch.empty_like(b.qd)
    kv = torch.zeros(3, 2, 64, dtype=torch.float16, device=dev)
    slots = torch.arange(3, device=dev)
    attn = lambda **k: ops.esimd_kv4_attention(*[k.get(n, d) for n, d in (  # noqa: E731
        ("q", b.qd), ("cache", b.cache), ("tables", b.tables), ("lens", b.kv_lens), ("cu", b.cu_q), ("out", out),
        ("scale", 0.1), ("mq", 1), ("mk", 20), ("window", 0))])
    attn()
    bad = [
        (lambda: attn(q=b.qd.float()), "fp16 or bf16"), (lambda: attn(out=out.bfloat16()), "dtype"),
        (lambda: attn(q=b.qd[:, :3]), "heads"), (lambda: attn(out=b.qd), "overlap"),
        (lambda: attn(lens=b.kv_lens.long()), "int32"), (lambda: attn(cu=b.cu_q[:1]), "cu_q"),
        (lambda: attn(tables=b.tables.long()), "block_tables"), (lambda: attn(tables=b.tables.cpu()), "GPU"),
        (lambda: attn(scale=0.0), "scale"), (lambda: attn(scale=math.nan), "scale"), (lambda: attn(window=-1), "window"),
        (lambda: attn(cache=b.cache[..., :-1]), "head_dim"), (lambda: attn(cache=b.cache[:, :, :8]), "block_size"),
        (lambda: attn(cache=b.cache.to(torch.int8)), "uint8"), (lambda: attn(cache=b.cache.transpose(1, 2)), "block"),
        (lambda: ops.esimd_kv4_cache_write(kv, kv[:2], b.cache, slots), "rows"),
        (lambda: ops.esimd_kv4_cache_write(kv, kv.bfloat16(), b.cache, slots), "dtype"),
        (lambda: ops.esimd_kv4_cache_write(kv, kv, b.cache, slots.int()), "int64"),
        (lambda: ops.esimd_kv4_cache_write(kv[:, :1], kv[:, :1], b.cache, slots), "k must be"),
        (lambda: ops.esimd_kv4_cache_write(kv.transpose(1, 2), kv, b.cache, slots), "k must be"),
        (lambda: ops.esimd_kv4_cache_write(kv, kv, b.cache, slots[:2]), "slot_mapping"),
        (lambda: ops.esimd_kv4_cache_read(b.cache, slots, kv, kv), "overlap"),
        (lambda: ops.esimd_kv4_cache_read(b.cache, slots, kv, kv[:2].clone()), "row for each"),
    ]
    for call, text in bad:
        with pytest.raises(RuntimeError, match=text):
            call()
