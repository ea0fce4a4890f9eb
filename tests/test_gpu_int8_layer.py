"""GPU: the int8 operators together -- decoder layers of int8 weights, eager and captured, with and without the
4-bit cache, products that split K in graphs that run side by side, other streams.

A layer is compared with the oracle stage by stage, each on the device's own inputs of that stage (a value that a
step before rounds differently can move a code, so the oracle's own inputs would not do), and a captured
step with the eager one, bit for bit.
"""

import pytest
import torch

from esimd_learning_amd import cabi, synthetic
from esimd_learning_amd.kv4 import KV4Cache
from esimd_learning_amd.layer import GemmaDecodeLayer, capture_forward, forward
from oracle import int8 as oint8

pytestmark = pytest.mark.gpu

SMALL = dict(hidden=512, n_q=4, n_kv=2, head_dim=64, mlp=1040)
WIDE = dict(hidden=2048, n_q=8, n_kv=4, head_dim=128, mlp=4096)


def _layer(dims, M, dev, seed=10, dtype=torch.float16, **kw):
    p = synthetic.gemma_layer(seed=seed, fmt=torch.int8, **dims)
    if kw.pop("silu", False):
        p["activation"] = "silu"
    return p, GemmaDecodeLayer(p, M, dev, dtype=dtype, **kw)


def _inputs(M, dims, dev, seed=20, dtype=torch.float16):
    h, r = (synthetic.activations(M, dims["hidden"], seed=seed + i, dtype=dtype) for i in (0, 1))
    return h, r, synthetic.positions(M, seed=seed + 2)


@pytest.mark.parametrize("dims,M,kw", [(SMALL, 1, {}), (SMALL, 3, dict(silu=True)), (SMALL, 6, dict(fuse_glu=False)),
                                       (SMALL, 37, {}), (SMALL, 130, dict(silu=True)), (WIDE, 2, {}), (WIDE, 64, {}),
                                       (WIDE, 300, dict(fuse_glu=False)), (WIDE, 5, dict(dtype=torch.bfloat16))])
def test_layer_by_stages(ops, dev, dims, M, kw):
    """Each stage of a step against the oracle on the device's own inputs of that stage: codes and products bit
    for bit, the gated block and the codes behind a norm within their bounds (those of test_gpu_int8.py)."""
    dtype = kw.get("dtype", torch.float16)
    p, layer = _layer(dims, M, dev, **kw)
    assert layer.int8 and not (layer.defer_norm or layer.fuse_tails or layer.fuse_norm)
    h, r, pos = _inputs(M, dims, dev, dtype=dtype)
    hd, rd = h.to(dev), r.to(dev)
    out = layer.step(hd, rd, pos.to(dev))
    assert torch.equal(hd.cpu(), h)

    def normed(x, res, w):
        """The operator's codes of a norm, checked, and its residual."""
        q, s, new = torch.empty(x.shape, dtype=torch.int8, device=dev), torch.empty(M, device=dev), res.clone()
        ops.esimd_fused_add_rms_norm_quant_int8(x, new, w, p["eps"], q, s)
        kept, exact = oint8.add_rms_norm(x.cpu(), res.cpu(), w.cpu(), p["eps"])
        assert torch.equal(new.cpu(), kept)
        rel = (x.shape[1] / 2 + 8) * 2.0 ** -24
        want_s = oint8.quant(exact)[1].double()
        assert ((s.cpu().double() - want_s).abs() <= want_s * rel).all()
        assert ((q.cpu().double() - exact / want_s[:, None]).abs() <= 0.5 + 254 * rel).all()
        return q, s, new

    nq, nk, hd_ = dims["n_q"], dims["n_kv"], dims["head_dim"]
    q, s, r1 = normed(h.to(dev), r.to(dev), layer.w_in)
    qkv = oint8.product(q, s, p["Wqkv"], p["sqkv"], dtype).to(dev)
    ops.esimd_qk_norm_rope(qkv[:, : nq * hd_], qkv[:, nq * hd_:(nq + nk) * hd_], layer.qw, layer.kw, pos.to(dev), p["eps"],
                           p["theta"], True)
    assert torch.equal(layer.qkv, qkv) and torch.equal(layer.attn, qkv[:, : nq * hd_])
    codes, scale = oint8.quant(layer.attn.cpu())
    assert torch.equal(layer.a8.cpu(), codes)
    assert torch.equal(layer.o.cpu(), oint8.product(codes, scale, p["Wo"], p["so"], dtype))
    q, s, r2 = normed(layer.o, r1, layer.w_post)
    assert torch.equal(layer.q8, q) and torch.equal(rd, r2)
    if layer.fuse_glu:
        want, bound = oint8.gated(q, s, p["Wgu"], p["sgu"], layer.activation)
        fi = torch.finfo(dtype)
        limit = bound + want.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
        assert ((layer.act.cpu().double() - want).abs() <= limit).all()
    else:
        gu, act = oint8.product(q, s, p["Wgu"], p["sgu"], dtype).to(dev), torch.empty_like(layer.act)
        ops.esimd_gelu_and_mul(act, gu)
        assert torch.equal(layer.gu, gu) and torch.equal(layer.act, act)
    codes, scale = oint8.quant(layer.act.cpu())
    assert torch.equal(layer.d8.cpu(), codes)
    assert torch.equal(out.cpu(), oint8.product(codes, scale, p["Wd"], p["sd"], dtype))


@pytest.mark.parametrize("M,requests", [(3, 3), (70, 5)])
def test_layers_attend_captured(ops, dev, M, requests):
    """Two int8 layers over a 4-bit cache, four steps: replays of one graph equal the eager steps."""
    dims, blocks = SMALL, 64

    def setup():
        stack = [_layer(dims, M, dev, seed=s)[1] for s in (50, 51)]
        return stack, KV4Cache(2, blocks, dims["n_kv"], dims["head_dim"], requests, M, 256, 16, dev)

    q_lens = torch.tensor([M // requests] * requests, dtype=torch.int32, device=dev)
    steps = [_inputs(M, dims, dev, seed=60 + 10 * i)[:2] for i in range(4)]
    stack, kv = setup()
    eager = []
    for h, r in steps:
        h, r = h.to(dev), r.to(dev)
        kv.advance(q_lens, fixed_rows=True)
        eager.append((forward(stack, h, r, kv.positions, kv).clone(), r))
    stack, kv = setup()
    hb, rb = (x.to(dev) for x in steps[0])
    g = capture_forward(stack, hb, rb, kv.positions, kv=kv, q_lens=q_lens)
    for (h, r), (out, res) in zip(steps, eager):
        hb.copy_(h)
        rb.copy_(r)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(stack[1].out, out) and torch.equal(rb, res)
        torch.randn(1000, device=dev).sum().item()


def test_graphs_with_split_products_side_by_side(ops, dev):
    """Two captured products that split K, each with its own partial sums, replayed together on two streams."""
    m, n, k = 128, 512, 8192
    lib = cabi.load()
    assert lib.cek_gemm_int8_plan(m, n, k, 0, 1 << 40) % 16 > 1
    jobs = []
    for i in range(2):
        a, b = (torch.randint(-127, 128, (rows, k), generator=synthetic.gen(70 + 2 * i + j), dtype=torch.int8)
                for j, rows in ((0, m), (1, 2 * n)))
        sa, sb = torch.rand(m, generator=synthetic.gen(80 + i)) * 1e-3, torch.rand(2 * n, generator=synthetic.gen(82 + i)) * 1e-3
        y, z = torch.empty(m, 2 * n, dtype=torch.float16, device=dev), torch.empty(m, n, dtype=torch.float16, device=dev)
        ad, bd, sad, sbd = (t.to(dev) for t in (a, b, sa, sb))
        ops.esimd_gemm_int8_a8w8_glu(ad, sad, bd, sbd, z, "silu")
        jobs.append((ad, bd, sad, sbd, y, z, oint8.product(a, sa, b, sb, torch.float16).to(dev), z.clone(), torch.cuda.Stream()))
    graphs = []
    for ad, bd, sad, sbd, y, z, _, _, st in jobs:
        st.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            for _ in range(4):
                ops.esimd_gemm_int8_a8w8(ad, sad, bd, sbd, y)
                ops.esimd_gemm_int8_a8w8_glu(ad, sad, bd, sbd, z, "silu")
        graphs.append(g)
    for _ in range(3):
        for (_, _, _, _, y, z, _, _, _) in jobs:
            y.zero_()
            z.zero_()
        torch.cuda.synchronize()
        for g, job in zip(graphs, jobs):
            with torch.cuda.stream(job[-1]):
                g.replay()
        torch.cuda.synchronize()
        for _, _, _, _, y, z, want, gated, _ in jobs:
            assert torch.equal(y, want) and torch.equal(z, gated)


def test_on_another_stream(ops, dev):
    p, layer = _layer(SMALL, 33, dev, seed=90)
    h, r, pos = _inputs(33, SMALL, dev, seed=91)
    hd, rd, pos_d = h.to(dev), r.to(dev), pos.to(dev)
    want = layer.step(hd, rd.clone(), pos_d).clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        big = torch.randn(4096, 4096, device=dev)
        late = h.to(dev) + (big @ big)[0, 0] * 0       # ready only when the product on this stream is done
        got = layer.step(late, rd, pos_d).clone()
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)


def test_refusals(dev):
    p = synthetic.gemma_layer(seed=10, fmt=torch.int8, **SMALL)
    mixed = dict(p, Wd=synthetic.gemma_layer(seed=10, **SMALL)["Wd"])
    for bad, kw in ((mixed, {}), (p, dict(act_fp8=True)), (dict(p, so=p["so"].half()), {}),
                    (dict(p, activation="silu"), dict(fuse_glu=False)), (dict(p, activation="relu"), {})):
        with pytest.raises(ValueError):
            GemmaDecodeLayer(bad, 2, dev, **kw)
    with pytest.raises(ValueError):
        GemmaDecodeLayer(dict(synthetic.gemma_layer(seed=10, **SMALL), activation="silu"), 2, dev)
    layer = GemmaDecodeLayer(p, 2, dev)
    h, r, pos = (t.to(dev) for t in _inputs(2, SMALL, dev))
    with pytest.raises(ValueError):
        layer.step(h, r, pos, next_norm=(layer.w_in, 0))
