"""GPU: the 4-bit cache's operators together, as a serving loop calls them -- tables, writes and attention of one cache
over many steps, and decoder layers that attend through it, eager and captured.

Tables and cached bytes are equal to the oracle's.  Attention is compared in fp64 with the tolerance of
tests/test_gpu_kv4.py, which is derived there.  In a layer each stage is compared on the device's own inputs of that
stage (a rounding of k can move a 4-bit code, so the oracle's own k would not do): the projections, the cache, the
attention, and what follows it.
"""

import sys

import pytest
import torch

from conftest import assert_close_fp
from esimd_learning_amd import synthetic
from esimd_learning_amd.kv4 import KV4Cache
from esimd_learning_amd.layer import GemmaDecodeLayer, capture_forward, forward
from oracle import kv4
from oracle import layer as olayer

pytestmark = pytest.mark.gpu

EPS = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
SMALL = dict(hidden=512, n_q=4, n_kv=2, head_dim=64, mlp=1024)
WIDE = dict(hidden=4096, n_q=16, n_kv=4, head_dim=256, mlp=4096)     # shapes of the deferred norms


def _say(*what):
    print(*what, flush=True)
    sys.stdout.flush()


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Mirror:
    """What the cache should hold: the oracle's tables, and each request's values by layer."""

    def __init__(self, layers, blocks, requests, tokens, max_len, bs):
        self.bs, self.T = bs, tokens
        self.ring, self.state = list(range(blocks)), [0, blocks]
        self.tables = [[0] * -(-max_len // bs) for _ in range(requests)]
        self.lens = [0] * requests
        self.rows = [[[] for _ in range(requests)] for _ in range(layers)]     # (k, v, spread of v) a token

    def advance(self, q_lens, keep=None):
        keep = self.lens if keep is None else [min(k, n) for k, n in zip(keep, self.lens)]
        for layer in self.rows:
            for r, n in enumerate(keep):
                del layer[r][n:]
        self.lens, self.state, self.cu, self.slots, self.positions, self.status = kv4.block_tables(
            self.lens, keep, q_lens, self.bs, self.ring, self.state, self.tables, self.T)

    def check(self, kv):
        assert kv.lens.tolist() == self.lens and kv.cu_q.tolist() == self.cu and kv.status.tolist() == self.status
        assert kv.slot_mapping.tolist() == self.slots and kv.positions.tolist() == self.positions
        assert kv.ring_state.tolist() == list(self.state)
        table = kv.block_tables.tolist()
        for r, n in enumerate(self.lens):
            used = -(-n // self.bs)
            assert table[r][:used] == self.tables[r][:used]

    def put(self, layer, k, v):
        """Rows k, v [T, n_kv, hd] of a step."""
        (ck, sk, mk), (cv, sv, mv) = kv4.quantise(k), kv4.quantise(v)
        vk, vv = kv4.values(ck, sk, mk), kv4.values(cv, sv, mv)
        for r in range(len(self.lens)):
            for t in range(self.cu[r], self.cu[r + 1]):
                self.rows[layer][r].append((vk[t], vv[t], 7.5 * sv[t].double()[..., None]))

    def check_attention(self, layer, q, out, scale, window=0):
        """q, out [T, n_q, hd] on the CPU: every row of a request, and no other."""
        for r, n in enumerate(self.lens):
            a, b = self.cu[r], self.cu[r + 1]
            if a == b:
                continue
            keys, vals, spread = (torch.stack(x) for x in zip(*self.rows[layer][r]))
            assert len(keys) == n
            ref, (sp, size) = kv4.attention(q[a:b], keys, vals, scale, window, weigh=(spread, vals.abs()))
            tol = EPS[q.dtype] / 2 * ref.abs() + 2.0 ** -11 * sp + 2.0 ** -13 * size + TINY[q.dtype]
            err = (out[a:b].double() - ref).abs()
            assert not (err > tol).any() and torch.isfinite(out[a:b]).all(), \
                f"layer {layer}, request {r} of {n}: worst {float((err / tol).max()):.3g} tolerances"


# (new tokens, kept of the cached ones or None: all) of four requests, step by step: prompts, a chunk beside decodes,
# drafts, their rollback, one that ends, one that starts over, one idle, and one too many for the blocks there are
STEPS = [([40, 0, 3, 0], None), ([1, 33, 1, 0], None), ([4, 1, 4, 17], None), ([4, 4, 2, 1], [42, 99, 5, 99]),
         ([1, 0, 1, 40], [99, 99, 0, 0]), ([0, 0, 0, 0], None), ([1, 7, 1, 1], [99, 0, 99, 99]), ([1, 1, 60, 1], None),
         ([1, 1, 1, 1], None), ([64, 0, 0, 0], [0, 0, 0, 0])]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq,nk,hd,bs,blocks,window", [(4, 2, 64, 16, 9, 0), (8, 1, 128, 16, 12, 20), (2, 2, 256, 32, 6, 0)])
def test_steps_of_a_serving_loop(ops, dev, nq, nk, hd, bs, blocks, window, dtype):
    _say("serving loop", nq, nk, hd, bs, blocks, window, dtype)
    R, T, L = 4, 64, 2
    kv = KV4Cache(L, blocks, nk, hd, R, T, max_len=112, block_size=bs, device=dev)
    for layer in kv.layers:
        layer.window = window
    m = Mirror(L, blocks, R, T, 112, bs)
    g = torch.Generator().manual_seed(hd + window)
    for q_lens, keep in STEPS:
        m.advance(q_lens, keep)
        kv.advance(_i32(q_lens, dev), None if keep is None else _i32(keep, dev))
        m.check(kv)
        for i, layer in enumerate(kv.layers):
            qkv = (torch.randn(T, nq + 2 * nk, hd, generator=g) * 1.5).to(dtype)
            d = qkv.to(dev)
            out = torch.full((T, nq * hd), 7.0, dtype=dtype, device=dev)
            layer.attend(d[:, :nq], d[:, nq:nq + nk], d[:, nq + nk:], out)
            m.put(i, qkv[:, nq:nq + nk], qkv[:, nq + nk:])
            out = out.cpu().view(T, nq, hd)
            m.check_attention(i, qkv[:, :nq], out, hd ** -0.5, window)
            assert (out[m.cu[-1]:] == 7.0).all(), "rows behind the last token stay"
    # what a request holds, read back through its slots
    r = max(range(R), key=lambda i: m.lens[i])
    k, v = kv.layers[1].read(kv.slots(r, 0, m.lens[r]), dtype)
    for got, ref in ((k, 0), (v, 1)):
        ref = torch.stack([x[ref] for x in m.rows[1][r]])
        assert ((got.cpu().double() - ref).abs() <= (EPS[dtype] / 2 + 2.0 ** -23) * ref.abs() + TINY[dtype]).all()


def _stack(dims, M, dev, n=2, **mode):
    params = [synthetic.gemma_layer(seed=70 + i, **dims) for i in range(n)]
    return params, [GemmaDecodeLayer(p, M, dev, **mode) for p in params]


MODES = [(SMALL, 6, {}), (SMALL, 3, dict(fuse_norm=True)), (SMALL, 6, dict(act_fp8=True)),
         (SMALL, 4, dict(fuse_tails=False)), (SMALL, 4, dict(fuse_norm=True, act_fp8=True)), (WIDE, 4, {})]


@pytest.mark.parametrize("dims,M,mode", MODES)
def test_layer_attends_through_its_cache(ops, dev, dims, M, mode):
    """One layer over four steps (a prompt, decodes with drafts, a rollback, a padded step)."""
    _say("layer", dims, M, mode)
    (p,), (layer,) = _stack(dims, M, dev, 1, **mode)
    hd, nq, nk = dims["head_dim"], dims["n_q"], dims["n_kv"]
    kv = KV4Cache(1, 8, nk, hd, 2, M, max_len=48, block_size=16, device=dev)
    m = Mirror(1, 8, 2, M, 48, 16)
    for step, (q_lens, keep) in enumerate([([M, 0], None), ([1, M - 1], None), ([M - 1, 1], [M, 99]), ([1, 0], None)]):
        m.advance(q_lens, keep)
        kv.advance(_i32(q_lens, dev), None if keep is None else _i32(keep, dev), max_q_len=M, max_kv_len=48)
        m.check(kv)
        h = synthetic.activations(M, dims["hidden"], seed=80 + step)
        r = synthetic.activations(M, dims["hidden"], seed=90 + step)
        rd = r.to(dev)
        out = layer.step(h.to(dev), rd, kv.positions, kv=kv.layers[0]).cpu()
        n = m.cu[-1]
        rows = layer.qkv.cpu().view(M, nq + 2 * nk, hd)
        attn = layer.attn.cpu()
        m.put(0, rows[:, nq:nq + nk], rows[:, nq + nk:])
        m.check_attention(0, rows[:, :nq], attn.view(M, nq, hd), hd ** -0.5)
        ref, ref_r, ref_qkv = olayer.decoder_step(p, h, r, kv.positions.cpu(), act_fp8=layer.act_fp8,
                                                  attend=lambda q, k, v: attn)
        assert_close_fp(rows.view(M, -1)[:n], ref_qkv.float()[:n], "projections")
        assert_close_fp(rd.cpu()[:n], ref_r.float()[:n], "residual after the layer")
        assert_close_fp(out[:n], ref[:n], "layer output")


@pytest.mark.parametrize("dims,M,mode", MODES)
def test_captured_steps_equal_eager_steps(ops, dev, dims, M, mode):
    """A captured forward that advances the cache: every replay is the next step, with the eager loop's bits; another
    graph over another cache is replayed in between, and eager work with it."""
    _say("captured", dims, M, mode)
    _, stack = _stack(dims, M, dev, **mode)
    hd, nk = dims["head_dim"], dims["n_kv"]
    mk = lambda: KV4Cache(2, 40, nk, hd, M, M, max_len=100, block_size=16, device=dev)  # noqa: E731
    ones = torch.ones(M, dtype=torch.int32, device=dev)
    steps = [(synthetic.activations(M, dims["hidden"], seed=100 + i).to(dev),
              synthetic.activations(M, dims["hidden"], seed=200 + i).to(dev)) for i in range(20)]
    eager, ref = mk(), []
    for h, r in steps:
        h, r = h.clone(), r.clone()
        eager.advance(ones, None, 1, 100)
        out = forward(stack, h, r, eager.positions, eager)
        ref.append((out.clone(), r))
    bufs = [(mk(), steps[0][0].clone(), steps[0][1].clone()) for _ in range(2)]
    graphs = [capture_forward(stack, h, r, c.positions, kv=c, q_lens=ones, max_q_len=1, max_kv_len=100)
              for c, h, r in bufs]
    at = [0, 0]
    for i in (0, 0, 1, 0, 1, 1, 1, 0) + (0, 1) * 12:
        c, h, r = bufs[i]
        h.copy_(steps[at[i]][0])
        r.copy_(steps[at[i]][1])
        graphs[i].replay()
        torch.randn(1000, device=dev).sum().item()
        assert torch.equal(stack[-1].out, ref[at[i]][0]), (i, at[i])
        assert torch.equal(r, ref[at[i]][1])
        at[i] += 1
    for i in (0, 1):
        assert bufs[i][0].lens.tolist() == [at[i]] * M


def test_forward_on_another_stream(ops, dev):
    _, stack = _stack(SMALL, 3, dev)
    res = []
    for side in (False, True):
        kv = KV4Cache(2, 9, 2, 64, 3, 3, max_len=40, block_size=16, device=dev)
        s = torch.cuda.Stream() if side else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for i in range(18):
                h = synthetic.activations(3, 512, seed=300 + i).to(dev)
                r = synthetic.activations(3, 512, seed=330 + i).to(dev)
                kv.advance(torch.ones(3, dtype=torch.int32, device=dev))
                out = forward(stack, h, r, kv.positions, kv).clone()
        s.synchronize()
        res.append((out, r, kv.lens.tolist()))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1]) and res[0][2] == res[1][2] == [18] * 3


def test_refusals(ops, dev):
    _, stack = _stack(SMALL, 3, dev)
    kv = KV4Cache(1, 4, 2, 64, 3, 3, max_len=16, block_size=16, device=dev)
    h = torch.zeros(3, 512, dtype=torch.float16, device=dev)
    with pytest.raises(ValueError, match="layer"):
        forward(stack, h, h.clone(), kv.positions, kv)
    with pytest.raises(ValueError, match="rows"):
        forward(stack, h, h.clone(), kv.positions, KV4Cache(2, 4, 2, 64, 3, 5, max_len=16, block_size=16, device=dev))
    with pytest.raises(RuntimeError, match="block_size"):
        KV4Cache(1, 4, 2, 64, 3, 3, max_len=16, block_size=24, device=dev).advance(torch.ones(3, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="q_lens"):
        kv.advance(torch.ones(2, dtype=torch.int32, device=dev))
