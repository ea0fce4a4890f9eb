"""CPU: the 4-bit cache's entry points refuse what they cannot do before any GPU work -- through the C ABI, and as torch
ops, which have no CPU form."""

import ctypes as C

import pytest
import torch

import esimd_learning_amd
from esimd_learning_amd import cabi

P, ODD, N = C.c_void_p(16), C.c_void_p(8), None     # never dereferenced: every call below fails its checks first
INVALID, UNSUPPORTED, OK = cabi.CEK_ERR_INVALID, cabi.CEK_ERR_UNSUPPORTED, cabi.CEK_OK
STRIDE = 2 * 16 * (64 + 8)                          # a block of 2 heads, 16 tokens, 64 values


def _call(fn, names, base, change):
    assert set(change) <= set(names), change
    return fn(*[change.get(n, base[n]) for n in names])


ROWS = dict(T=4, n_kv=2, hd=64, bs=16, blocks=8, ks=128, vs=128, stride=STRIDE, io=0, stream=N)
ROWS_BAD = [
    (dict(T=-1), INVALID), (dict(T=2 ** 31), INVALID), (dict(n_kv=0), INVALID), (dict(n_kv=5000), INVALID),
    (dict(hd=96), UNSUPPORTED), (dict(hd=512), UNSUPPORTED), (dict(bs=8), UNSUPPORTED), (dict(bs=48), UNSUPPORTED),
    (dict(bs=512), UNSUPPORTED), (dict(blocks=0), INVALID), (dict(blocks=2 ** 31), INVALID), (dict(ks=127), INVALID),
    (dict(vs=127), INVALID), (dict(stride=STRIDE - 16), INVALID), (dict(stride=STRIDE + 8), INVALID),
    (dict(stride=2 ** 32), UNSUPPORTED), (dict(io=2), INVALID), (dict(io=-1), INVALID), (dict(k=N), INVALID),
    (dict(v=N), INVALID), (dict(cache=N), INVALID), (dict(cache=ODD), INVALID), (dict(slots=N), INVALID),
    (dict(T=0, k=N, v=N, slots=N), OK),
]


@pytest.mark.parametrize("change,rc", ROWS_BAD)
def test_cache_write_and_read(change, rc):
    lib = cabi.load()
    tail = list(ROWS)
    base = dict(ROWS, k=P, v=P, cache=P, slots=P)
    assert _call(lib.cek_kv4_cache_write, ["k", "v", "cache", "slots"] + tail, base, change) == rc
    assert _call(lib.cek_kv4_cache_read, ["cache", "slots", "k", "v"] + tail, base, change) == rc


ATTN = dict(q=P, cache=P, tables=P, lens=P, cu=P, out=P, T=4, R=2, n_q=8, n_kv=2, hd=64, bs=16, blocks=8, qs=512, os=512,
            stride=STRIDE, ts=4, width=4, scale=0.125, mq=0, mk=0, window=0, io=1, ws=P, ws_bytes=0, stream=N)


@pytest.mark.parametrize("change,rc", [
    (dict(q=N), INVALID), (dict(cache=N), INVALID), (dict(cache=ODD), INVALID), (dict(tables=N), INVALID),
    (dict(lens=N), INVALID), (dict(cu=N), INVALID), (dict(out=N), INVALID), (dict(T=-1), INVALID), (dict(R=-1), INVALID),
    (dict(n_q=7), INVALID), (dict(n_q=0), INVALID), (dict(hd=80), UNSUPPORTED), (dict(bs=20), UNSUPPORTED),
    (dict(blocks=0), INVALID), (dict(qs=511), INVALID), (dict(os=100), INVALID), (dict(stride=16), INVALID),
    (dict(ts=3), INVALID), (dict(width=0), INVALID), (dict(width=2 ** 28, ts=2 ** 28), INVALID), (dict(scale=0.0), INVALID),
    (dict(scale=-1.0), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(mq=-1), INVALID), (dict(mk=-1), INVALID), (dict(window=-1), INVALID), (dict(window=2 ** 31), INVALID),
    (dict(io=7), INVALID), (dict(ws=ODD), INVALID), (dict(ws_bytes=-1), INVALID),
    (dict(T=2 ** 28), UNSUPPORTED),                       # 2^30 rows of a kv head
    (dict(R=2 ** 26 + 1), UNSUPPORTED),
    (dict(T=0, q=N, out=N), OK), (dict(R=0, lens=N), OK),
])
def test_attention(change, rc):
    lib = cabi.load()
    assert _call(lib.cek_kv4_attention, list(ATTN), ATTN, change) == rc


def test_attention_workspace():
    """Keys that may be long are shared, which takes room; short ones are not; nonsense needs none."""
    size = cabi.load().cek_kv4_attention_workspace_size
    assert size(1, 1, 32, 8, 128, 1, 1024) == 0
    assert 0 < size(1, 1, 32, 8, 128, 1, 1025) <= 2 ** 26
    assert size(1, 1, 32, 8, 128, 0, 0) > 0
    for bad in ((0, 1, 32, 8, 128, 1, 0), (1, 0, 32, 8, 128, 1, 0), (1, 1, 30, 8, 128, 1, 0), (1, 1, 32, 8, 100, 1, 0),
                (-5, 1, 32, 8, 128, 1, 0), (1, 1, 0, 8, 128, 1, 0), (1, 1, 32, 0, 128, 1, 0)):
        assert size(*bad) == 0, bad


TABLES = dict(lens=P, keep=P, q=P, R=3, bs=16, ring=P, blocks=8, state=P, tables=P, ts=4, width=4, lens_out=P, state_out=P,
              cu=P, slots=P, pos=P, T=4, status=P, stream=N)


@pytest.mark.parametrize("change,rc", [
    *[({n: N}, INVALID) for n in ("lens", "keep", "q", "ring", "state", "tables", "lens_out", "state_out", "cu", "slots",
                                  "pos", "status")],
    (dict(R=-1), INVALID), (dict(R=4097), UNSUPPORTED), (dict(bs=8), UNSUPPORTED), (dict(bs=24), UNSUPPORTED),
    (dict(blocks=0), INVALID), (dict(ts=3), INVALID), (dict(width=0), INVALID),
    (dict(width=2 ** 28, ts=2 ** 28), UNSUPPORTED), (dict(T=-1), INVALID), (dict(T=2 ** 31), INVALID),
])
def test_block_tables(change, rc):
    lib = cabi.load()
    assert _call(lib.cek_kv_block_tables, list(TABLES), TABLES, change) == rc


def test_torch_ops():
    """Registered, with the written tensors marked, and loud about CPU tensors."""
    ops = esimd_learning_amd.ops()
    for name, written in (("esimd_kv_block_tables", 8), ("esimd_kv4_cache_write", 1), ("esimd_kv4_cache_read", 2),
                          ("esimd_kv4_attention", 1)):
        schema = str(getattr(torch.ops.custom_esimd_kernels_vllm, name).default._schema)
        assert len({x.split("!")[0][-1] for x in schema.split("Tensor(")[1:]}) == written, schema
    cache = ops.kv4_cache(4, 2, 16, 64, "cpu")
    assert cache.shape == (4, 2, 16, 72) and cache.dtype == torch.uint8
    ring, state = ops.kv_free_ring(4, "cpu")
    assert ring.tolist() == [0, 1, 2, 3] and state.tolist() == [0, 4]
    x, slots = torch.zeros(3, 2, 64, dtype=torch.float16), torch.arange(3)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    for call in (lambda: ops.esimd_kv4_cache_write(x, x, cache, slots),
                 lambda: ops.esimd_kv4_cache_read(cache, slots, x, x.clone()),
                 lambda: ops.esimd_kv4_attention(x, cache, torch.zeros(1, 4, dtype=torch.int32), i32(1), i32(2), x.clone(), 1.0),
                 lambda: ops.esimd_kv_block_tables(i32(1), i32(1), i32(1), 16, ring, state, torch.zeros(1, 4, dtype=torch.int32),
                                                   i32(1), i32(2), i32(2), slots, slots.clone(), i32(1))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
