"""Every compiled form of the int8 product and gated block: rings, v_dot4 and split tiles, at ragged sizes.

Sums are integers below 2^53, exact in float64 in any order, so products are equal bit for bit; the gated block lies
within the bound that oracle.int8.gated derives plus half a step of its type.
"""

import math

import pytest
import torch

from esimd_learning_amd import cabi

ALL = 1 << 40                          # a workspace that holds any split

# Rings: rows of b of a workgroup -> outputs that make the planner take them (a workgroup per CU: more than 256 times
# the next smaller form's rows), and rows of a -> batches and a K with more stages than the ring has slots.
OUTPUTS = {8: 1301, 12: 2087, 16: 3077, 24: 5303, 32: 6507, 40: 9529, 48: 11525, 56: 13535, 64: 15541}
BATCHES = {8: ((5, 8), 5648), 16: ((9, 16), 5648), 32: ((17, 30), 4624), 48: ((33, 47), 3088), 64: ((49, 64), 2576)}
def _far(ar, rw):                      # (of many wide rows with a longer K the tiles take care)
    return BATCHES[ar][1] if ar < 48 or rw < 48 else 2064 if ar + rw < 128 else 1552


RINGS = [(gated, ar, rw, ms[long], n // (1 + gated), k)
         for gated in (0, 1) for ar, (ms, _) in BATCHES.items() for rw, n in OUTPUTS.items() if not (gated and rw == 12)
         for long, k in enumerate((80 if rw % 16 else 528, _far(ar, rw)))]
# the gated block's rotated first stage, from 8192 outputs on
ROTATED = [(1, 8, 24, 6, 8515, 1552), (1, 32, 40, 27, 8515, 2064), (1, 32, 64, 31, 14539, 2064), (0, 8, 16, 7, 18555, 3088)]

# v_dot4: rows of a thread, by the outputs, in each of the four lengths of K that have a form
LENGTHS = (528, 1552, 3088, 8208)
DOT = [(0, m, 4 if n > 8192 and k <= 2048 else 2, n, k) for m in (1, 2, 3) for k in LENGTHS for n in (331, 8195)]
DOT += [(1, m, 2, n, k) for m in (1, 2, 3, 4) for k in LENGTHS for n in (165,)]

# Tiles that split K: (tile, parts) -> rows, rows of b, K
SPLIT = {(0, 2): (513, 10242, 24592), (0, 3): (385, 8194, 12304), (0, 6): (130, 8194, 24592),
         (1, 2): (1030, 4610, 16400), (1, 3): (385, 6146, 16400), (1, 8): (2050, 514, 24592),
         (2, 2): (385, 6146, 12304), (2, 4): (130, 6146, 12304), (2, 12): (130, 2050, 24592),
         (3, 2): (257, 8194, 12304), (3, 3): (513, 3586, 8208), (3, 6): (65, 8194, 12304), (3, 12): (65, 4098, 24592),
         (4, 2): (513, 4610, 12304), (4, 4): (257, 3586, 12304), (4, 6): (3000, 130, 8208), (4, 12): (1500, 130, 16400),
         (5, 3): (65, 8194, 8208), (5, 4): (3000, 130, 5136), (5, 12): (65, 2050, 16400),
         (6, 2): (130, 3586, 5136), (6, 4): (1000, 130, 3088), (6, 6): (65, 70, 3088), (6, 12): (65, 70, 8208)}


def test_every_form_is_listed():
    lib = cabi.load()
    seen = set()
    for gated, ar, rw, m, n, k in RINGS + ROTATED:
        assert lib.cek_gemm_int8_few_plan(m, n, k, gated, ALL) == 256 * ar + rw, (gated, ar, rw, m, n, k)
        assert lib.cek_gemm_int8_plan(m, n, k, gated, ALL) == -1
        seen.add((gated, ar, rw))
    assert len(seen) == 5 * 9 + 5 * 8
    for gated, m, rows, n, k in DOT:
        assert lib.cek_gemm_int8_few_plan(m, n, k, gated, ALL) == 16 * m + rows, (gated, m, rows, n, k)
    assert len({(g, m, r, k) for g, m, r, _, k in DOT}) == 3 * (4 + 2) + 4 * 4
    for (tile, parts), (m, n, k) in SPLIT.items():
        for gated in (0, 1):
            assert lib.cek_gemm_int8_plan(m, n // (1 + gated), k, gated, ALL) == 16 * tile + parts, (tile, parts, gated)
            assert lib.cek_gemm_int8_few_plan(m, n // (1 + gated), k, gated, ALL) == 0
    assert {tile for tile, _ in SPLIT} == set(range(7))
    for bad in ((0, 8, 64), (8, 0, 64), (-1, 8, 64), (8, 8, 72), (8, 2 ** 31, 64), (8, 8, 131072)):
        assert lib.cek_gemm_int8_few_plan(*bad, 0, ALL) == -1


def _check(ops, dev, m, n, k, act, dtype):
    """n: outputs.  The op on random codes, its output between guards."""
    g = torch.Generator(device=dev).manual_seed(m + n + k)
    rows = 2 * n if act else n
    a, b = (torch.randint(-128, 128, (r, k), generator=g, dtype=torch.int8, device=dev) for r in (m, rows))
    sa, sb = torch.rand(m, generator=g, device=dev) * 0.01, torch.rand(rows, generator=g, device=dev) * 0.01
    if act:
        sb /= 127 * math.sqrt(k)                      # gates of some units
    buf = torch.full((m * n + 128,), math.nan, dtype=dtype, device=dev)
    y = buf[64:64 + m * n].view(m, n)
    acc = a.double() @ b.double().t()
    if act:
        ops.esimd_gemm_int8_a8w8_glu(a, sa, b, sb, y, act)
        gu = acc * sb.double() * sa.double()[:, None]
        gate, up = gu[:, :n], gu[:, n:]
        z = gate if act == "silu" else 2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
        f = gate * torch.sigmoid(z) * up
        fi = torch.finfo(dtype)
        rel = (16 + 16 * z.abs() * torch.sigmoid(-z)) * 2.0 ** -24 + fi.eps / 2
        limit = f.abs() * rel + gate.abs() * up.abs() * 2.0 ** -126 + fi.smallest_normal * fi.eps / 2 + 2.0 ** -149
        assert ((y.double() - f).abs() <= limit).all()
    else:
        ops.esimd_gemm_int8_a8w8(a, sa, b, sb, y)
        assert torch.equal(y, (acc.float() * sb * sa[:, None]).to(dtype))
    assert torch.isnan(buf[:64]).all() and torch.isnan(buf[64 + m * n:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("gated,ar,rw,m,n,k", RINGS + ROTATED)
def test_rings(ops, dev, gated, ar, rw, m, n, k):
    _check(ops, dev, m, n, k, ("silu" if k < 1000 else "gelu_tanh") if gated else None, torch.bfloat16 if rw % 16 else torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("gated,m,rows,n,k", DOT)
def test_dot(ops, dev, gated, m, rows, n, k):
    _check(ops, dev, m, n, k, ("silu" if m % 2 else "gelu_tanh") if gated else None, torch.bfloat16 if m % 2 else torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("tile,parts", SPLIT)
def test_split_tiles(ops, dev, tile, parts, gated):
    m, n, k = SPLIT[tile, parts]
    _check(ops, dev, m, n // (1 + gated), k, "silu" if gated else None, torch.bfloat16 if parts % 2 else torch.float16)


# A workspace for fewer parts than the planner would take: (rows, rows of b, K, its parts)
SHORT = [(66, 5442, 4944, 4), (65, 70, 8208, 12), (500, 4090, 14320, 4)]


def _rooms(m, n, k, gated):
    """Bytes to give, and the parts that they hold at most."""
    lib = cabi.load()
    size = lib.cek_gemm_int8_a8w8_glu_workspace_size if gated else lib.cek_gemm_int8_a8w8_workspace_size
    full, one = size(m, n // (1 + gated), k), 4 * m * n
    return full, [(b, b // one) for b in (full, full - 16, full * 3 // 4, full // 2, 2 * one + 15, 2 * one - 16, 0)]


@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("m,n,k,most", SHORT)
def test_parts_fit_their_workspace(m, n, k, most, gated):
    full, rooms = _rooms(m, n, k, gated)
    parts = [cabi.load().cek_gemm_int8_plan(m, n // (1 + gated), k, gated, b) % 16 for b, _ in rooms]
    assert parts[0] == most and parts[-1] == 1 and all(p <= max(1, room) for p, (_, room) in zip(parts, rooms))
    assert any(1 < p < most for p in parts)            # less room, still a split


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("m,n,k,most", SHORT)
def test_workspaces_that_are_too_small(dev, m, n, k, most, gated):
    """The same bits from any workspace, and nothing written behind its end."""
    lib = cabi.load()
    g = torch.Generator(device=dev).manual_seed(m)
    a, b = (torch.randint(-128, 128, (r, k), generator=g, dtype=torch.int8, device=dev) for r in (m, n))
    sa, sb = torch.rand(m, generator=g, device=dev) * 0.01, torch.rand(n, generator=g, device=dev) * 1e-4
    want = None
    full, rooms = _rooms(m, n, k, gated)
    for room, _ in reversed(rooms):
        ws = torch.full((full + 4096,), 0x5A, dtype=torch.uint8, device=dev)
        y = torch.full((m, n // (1 + gated)), math.nan, dtype=torch.bfloat16, device=dev)
        ptrs = [cabi.ptr(t) for t in (a, sa, b, sb, y)]
        if gated:
            rc = lib.cek_gemm_int8_a8w8_glu(*ptrs, m, n // 2, k, cabi.CEK_SILU, cabi.CEK_BF16, cabi.ptr(ws), room, cabi.stream_ptr())
        else:
            rc = lib.cek_gemm_int8_a8w8(*ptrs, m, n, k, cabi.CEK_BF16, cabi.ptr(ws), room, cabi.stream_ptr())
        cabi.check(rc)
        want = y if want is None else want               # none: one part
        assert not torch.isnan(y).any() and torch.equal(y, want) and (ws[room:] == 0x5A).all(), room
