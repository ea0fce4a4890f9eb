"""The 4-bit cache's oracle, pinned against closed forms and hand-made cases (CPU)."""

import math

import pytest
import torch

from oracle import kv4


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantise_error_is_half_a_step(dtype):
    """|x - value| <= s / 2 (and a bit: s is bf16, so the ends lie up to 7.5 * 2^-9 steps outside the codes)."""
    x = (torch.randn(200, 128, generator=torch.Generator().manual_seed(1)) * 3 + 1).to(dtype)
    c, s, m = kv4.quantise(x)
    err = (x.double() - kv4.values(c, s, m)).abs()
    assert (err <= s.double()[:, None] * (0.5 + 7.5 * 2.0 ** -9 + 1e-6)).all()
    assert c.min() == 0 and c.max() == 15


def test_quantise_special_rows():
    x = torch.tensor([[2.5] * 64, [0.0] * 64, [0.0] * 63 + [math.inf], [0.0] * 63 + [math.nan], [1e-38, -1e-38] * 32,
                      [3e38, -3e38] * 32])
    c, s, m = kv4.quantise(x)
    v = kv4.values(c, s, m)
    assert (v[0] == 2.5).all() and (v[1] == 0).all()
    assert v[2].isnan().all() and v[3].isnan().all()
    assert (s[4] == 0) and (v[4].abs() < 1e-38).all()
    assert (v[5] / x[5].double() - 1).abs().max() < 2.0 ** -8


@pytest.mark.parametrize("bs,hd", [(16, 64), (32, 128), (256, 256)])
def test_put_get_round_trip_and_neighbours(bs, hd):
    g = torch.Generator().manual_seed(2)
    cache = kv4.empty(3, 2, bs, hd, fill=0)
    before = cache.clone()
    k, v = torch.randn(2, hd, generator=g), torch.randn(2, hd, generator=g)
    kv4.put(cache, bs + 5, k, v)
    for x, got in zip((k, v), kv4.get(cache, bs + 5)):
        assert torch.equal(got, kv4.values(*kv4.quantise(x)))
    # exactly hd / 2 code bytes and 4 parameter bytes a head and part, in block 1 alone
    assert torch.equal(cache[0], before[0]) and torch.equal(cache[2], before[2])
    assert int((cache[1] != before[1]).sum()) <= 2 * 2 * (hd // 2 + 4)


def test_attention_against_plain_loops():
    g = torch.Generator().manual_seed(3)
    q, k, v = torch.randn(3, 4, 8, generator=g), torch.randn(7, 2, 8, generator=g), torch.randn(7, 2, 8, generator=g)
    for window in (0, 2):
        out = kv4.attention(q, k, v, 0.5, window)
        for i in range(3):
            p = 4 + i
            lo = max(0, p - window + 1) if window else 0
            for h in range(4):
                w = [math.exp(0.5 * float(q[i, h].double() @ k[j, h // 2].double())) for j in range(lo, p + 1)]
                ref = sum(a * v[j, h // 2].double() for a, j in zip(w, range(lo, p + 1))) / sum(w)
                assert torch.allclose(out[i, h], ref, rtol=1e-12)


def test_tables_blocks_are_conserved():
    """Random steps: every block is free or in exactly one request's row; slots are distinct; a dropped request
    returns all it had."""
    rng = torch.Generator().manual_seed(4)
    ri = lambda hi, n: torch.randint(0, hi, (n,), generator=rng).tolist()  # noqa: E731
    R, width, bs, blocks, T = 6, 9, 16, 30, 200
    ring, state = list(range(blocks)), [0, blocks]
    tables, lens = [[-1] * width for _ in range(R)], [0] * R
    refused = 0
    for _ in range(200):
        keep = [0 if z == 0 else max(0, n - d) for z, n, d in zip(ri(6, R), lens, ri(5, R))]
        q = ri(50, R)
        old = lens
        lens, state, cu, slots, pos, status = kv4.block_tables(old, keep, q, bs, ring, state, tables, T)
        refused += sum(s != 0 for s in status)
        used = [b for r, n in enumerate(lens) for b in tables[r][:-(-n // bs)]]
        free = [ring[(state[0] + i) % blocks] for i in range(state[1])]
        assert sorted(used + free) == list(range(blocks))
        real = [s for s in slots if s >= 0]
        assert len(set(real)) == len(real) == cu[-1]
    assert refused > 0
