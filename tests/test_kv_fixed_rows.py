"""CPU: steps whose refused requests keep their rows -- the oracle against the closed-up form, and the C entry's refusals."""

import pytest
import torch

from esimd_learning_amd import cabi
from oracle import kv4
from test_cabi_kv4 import INVALID, N, TABLES, UNSUPPORTED, _call


def test_oracle_only_rows_differ():
    """But for requests that its rows cost their place (status 3), who gets what is the same; a granted request's slots
    stand where the wishes before it put them, all else is padding."""
    rng = torch.Generator().manual_seed(6)
    ri = lambda hi, n: torch.randint(0, hi, (n,), generator=rng).tolist()  # noqa: E731
    R, width, bs, blocks, T = 6, 4, 16, 18, 400
    ring, state = list(range(blocks)), [0, blocks]
    tables, lens, seen = [[-1] * width for _ in range(R)], [0] * R, set()
    for _ in range(200):
        keep = [0 if z == 0 else max(0, n - d) for z, n, d in zip(ri(6, R), lens, ri(5, R))]
        q = [n - 3 for n in ri(40, R)]
        ring2, tables2 = list(ring), [list(t) for t in tables]
        a = kv4.block_tables(lens, keep, q, bs, ring, state, tables, T)
        b = kv4.block_tables(lens, keep, q, bs, ring2, state, tables2, T, fixed_rows=True)
        assert ring == ring2 and tables == tables2 and a[0] == b[0] and a[1] == b[1] and a[5] == b[5]
        rest, at = set(range(T)), 0
        for r in range(R):
            assert b[2][r] == at
            at += max(q[r], 0)
            if b[5][r] == 0:
                assert b[3][b[2][r]:at] == a[3][a[2][r]:a[2][r + 1]] and b[4][b[2][r]:at] == a[4][a[2][r]:a[2][r + 1]]
                rest -= set(range(b[2][r], at))
        assert b[2][R] == at and all(b[3][t] == -1 and b[4][t] == 0 for t in rest)
        seen |= set(b[5])
        lens, state = a[0], a[1]
    assert seen == {0, 1, 2}


def test_oracle_more_rows_than_there_are():
    cu, slots, _, status = kv4.block_tables([0, 0, 0], [0] * 3, [3, 40, 2], 16, [0, 1], [0, 2], [[-1], [-1], [-1]], 8,
                                            fixed_rows=True)[2:]
    assert cu == [0, 3, 8, 8] and status == [0, 2, 3] and slots == [0, 1, 2] + [-1] * 5


@pytest.mark.parametrize("change,rc", [
    *[({n: N}, INVALID) for n in ("lens", "keep", "q", "ring", "state", "tables", "lens_out", "state_out", "cu", "slots",
                                  "pos", "status")],
    (dict(R=-1), INVALID), (dict(R=4097), UNSUPPORTED), (dict(bs=24), UNSUPPORTED), (dict(blocks=0), INVALID),
    (dict(ts=3), INVALID), (dict(T=-1), INVALID), (dict(T=2 ** 31), INVALID),
])
def test_c_refusals(change, rc):
    assert _call(cabi.load().cek_kv_block_tables_fixed_rows, list(TABLES), TABLES, change) == rc
