"""GPU: block tables of steps whose refused requests keep their rows, against plain loops; whole numbers, so equal."""

import pytest
import torch

from oracle import kv4
from test_gpu_kv_tables import State

pytestmark = pytest.mark.gpu


class Fixed(State):
    def step(self, ops, keep, q):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)  # noqa: E731
        ops.esimd_kv_block_tables(self.lens, i32(keep), i32(q), self.bs, self.ring, self.state, self.tables, self.lens_out,
                                  self.state_out, self.cu, self.slots, self.pos, self.status, fixed_rows=True)
        ref = kv4.block_tables(self.h_lens, keep, q, self.bs, self.h_ring, self.h_state, self.h_tables, self.T, True)
        got = (self.lens_out, self.state_out, self.cu, self.slots, self.pos, self.status)
        for name, a, b in zip(("lens", "state", "cu", "slots", "positions", "status"), got, ref):
            assert a.tolist() == b, name
        assert self.tables.tolist() == self.h_tables and self.ring.tolist() == self.h_ring
        self.h_lens, self.h_state = ref[0], ref[1]
        if self.lens_out is not self.lens:
            self.lens.copy_(self.lens_out)
            self.state.copy_(self.state_out)
        return ref


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("R,width,bs,blocks,T", [(1, 4, 16, 3, 40), (7, 9, 16, 33, 250), (64, 6, 32, 300, 4000),
                                                 (300, 5, 64, 1200, 9000), (4096, 2, 16, 8000, 70000)])
def test_random_steps(ops, dev, R, width, bs, blocks, T, in_place):
    """Growth, rollbacks, ends, and wishes beyond the blocks, the tables and the rows; one launch and two."""
    print("fixed rows", R, width, bs, blocks, T, in_place, flush=True)
    g = torch.Generator().manual_seed(R + 1)
    ri = lambda lo, hi: torch.randint(lo, hi, (R,), generator=g).tolist()  # noqa: E731
    s = Fixed(R, width, bs, blocks, T, dev, head=blocks - 2, in_place=in_place)
    seen = set()
    for i in range(8):
        keep = [0 if z == 0 else n - d for z, n, d in zip(ri(0, 5), s.h_lens, ri(-2, 4))]
        big = width * bs // 2 if i < 6 else 3 * width * bs
        q = [x if z else 0 for x, z in zip(ri(-1, big), ri(0, 4))]
        if i == 7:
            q[0] = 2 ** 31 - 1
        seen |= set(s.step(ops, keep, q)[5])
    assert {0, 2, 3} <= seen or R == 1


def test_nobody_refused_is_the_other_form(ops, dev):
    a, b = State(3, 4, 16, 12, 20, dev), Fixed(3, 4, 16, 12, 20, dev)
    for keep, q in (([0, 0, 0], [5, 0, 12]), ([5, 0, 7], [1, 16, 2]), ([0, 16, 9], [0, 1, 1])):
        assert a.step(ops, keep, q) == b.step(ops, keep, q)
