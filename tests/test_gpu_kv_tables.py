"""GPU: block tables, slots and positions of a step against plain loops; all of it whole numbers, so equal."""

import sys

import pytest
import torch

from oracle import kv4

pytestmark = pytest.mark.gpu


class State:
    def __init__(self, R, width, bs, blocks, T, dev, head=0, in_place=False):
        self.bs, self.T, self.R = bs, T, R
        self.h_ring = [(i - head) % blocks for i in range(blocks)]
        self.h_state = [head, blocks]
        self.h_tables = [[-1] * width for _ in range(R)]
        self.h_lens = [0] * R
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        self.dev = dev
        self.ring, self.state, self.tables = i32(self.h_ring), i32(self.h_state), i32(self.h_tables).view(R, width)
        self.lens = i32(self.h_lens)
        self.lens_out, self.state_out = (self.lens, self.state) if in_place else (i32(self.h_lens), i32([0, 0]))
        self.cu, self.status = i32([9] * (R + 1)), i32([9] * R)
        self.slots, self.pos = (torch.full((T,), 9, dtype=torch.int64, device=dev) for _ in range(2))

    def step(self, ops, keep, q):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)  # noqa: E731
        ops.esimd_kv_block_tables(self.lens, i32(keep), i32(q), self.bs, self.ring, self.state, self.tables, self.lens_out,
                                  self.state_out, self.cu, self.slots, self.pos, self.status)
        ref = kv4.block_tables(self.h_lens, keep, q, self.bs, self.h_ring, self.h_state, self.h_tables, self.T)
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
@pytest.mark.parametrize("R,width,bs,blocks,T", [(1, 4, 16, 3, 40), (7, 9, 16, 33, 150), (64, 6, 32, 300, 3000),
                                                 (300, 5, 64, 1200, 9000), (1100, 3, 16, 2500, 20000), (4096, 2, 16, 8000, 70000)])
def test_random_steps(ops, dev, R, width, bs, blocks, T, in_place):
    """Requests that grow, drop tokens, end, start over, wish for more than there is, and lengths out of range."""
    print("tables", R, width, bs, blocks, T, in_place, flush=True)
    sys.stdout.flush()
    g = torch.Generator().manual_seed(R)
    ri = lambda lo, hi: torch.randint(lo, hi, (R,), generator=g).tolist()  # noqa: E731
    s = State(R, width, bs, blocks, T, dev, head=blocks - 2, in_place=in_place)
    seen = set()
    for i in range(8):
        keep = [0 if z == 0 else n - d for z, n, d in zip(ri(0, 5), s.h_lens, ri(-2, 4))]
        big = width * bs // 2 if i < 6 else 3 * width * bs
        q = [x if z else 0 for x, z in zip(ri(-1, big), ri(0, 4))]
        seen |= set(s.step(ops, keep, q)[5])
    assert 0 in seen and (R < 7 or len(seen) > 1)


def test_decode_across_block_ends(ops, dev):
    s = State(3, 4, 16, 12, 5, dev, in_place=True)
    s.step(ops, [0, 0, 0], [1, 1, 1])
    for i in range(40):
        s.step(ops, list(s.h_lens), [1, 1, 0])
    assert s.h_lens == [41, 41, 1]
    s.step(ops, [0, 41, 1], [0, 0, 0])
    assert s.h_state[1] == 12 - 3 - 1


def test_impossible_state_stays_in_bounds(ops, dev):
    """Lengths of more blocks than there are, ring states out of range: nothing outside the arrays is touched."""
    R, width, blocks = 6, 50, 16
    guard = torch.full((3, 64 + blocks), 123, dtype=torch.int32, device=dev)
    ring = guard[1, 32:32 + blocks]
    ring.copy_(torch.arange(blocks))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for state in ((0, 0), (5, 16), (-7, 99), (10 ** 9, -4)):
        for lens, keep, q in (((800,) * 6, (0,) * 6, (0,) * 6), ((2 ** 31 - 1,) * 6, (5,) * 6, (2 ** 31 - 1, 1, 0, 40, 9, 3)),
                              ((-5,) * 6, (3,) * 6, (16, 0, 17, -1, 100, 2 ** 31 - 1))):
            tables = torch.zeros(R, width, dtype=torch.int32, device=dev)
            cu, out, so = i32(*[0] * 7), i32(*[0] * 6), i32(0, 0)
            slots, pos = (torch.zeros(20, dtype=torch.int64, device=dev) for _ in range(2))
            ops.esimd_kv_block_tables(i32(*lens), i32(*keep), i32(*q), 16, ring, i32(*state), tables, out, so, cu, slots,
                                      pos, i32(*[0] * 6))
            head, count = so.tolist()
            assert 0 <= head < blocks and 0 <= count <= blocks
            assert (guard[0] == 123).all() and (guard[2] == 123).all()
            assert (guard[1, :32] == 123).all() and (guard[1, 32 + blocks:] == 123).all()
            assert 0 <= int(cu.max()) <= 20 and int(out.min()) >= 0


def test_no_new_tokens_and_no_requests(ops, dev):
    s = State(2, 3, 16, 6, 0, dev)
    s.step(ops, [0, 0], [0, 0])
    s = State(1, 3, 16, 6, 4, dev)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    ops.esimd_kv_block_tables(none, none, none, 16, s.ring, s.state, s.tables[:0], none.clone(), s.state_out, s.cu[:1],
                              s.slots, s.pos, none.clone())
    assert s.state_out.tolist() == [0, 6] and s.cu[0] == 0
    assert s.slots.tolist() == [-1] * 4 and s.pos.tolist() == [0] * 4


def test_table_rows_apart(ops, dev):
    """block_tables as columns of a wider buffer: the rest stays."""
    s = State(5, 4, 16, 20, 60, dev, in_place=True)
    buf = torch.full((5, 11), 77, dtype=torch.int32, device=dev)
    buf[:, 3:7] = s.tables
    s.tables = buf[:, 3:7]
    s.step(ops, [0] * 5, [5, 17, 0, 1, 20])
    s.step(ops, [3, 17, 0, 0, 5], [4, 17, 3, 0, 1])
    assert (buf[:, :3] == 77).all() and (buf[:, 7:] == 77).all()


def test_graph_replays_advance(ops, dev):
    """A captured in-place step, replayed: every replay is the next step."""
    R, bs = 4, 16
    s = State(R, 8, bs, 40, 12, dev, in_place=True)
    s.step(ops, [0] * R, [3, 2, 3, 1])
    q = torch.tensor([1, 2, 3, 1], dtype=torch.int32, device=dev)
    keep = s.lens.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        keep.copy_(s.lens)
        ops.esimd_kv_block_tables(s.lens, keep, q, bs, s.ring, s.state, s.tables, s.lens, s.state, s.cu, s.slots, s.pos,
                                  s.status)
    for _ in range(20):
        g.replay()
        torch.randn(100, device=dev).sum().item()
        torch.cuda.synchronize()
        ref = kv4.block_tables(s.h_lens, s.h_lens, q.tolist(), bs, s.h_ring, s.h_state, s.h_tables, s.T)
        s.h_lens, s.h_state = ref[0], ref[1]
        assert s.lens.tolist() == ref[0] and s.state.tolist() == ref[1] and s.slots.tolist() == ref[3]
        assert s.tables.tolist() == s.h_tables and s.pos.tolist() == ref[4] and s.ring.tolist() == s.h_ring


def test_refusals(ops, dev):
    s = State(3, 4, 16, 12, 8, dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    keep, q = i32(0, 0, 0), i32(1, 1, 1)
    base = dict(lens=s.lens, keep=keep, q=q, bs=16, ring=s.ring, state=s.state, tables=s.tables, lens_out=s.lens_out,
                state_out=s.state_out, cu=s.cu, slots=s.slots, pos=s.pos, status=s.status)

    def call(**k):
        a = {**base, **k}
        ops.esimd_kv_block_tables(*[a[n] for n in base])

    call()
    for k, text in [(dict(bs=24), "power of two"), (dict(bs=8), "power of two"), (dict(bs=512), "power of two"),
                    (dict(q=q.long()), "q_lens"), (dict(q=q[:2]), "q_lens"), (dict(cu=s.cu[:3]), "cu_q"),
                    (dict(pos=s.pos[:4]), "positions"), (dict(slots=s.slots.int()), "slot_mapping"),
                    (dict(ring=s.ring[:0]), "free_ring"), (dict(tables=s.tables[:2]), "block_tables"),
                    (dict(tables=s.tables.t()), "block_tables"), (dict(lens_out=keep), "overlaps"),
                    (dict(status=s.lens_out), "overlap"), (dict(state_out=s.ring[:2]), "overlap"),
                    (dict(keep=keep.cpu()), "GPU"), (dict(lens=torch.zeros(4097, dtype=torch.int32, device=dev)), "4096")]:
        with pytest.raises(RuntimeError, match=text):
            call(**k)
