"""advance_block_tables against the reference's allocator run call by call:
tables, stack, slots and counts bit for bit, over runs of random steps, at the
sizes of the one-launch and the two-launch form, in place and out of place;
refused steps keep the state."""
import random

import pytest
import torch

from cloverinfer_amd import _native, kernels
from oracle import differential as od

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class State:
    """The device state of a cache, and the host's copy of it as lists."""

    def __init__(self, rows, width, num_blocks, block_size, order=None):
        self.bs, self.width, self.num_blocks = block_size, width, num_blocks
        self.table = [[-1] * width for _ in range(rows)]
        self.held, self.lens = [0] * rows, [0] * rows
        self.stack = list(order if order is not None else range(num_blocks))
        self.dev = [_i32(self.table).view(rows, width), _i32(self.held), _i32(self.lens)]
        self.free = torch.full((num_blocks,), -7, dtype=torch.int32, device=DEV)
        self.free[:len(self.stack)] = _i32(self.stack)
        self.num_free = _i32([len(self.stack)])
        self.status = _i32([99])

    def step(self, new, num_slots, reserve=1, in_place=True):
        rows = len(new)
        slots = torch.full((num_slots,), -9, dtype=torch.int64, device=DEV)
        qsl = torch.full((rows + 1,), -9, dtype=torch.int32, device=DEV)
        before = self.free.clone()
        old = [t.clone() for t in self.dev[1:]] + [self.num_free.clone()]
        outs = {} if in_place else {"blocks_held_out": torch.empty_like(self.dev[1]),
                                    "context_lens_out": torch.empty_like(self.dev[2]),
                                    "num_free_out": torch.empty_like(self.num_free)}
        kernels.advance_block_tables(*self.dev, _i32(new), self.free, self.num_free, self.bs, slots,
                                     qsl, self.status, reserve=reserve, **outs)
        torch.cuda.synchronize()
        if not in_place:
            for t, o in zip(self.dev[1:] + [self.num_free], old):
                assert torch.equal(t, o)
            self.dev[1:] = [outs["blocks_held_out"], outs["context_lens_out"]]
            self.num_free = outs["num_free_out"]
        want = od.advance(self.table, self.held, self.lens, new, self.stack, self.bs, num_slots,
                          self.width, self.num_blocks, reserve)
        had = len(self.stack)
        status, self.table, self.held, self.lens, self.stack, want_slots, want_qsl = want
        assert self.status.tolist() == [status]
        assert self.dev[0].tolist() == self.table
        assert self.dev[1].tolist() == self.held and self.dev[2].tolist() == self.lens
        n = len(self.stack)
        assert self.num_free.tolist() == [n] and self.free[:n].tolist() == self.stack
        assert torch.equal(self.free[max(n, had):], before[max(n, had):])
        assert slots.tolist() == want_slots and qsl.tolist() == want_qsl
        return status


@pytest.mark.parametrize("rows,bs,big", [(1, 16, 40), (7, 4, 30), (130, 16, 200), (1500, 16, 9),
                                         (64, 1, 20), (300, 32, 700)])
@pytest.mark.parametrize("in_place", [True, False])
def test_random_steps(rows, bs, big, in_place):
    r = random.Random(rows * 100 + bs)
    width = 3 * big // bs + 4
    num_blocks = rows * width * 3 // 4 + 1
    order = list(range(num_blocks))
    r.shuffle(order)
    st = State(rows, width, num_blocks, bs, order)
    seen = set()
    for i in range(14):
        new = []
        for c in st.lens:
            u = r.random()
            room = max(0, width * bs - c - 2)
            new.append(-r.randint(1, 5) if u < 0.15 else 0 if u < 0.3 else
                       min(1, room) if u < 0.6 else min(room, r.randint(1, big)))
        total = sum(max(0, n) for n in new)
        pad = r.choice([0, 3, 9000])
        print(f"step {i}: rows {rows} bs {bs} tokens {total} + {pad}", flush=True)
        seen.add(st.step(new, total + pad, reserve=r.choice([0, 1, 1, 20]), in_place=in_place))
    assert od.TABLES_OK in seen


@pytest.mark.parametrize("tokens", [8192, 8193, 300000])
def test_admission_and_release_of_long_rows(tokens):
    rows = 5
    per = tokens // rows
    st = State(rows, per // 16 + 2, tokens // 16 + 20, 16)
    new = [per] * (rows - 1) + [tokens - per * (rows - 1)]
    assert st.step(new, tokens) == od.TABLES_OK
    assert st.step([-1, 0, 1, -1, 1], tokens) == od.TABLES_OK
    assert st.step([3, -1, -1, per // 2, 0], tokens) == od.TABLES_OK


@pytest.mark.parametrize("slots", [128, 9000])
def test_refused_steps_keep_the_state(slots):
    st = State(4, 6, 12, 16)
    assert st.step([40, 17, 0, 1], slots) == od.TABLES_OK       # 3 + 2 + 1 blocks
    assert st.step([0, 0, 0, 95], slots) == od.TABLES_OK        # 5 more: row 3 full, 1 left
    assert st.step([0, 0, 32, 0], slots) == od.TABLES_NO_BLOCKS
    assert st.step([-1, 0, 0, 1], slots) == od.TABLES_ROW_FULL
    assert st.step([-1, 0, 32, 0], slots) == od.TABLES_OK       # served by the ended row's blocks
    assert st.step([60, 10, 0, 0], 12) == od.TABLES_NO_BLOCKS
    assert st.step([12, 1, 0, 0], 12) == od.TABLES_NO_SLOTS
    assert st.step([12, 0, 0, 0], 12) == od.TABLES_OK
    for field, value in ((1, [7, 0, 0, 0]), (1, [-1, 2, 3, 6]), (2, [-1, 17, 32, 96]),
                         (2, [500, 17, 32, 96])):
        keep = st.dev[field].clone(), list((st.held, st.lens)[field - 1])
        st.dev[field].copy_(_i32(value))
        (st.held, st.lens)[field - 1][:] = value
        assert st.step([1, 0, 0, 0], slots) == od.TABLES_BAD_STATE
        st.dev[field].copy_(keep[0])
        (st.held, st.lens)[field - 1][:] = keep[1]


@pytest.mark.parametrize("count", [-1, 13, 2 ** 31 - 1])
def test_a_stack_that_cannot_be_is_refused(count):
    st = State(2, 4, 12, 16)
    st.step([20, 0], 32)
    st.num_free.fill_(count)
    before = [t.clone() for t in st.dev] + [st.free.clone()]
    slots = torch.zeros(32, dtype=torch.int64, device=DEV)
    qsl = torch.zeros(3, dtype=torch.int32, device=DEV)
    kernels.advance_block_tables(*st.dev, _i32([-1, 5]), st.free, st.num_free, 16, slots, qsl,
                                 st.status)
    assert st.status.tolist() == [od.TABLES_BAD_STATE] and st.num_free.tolist() == [count]
    assert all(torch.equal(a, b) for a, b in zip(before, st.dev + [st.free]))
    assert (slots == -1).all() and (qsl == 0).all()


def test_lengths_near_the_type_s_end():
    """Sums past 32 bits are refused, not wrapped."""
    st = State(3, 4, 12, 16)
    assert st.step([2 ** 31 - 1, 2 ** 31 - 1, 1], 64) == od.TABLES_NO_BLOCKS
    assert st.step([-2 ** 31, 5, 1], 64) == od.TABLES_OK


def test_no_rows():
    st = State(0, 4, 12, 16)
    assert st.step([], 5) == od.TABLES_OK


@pytest.mark.parametrize("tokens", [64, 9000])
def test_graph_replays_advance_the_state(tokens):
    """A captured step replayed: each replay is one more step, with eager steps
    between."""
    rows, st = 6, State(6, 40, 200, 16)
    st.step([100, 3, 0, 17, 31, 1], 9000)
    new = _i32([1, 1, 0, 1, 2, 1])
    slots = torch.empty(tokens, dtype=torch.int64, device=DEV)
    qsl = torch.empty(rows + 1, dtype=torch.int32, device=DEV)

    def call():
        kernels.advance_block_tables(*st.dev, new, st.free, st.num_free, 16, slots, qsl, st.status)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(40):
        step = [1, 1, 0, 1, 2, 1] if i % 7 else [-1, 5, 0, 1, 1, 1]
        new.copy_(_i32(step))
        graph.replay()
        torch.cuda.synchronize()
        want = od.advance(st.table, st.held, st.lens, step, st.stack, 16, tokens, 40, 200)
        status, st.table, st.held, st.lens, st.stack, want_slots, want_qsl = want
        assert st.status.tolist() == [status] and slots.tolist() == want_slots, i
        assert st.dev[0].tolist() == st.table and qsl.tolist() == want_qsl
        if i % 5 == 2:
            st.step([0, 0, 1, 0, 0, 0], 9000)


def test_native_argument_block_is_the_python_one(monkeypatch):
    """The native host code fills the block that the Python checks fill, in
    place and out of place, and leaves what they refuse to them."""
    n = 5
    t = [_i32([[-1] * 3] * n), _i32([0] * n), _i32([0] * n), _i32([1] * n), _i32(list(range(9))),
         _i32([9]), 16, torch.zeros(n, dtype=torch.int64, device=DEV), _i32([0] * (n + 1)),
         _i32([0]), 1]
    outs = [torch.empty_like(t[1]), torch.empty_like(t[2]), torch.empty_like(t[5])]
    real = kernels._filled
    for o in (outs, [t[1], t[2], t[5]]):
        assert real("fill_tables_args", _native.TablesArgs(), *t, *o) is not None
        native = bytes(kernels._tables_args(*t, *o))
        monkeypatch.setattr(kernels, "_filled", lambda *a: None)
        assert bytes(kernels._tables_args(*t, *o)) == native
        monkeypatch.setattr(kernels, "_filled", real)
    wrong = {0: t[0].long(), 1: t[1][:4], 2: t[2].cpu(), 3: t[3][::2], 4: t[4][None], 5: _i32([1, 2]),
             7: t[7].int(), 8: t[8][1:], 9: t[9][:0]}
    for i, w in wrong.items():
        bad = list(t)
        bad[i] = w
        assert real("fill_tables_args", _native.TablesArgs(), *bad, *outs) is None, i
        with pytest.raises((ValueError, RuntimeError)):
            kernels._tables_args(*bad, *outs)


@pytest.mark.parametrize("new", [[2 ** 31 - 1, 2 ** 31 - 1, 2], [2 ** 31 - 1] * 130,
                                 [0, 2 ** 31 - 1] * 700])
@pytest.mark.parametrize("bs", [1, 16])
def test_sums_past_32_bits_are_refused(new, bs):
    """Totals that would wrap to a small number: the step is refused for what
    it asks (the allocator runs out of blocks), and nothing moves."""
    s = State(len(new), 4, 50, bs)
    assert s.step(new, 64, reserve=0) == od.TABLES_NO_BLOCKS
    assert s.step([1] * min(len(new), 40) + [0] * max(0, len(new) - 40), 64,
                  in_place=False, reserve=0) == od.TABLES_OK
