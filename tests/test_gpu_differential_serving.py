"""The differential operators as a server runs them: every step advances the
block tables on the GPU, appends the new tokens' keys and values at the slots
that the step gave out, and attends with the lengths and tables it left behind,
nothing read back in between. Against the allocator run call by call and the
float64 restatement, eagerly and as one captured graph."""
import random

import pytest
import torch

from cloverinfer_amd import kernels
from oracle import differential as od
from tests.test_gpu_differential import DECODE_BITS, PREFILL_BITS, _check

pytestmark = pytest.mark.gpu
DEV = "cuda"
OUT_SCALE, LAM, PAD = 0.4, 0.35, 7


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Server:
    """Device state of a cache of one layer, and on the host the allocator's
    state and every row's keys and values."""

    def __init__(self, rows, width, num_blocks, bs, hq, hkv, d, dtype, seed, reserve=1):
        self.bs, self.width, self.num_blocks, self.dtype = bs, width, num_blocks, dtype
        self.hq, self.hkv, self.d, self.reserve = hq, hkv, d, reserve
        self.g = torch.Generator().manual_seed(seed)
        self.table = [[-1] * width for _ in range(rows)]
        self.held, self.lens = [0] * rows, [0] * rows
        self.stack = list(range(num_blocks))
        random.Random(seed).shuffle(self.stack)
        self.keys = [torch.zeros(0, hkv, d, dtype=dtype) for _ in range(rows)]
        self.values = [k.clone() for k in self.keys]
        # what no token was written to must not be read
        self.pools = [torch.full((num_blocks, bs, hkv, d), float("nan"), dtype=dtype, device=DEV)
                      for _ in range(2)]
        self.bt, self.bh, self.cl = _i32(self.table), _i32(self.held), _i32(self.lens)
        self.free, self.nfree, self.status = _i32(self.stack), _i32([num_blocks]), _i32([9])
        self.qsl = torch.zeros(rows + 1, dtype=torch.int32, device=DEV)
        self.weight = torch.rand(d, generator=self.g) + 0.5

    def rand(self, n, heads):
        return torch.randn(n, heads, self.d, generator=self.g).to(self.dtype)

    def host_step(self, new, key, value, slots):
        """The step on the host: what the device state must be after it."""
        want = od.advance(self.table, self.held, self.lens, new, self.stack, self.bs, slots,
                          self.width, self.num_blocks, self.reserve)
        status, self.table, self.held, self.lens, self.stack, want_slots, qsl = want
        if status == od.TABLES_OK:
            for r, n in enumerate(new):
                if n < 0:
                    self.keys[r], self.values[r] = self.keys[r][:0], self.values[r][:0]
                else:
                    self.keys[r] = torch.cat([self.keys[r], key[qsl[r]:qsl[r + 1]]])
                    self.values[r] = torch.cat([self.values[r], value[qsl[r]:qsl[r + 1]]])
        return status, want_slots, qsl

    def check_state(self, status, slots, want_slots, qsl):
        assert self.status.tolist() == [status] and slots.tolist() == want_slots
        assert self.qsl.tolist() == qsl
        assert self.bt.tolist() == self.table and self.bh.tolist() == self.held
        assert self.cl.tolist() == self.lens
        n = len(self.stack)
        assert self.nfree.tolist() == [n] and self.free[:n].tolist() == self.stack

    def reference(self, q, r, first):
        """Rows of table row r, the first of them seeing first + 1 tokens."""
        return od.rows(q, self.keys[r], self.values[r],
                       [min(first + i + 1, len(self.keys[r])) for i in range(len(q))], LAM,
                       self.weight, out_scale=OUT_SCALE)


HEADS = [(14, 2, 256, torch.bfloat16), (28, 4, 128, torch.float16), (6, 6, 128, torch.float32)]


@pytest.mark.parametrize("hq,hkv,d,dtype", HEADS)
@pytest.mark.parametrize("bs", [16, 32])
def test_steps_of_a_server(hq, hkv, d, dtype, bs):
    s = Server(5, 1600 // bs, 160, bs, hq, hkv, d, dtype, seed=3)
    weight = s.weight.to(DEV)
    steps = [
        [300, 1, 0, 513, 40],      # prompts
        [1, 1, 77, 1, 1],          # a chunk beside decodes
        [1, 1, 1, 1, 1],           # decode
        [-1, 1, 0, -1, 1],         # two end, one waits
        [900, 1, 1, 0, 700],       # their blocks serve new prompts
        [0, 0, 0, 0, 0],
        [1, 1, 1, 1, 1],
        [200000, 0, 0, 0, 0],      # does not fit: nothing moves
        [16, -1, 31, 1, -1],
    ]
    for i, new in enumerate(steps):
        print("step", i, new, flush=True)
        fits = sum(max(n, 0) for n in new) < 4000
        t = (sum(max(n, 0) for n in new) if fits else 64) + PAD
        key, value, q = s.rand(t, hkv), s.rand(t, hkv), s.rand(t, hq)
        slots = torch.full((t,), -9, dtype=torch.int64, device=DEV)
        out = torch.full((t, hq, d), float("nan"), dtype=dtype, device=DEV)
        decode = torch.full((5, hq, d), float("nan"), dtype=dtype, device=DEV)
        kernels.advance_block_tables(s.bt, s.bh, s.cl, _i32(new), s.free, s.nfree, bs, slots,
                                     s.qsl, s.status)
        kernels.reshape_and_cache(key.to(DEV), value.to(DEV), *s.pools, slots)
        kernels.differential_prefill(out, q.to(DEV), *s.pools, s.bt, s.cl, s.qsl,
                                     max(1, min(t, max(new))), LAM, norm_weight=weight,
                                     out_scale=OUT_SCALE)
        # the decode form over the same tables: one row of each sequence
        kernels.differential_attention(decode, q[:5].to(DEV), *s.pools, s.bt, s.cl, bs, 1600, LAM,
                                       norm_weight=weight, out_scale=OUT_SCALE)
        torch.cuda.synchronize()
        status, want_slots, qsl = s.host_step(new, key, value, t)
        assert (status == od.TABLES_OK) == fits
        s.check_state(status, slots, want_slots, qsl)
        for r in range(5):
            rows = slice(qsl[r], qsl[r + 1])
            if rows.stop > rows.start:
                ref = s.reference(q[rows], r, len(s.keys[r]) - (rows.stop - rows.start))
                _check(out[rows], ref, dtype, PREFILL_BITS[dtype], f"step {i} row {r}")
            if len(s.keys[r]):
                ref = s.reference(q[r:r + 1], r, len(s.keys[r]) - 1)
                _check(decode[r:r + 1], ref, dtype, DECODE_BITS[dtype], f"step {i} decode {r}")
            else:
                assert not decode[r].any()
        assert torch.isnan(out[qsl[-1]:]).all()  # rows past the step's stay


@pytest.mark.parametrize("hq,hkv,d,dtype", HEADS)
@pytest.mark.parametrize("max_len", [512, 4096])  # one launch; balanced and merge
def test_decode_steps_as_a_graph(hq, hkv, d, dtype, max_len):
    """Capture the whole decode step once and replay it: lengths, tables and
    slots come from the step itself, new tokens are written over its inputs."""
    rows, bs = 6, 16
    s = Server(rows, 40, 80, bs, hq, hkv, d, dtype, seed=5, reserve=0)
    weight = s.weight.to(DEV)
    new = torch.zeros(rows, dtype=torch.int32, device=DEV)
    key = torch.zeros(rows, hkv, d, dtype=dtype, device=DEV)
    value, q = key.clone(), torch.zeros(rows, hq, d, dtype=dtype, device=DEV)
    slots = torch.zeros(rows, dtype=torch.int64, device=DEV)
    out = torch.zeros(rows, hq, d, dtype=dtype, device=DEV)

    def step():
        kernels.advance_block_tables(s.bt, s.bh, s.cl, new, s.free, s.nfree, bs, slots, s.qsl,
                                     s.status, reserve=0)
        kernels.reshape_and_cache(key, value, *s.pools, slots)
        kernels.differential_attention(out, q, *s.pools, s.bt, s.cl, bs, max_len, LAM,
                                       norm_weight=weight, out_scale=OUT_SCALE)

    # prompts, eagerly, with more tokens than the graph's step has
    lens = [0, 15, 16, 120, 300, 1]
    k0, v0 = s.rand(sum(lens), hkv), s.rand(sum(lens), hkv)
    slots0 = torch.zeros(sum(lens), dtype=torch.int64, device=DEV)
    kernels.advance_block_tables(s.bt, s.bh, s.cl, _i32(lens), s.free, s.nfree, bs, slots0, s.qsl,
                                 s.status, reserve=0)
    kernels.reshape_and_cache(k0.to(DEV), v0.to(DEV), *s.pools, slots0)
    torch.cuda.synchronize()
    status, want_slots, qsl = s.host_step(lens, k0, v0, sum(lens))
    s.check_state(status, slots0, want_slots, qsl)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # an idle step: no row grows
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    plans = [[1] * rows, [1] * rows, [1, 0, 1, -1, 1, 1], [1] * rows, [0, 1, 1, 1, -1, 0],
             [1] * rows]
    for i, plan in enumerate(plans):
        total = sum(max(n, 0) for n in plan)
        kn, vn, qn = s.rand(rows, hkv), s.rand(rows, hkv), s.rand(rows, hq)
        new.copy_(torch.tensor(plan, dtype=torch.int32))
        key.copy_(kn), value.copy_(vn), q.copy_(qn)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        status, want_slots, qsl = s.host_step(plan, kn, vn, rows)
        assert status == od.TABLES_OK and qsl[-1] == total
        s.check_state(status, slots, want_slots, qsl)
        for r in range(rows):
            if len(s.keys[r]):
                _check(out[r:r + 1], s.reference(qn[r:r + 1], r, len(s.keys[r]) - 1), dtype,
                       DECODE_BITS[dtype], f"replay {i} row {r}")
            else:
                assert not out[r].any()
        torch.randn(1000, device=DEV).sum().item()  # the program's own work between replays
        eager = torch.full_like(out, float("nan"))
        kernels.differential_attention(eager, q, *s.pools, s.bt, s.cl, bs, max_len, LAM,
                                       norm_weight=weight, out_scale=OUT_SCALE)
        assert torch.equal(eager, out)
