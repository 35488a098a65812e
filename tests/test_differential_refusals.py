"""What differential attention and the block tables' step refuse on the host,
on CPU tensors (with the device check alone taken out) and through the C ABI
without a GPU; and the float64 restatements on their own."""
import ctypes
import types

import pytest
import torch

from cloverinfer_amd import _native, kernels
from oracle import blocks as ob
from oracle import differential as od


@pytest.fixture
def cpu_tensors(monkeypatch):
    monkeypatch.setattr(kernels, "_require_device", lambda *t: t[0].device)

    def launched(*a):
        raise AssertionError("the call was not refused")

    monkeypatch.setattr(kernels, "_stream", launched)


def decode_tensors(dtype=torch.bfloat16, pool=None, n=3, hq=8, hkv=2, d=128, bs=16):
    q = torch.zeros(n, hq, d, dtype=dtype)
    k = torch.zeros(6, bs, hkv, d).to(pool or dtype)
    return [torch.empty_like(q), q, k, k.clone(), torch.zeros(n, 2, dtype=torch.int32),
            torch.ones(n, dtype=torch.int32)]


@pytest.mark.parametrize("lam", [torch.zeros(8, dtype=torch.float64), torch.zeros(7),
                                 torch.zeros(2, 8), torch.zeros(3, 8, dtype=torch.bfloat16),
                                 torch.zeros(3, 8, 1)])
def test_lambda_shapes(cpu_tensors, lam):
    t = decode_tensors()
    with pytest.raises(ValueError, match="lam"):
        kernels.differential_attention(*t, 16, 32, lam)
    with pytest.raises(ValueError, match="lam"):
        kernels.differential_prefill(*t, torch.arange(4, dtype=torch.int32), 1, lam)


@pytest.mark.parametrize("weight", [torch.zeros(64), torch.zeros(128, dtype=torch.bfloat16),
                                    torch.zeros(256)[::2], torch.zeros(1, 128)])
def test_norm_weight(cpu_tensors, weight):
    t = decode_tensors()
    with pytest.raises(ValueError, match="norm_weight"):
        kernels.differential_attention(*t, 16, 32, 0.5, norm_weight=weight)
    with pytest.raises(ValueError, match="norm_weight"):
        kernels.differential_prefill(*t, torch.arange(4, dtype=torch.int32), 1, 0.5,
                                     norm_weight=weight)


def test_tensors_on_another_device_are_refused(cpu_tensors):
    t = decode_tensors()
    for kw in ({"lam": torch.zeros(8, device="meta")},
               {"lam": 0.5, "norm_weight": torch.zeros(128, device="meta")}):
        with pytest.raises(ValueError, match="must be on"):
            kernels.differential_attention(*t, 16, 32, **kw)


def test_fp8_pools_need_scales_and_are_for_decode(cpu_tensors, monkeypatch):
    t = decode_tensors(pool=kernels.FP8)
    with pytest.raises(ValueError):
        kernels.differential_prefill(*t, torch.arange(4, dtype=torch.int32), 1, 0.5)
    monkeypatch.setattr(kernels, "_stream", lambda dev: 0)
    with pytest.raises(ValueError, match="k_scale"):
        kernels.differential_attention(*t, 16, 32, 0.5)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="HIP device"):
        kernels.differential_attention(*decode_tensors(), 16, 32, 0.5)
    with pytest.raises(RuntimeError, match="HIP device"):
        kernels.differential_prefill(*decode_tensors(), torch.arange(4, dtype=torch.int32), 1, 0.5)
    with pytest.raises(RuntimeError, match="HIP device"):
        kernels.advance_block_tables(**tables())


def tables(rows=3, width=4, num_blocks=8, tokens=5):
    def i32(*shape):
        return torch.zeros(*shape, dtype=torch.int32)

    return dict(block_tables=i32(rows, width), blocks_held=i32(rows), context_lens=i32(rows),
                new_lens=i32(rows), free_blocks=i32(num_blocks), num_free=i32(1), block_size=16,
                slot_mapping=torch.zeros(tokens, dtype=torch.int64), query_start_loc=i32(rows + 1),
                status=i32(1))


@pytest.mark.parametrize("name,value", [
    ("block_tables", torch.zeros(3, 4)),
    ("block_tables", torch.zeros(4, 3, dtype=torch.int32).t()),
    ("blocks_held", torch.zeros(2, dtype=torch.int32)),
    ("context_lens", torch.zeros(3, dtype=torch.int64)),
    ("new_lens", torch.zeros(6, dtype=torch.int32)[::2]),
    ("free_blocks", torch.zeros(8, dtype=torch.int64)),
    ("num_free", torch.zeros(2, dtype=torch.int32)),
    ("slot_mapping", torch.zeros(5, dtype=torch.int32)),
    ("slot_mapping", torch.zeros(10, dtype=torch.int64)[::2]),
    ("query_start_loc", torch.zeros(3, dtype=torch.int32)),
    ("status", torch.zeros(1)),
    ("blocks_held_out", torch.zeros(4, dtype=torch.int32)),
    ("context_lens_out", torch.zeros(3)),
    ("num_free_out", torch.zeros(0, dtype=torch.int32)),
])
def test_tables_tensors(cpu_tensors, name, value):
    with pytest.raises(ValueError):
        kernels.advance_block_tables(**{**tables(), name: value})


def _decode_args(head_dim=128, block_size=16, dtype=_native.CLV_BF16, max_len=64):
    a = _native.DecodeArgs()
    a.out = a.q = a.k_cache = a.v_cache = 0x1000
    a.block_tables = a.context_lens = 0x2000
    a.q_stride_seq, a.q_stride_head = 28 * 256, 256
    a.out_stride_seq, a.out_stride_head = 28 * 256, 256
    a.kv_stride_block, a.kv_stride_token, a.kv_stride_head = 16 * 4 * 256, 4 * 256, 256
    a.num_seqs, a.num_heads, a.num_kv_heads, a.head_dim = 0, 28, 4, head_dim
    a.block_size, a.max_blocks_per_seq, a.max_context_len, a.num_blocks = block_size, 4, max_len, 16
    a.dtype, a.scale = dtype, 0.125
    return a


def _diff():
    d = _native.DiffArgs()
    d.lambda_value, d.norm_eps, d.out_scale = 0.5, 1e-5, 1.0
    return d


def test_decode_arguments(native_lib):
    def call(a, d, ks=None, vs=None):
        return native_lib.clv_diff_decode(a, d, ks, vs, 0, None, 0, None)

    assert call(_decode_args(), _diff()) == _native.CLV_OK  # no sequences
    assert call(None, _diff()) == _native.CLV_EINVAL
    assert call(_decode_args(), None) == _native.CLV_EINVAL
    for field, value in (("out_scale", float("nan")), ("lambda_value", float("inf"))):
        d = _diff()
        setattr(d, field, value)
        assert call(_decode_args(), d) == _native.CLV_EINVAL
    d = _diff()
    d.norm_weight, d.norm_eps = 0x3000, -1.0
    assert call(_decode_args(), d) == _native.CLV_EINVAL
    assert call(_decode_args(head_dim=96), _diff()) == _native.CLV_EUNSUPPORTED
    assert call(_decode_args(block_size=12), _diff()) == _native.CLV_EUNSUPPORTED
    # fp8 pools: both scales, 16-bit queries, head_dim 128, pages of 16
    assert call(_decode_args(), _diff(), 0x3000, None) == _native.CLV_EINVAL
    assert call(_decode_args(dtype=_native.CLV_F32), _diff(), 0x3000, 0x3000) == _native.CLV_EINVAL
    assert call(_decode_args(head_dim=256), _diff(), 0x3000, 0x3000) == _native.CLV_EUNSUPPORTED
    assert call(_decode_args(block_size=8), _diff(), 0x3000, 0x3000) == _native.CLV_EUNSUPPORTED
    a = _decode_args(max_len=4000)
    a.num_seqs = 1
    assert native_lib.clv_diff_decode_workspace_bytes(a, 0, 0) > 0
    assert call(a, _diff()) == _native.CLV_EWORKSPACE
    a.max_context_len = 512
    assert native_lib.clv_diff_decode_workspace_bytes(a, 0, 0) == 0
    assert native_lib.clv_diff_decode_workspace_bytes(a, 1, 0) == 0
    assert native_lib.clv_diff_decode_workspace_bytes(a, 0, 64) > 0
    assert native_lib.clv_diff_decode_workspace_bytes(a, 1, 64) > 0
    a.num_heads = 30
    assert call(a, _diff()) == _native.CLV_EINVAL


def test_prefill_arguments(native_lib):
    p = _native.PrefillArgs()
    p.num_heads, p.num_kv_heads, p.head_dim, p.block_size, p.num_blocks = 8, 2, 128, 16, 4
    p.dtype, p.scale = _native.CLV_F16, 0.1
    call = native_lib.clv_diff_prefill
    assert call(p, _diff(), None, 0, None) == _native.CLV_OK  # nothing to do
    assert call(p, None, None, 0, None) == _native.CLV_EINVAL
    assert call(None, _diff(), None, 0, None) == _native.CLV_EINVAL
    p.head_dim = 100
    assert call(p, _diff(), None, 0, None) == _native.CLV_EUNSUPPORTED


@pytest.mark.parametrize("field,value,code", [
    ("rows", -1, _native.CLV_EINVAL),
    ("rows", 2049, _native.CLV_EUNSUPPORTED),
    ("block_size", 12, _native.CLV_EUNSUPPORTED),
    ("width", 1 << 28, _native.CLV_EINVAL),       # positions past 32 bits
    ("reserve", -1, _native.CLV_EINVAL),
    ("num_tokens", 1 << 31, _native.CLV_EINVAL),
    ("num_free", None, _native.CLV_EINVAL),
    ("status", None, _native.CLV_EINVAL),
    ("new_lens", None, _native.CLV_EINVAL),
    ("slot_mapping", None, _native.CLV_EINVAL),
])
def test_tables_arguments(native_lib, field, value, code):
    a = _native.TablesArgs()
    for name, _ in _native.TablesArgs._fields_[:12]:
        setattr(a, name, 0x1000)
    a.num_tokens, a.rows, a.width, a.block_size, a.num_blocks, a.reserve = 9000, 3, 4, 16, 8, 1
    setattr(a, field, value)
    assert native_lib.clv_advance_block_tables(a, None) == code


def test_tables_outputs_that_overlap_inputs(native_lib):
    """An output may be its own input, not a part of one or another one."""
    def call(**kw):
        a = _native.TablesArgs()
        for i, (name, _) in enumerate(_native.TablesArgs._fields_[:12]):
            setattr(a, name, 0x1000 * (i + 1))
        a.rows, a.width, a.block_size, a.num_blocks = 100, 4, 16, 8
        for k, v in kw.items():
            setattr(a, k, v)
        return native_lib.clv_advance_block_tables(a, None)

    held, lens, new, count = 0x2000, 0x3000, 0x4000, 0x6000
    for kw in ({"blocks_held_out": held + 4}, {"blocks_held_out": lens}, {"context_lens_out": new},
               {"context_lens_out": lens - 4}, {"num_free_out": held + 396}, {"num_free_out": count + 0,
                "blocks_held_out": count - 8}):
        assert call(**kw) == _native.CLV_EINVAL, kw
    # what every step writes, on an input, on the state or on each other
    table, stack, slots, qsl, status = 0x1000, 0x5000, 0xa000, 0xb000, 0xc000
    for kw in ({"query_start_loc": lens}, {"query_start_loc": new + 396}, {"status": count},
               {"status": table + 1596}, {"status": qsl + 400}, {"new_lens": stack + 28},
               {"num_tokens": 4, "slot_mapping": stack + 24},
               {"num_tokens": 4, "slot_mapping": held - 24}, {"blocks_held_out": table},
               {"num_tokens": 600, "slot_mapping": slots}, {"num_free_out": status}):
        assert call(**kw) == _native.CLV_EINVAL, kw


def test_struct_layouts(tmp_path):
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = {"clv_diff_args": _native.DiffArgs, "clv_tables_args": _native.TablesArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "clover_attn.h"',
             "int main(void) {"]
    for c, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f.rstrip("_")}));' for f, _ in cls._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(tmp_path / "l.c"),
                    "-o", str(tmp_path / "l")], check=True)
    got = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout
    want = []
    for cls in structs.values():
        want += [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert [int(x) for x in got.split()] == want


def test_step_restates_the_manager():
    """oracle.differential.advance against the restated block manager: the
    same blocks, call by call."""
    m = ob.BlockBookkeeping(40, 4)
    table, held, lens, stack = [[-1] * 10 for _ in range(4)], [0] * 4, [0] * 4, list(range(40))
    for new in ([9, 3, 0, 4], [1, 1, 2, 1], [-1, 1, 5, 1], [6, 1, 0, -1], [1, 0, 1, 30]):
        for r, n in enumerate(new):
            if n < 0:
                m.free(str(r))
        for r, n in enumerate(new):
            if n > 0 and str(r) not in m.block_tables:
                m.allocate(str(r), n)
            else:
                for _ in range(max(0, n)):
                    m.append_slot(str(r))
        status, table, held, lens, stack, slots, qsl = od.advance(table, held, lens, new, stack, 4, 60,
                                                                  10, 40)
        assert status == od.TABLES_OK and stack == m.free_blocks
        for r in range(4):
            assert table[r][:held[r]] == m.block_tables.get(str(r), [])
            assert lens[r] == m.context_lens.get(str(r), 0)


def test_restated_rows_by_hand():
    """Two tokens, one head: weights and difference by hand."""
    q = torch.tensor([[[1.0, 0.0, 0.0, 2.0]]])
    k = torch.tensor([[[1.0, 5.0, 7.0, 0.0]], [[0.0, 0.0, 0.0, 1.0]]])
    v = torch.tensor([[[1.0, 2.0, 3.0, 4.0]], [[-1.0, 0.0, 1.0, 2.0]]])
    r = od.rows(q, k, v, [2], 0.5, scale=1.0)
    w1 = torch.softmax(torch.tensor([1.0, 0.0], dtype=torch.float64), 0)
    w2 = torch.softmax(torch.tensor([0.0, 2.0], dtype=torch.float64), 0)
    want = (w1 - 0.5 * w2) @ v[:, 0].double()
    assert torch.allclose(r["out"][0, 0], want)
    n = od.rows(q, k, v, [2], 0.5, torch.full((4,), 2.0), eps=0.0, out_scale=0.3, scale=1.0)
    assert torch.allclose(n["out"][0, 0], 0.3 * 2.0 * want / want.square().mean().sqrt())


@pytest.mark.parametrize("room", [True, False])
def test_prefill_without_room_for_a_workspace(monkeypatch, room):
    """On a full device the call runs as the form that needs no memory."""
    t = decode_tensors()
    calls = []
    lib = types.SimpleNamespace(
        clv_diff_prefill_workspace_bytes=lambda a: 4096,
        clv_diff_prefill=lambda a, d, ws, n, s: calls.append((ws is not None, n)) or 0)

    def empty(*size, **kw):
        if not room:
            raise torch.cuda.OutOfMemoryError("no room")
        return torch.zeros(*size, **kw)

    monkeypatch.setattr(kernels, "_require_device", lambda *t: t[0].device)
    monkeypatch.setattr(kernels._native, "load", lambda: lib)
    monkeypatch.setattr(kernels, "_stream", lambda dev: 0)
    monkeypatch.setattr(torch, "empty", empty)
    kernels.differential_prefill(*t, torch.arange(4, dtype=torch.int32), 1, 0.5)
    assert calls == [(True, 4096) if room else (False, 0)]


def test_launches_run_with_their_tensors_device_current(monkeypatch):
    """On tensors of another device than the current one the call changes to
    it: the default stream and the device queries are the current device's."""
    here, trace = [0], []

    class Guard:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            trace.append(self.dev.index)
            here[0] = self.dev.index

        def __exit__(self, *exc):
            here[0] = 0

    monkeypatch.setattr(kernels, "_current_device", lambda: here[0])
    monkeypatch.setattr(torch.cuda, "device", Guard)
    for index in (0, 1):
        with kernels._on(torch.device("cuda", index)):
            assert here[0] == index
        assert here[0] == 0
    with kernels._on(torch.device("cpu")):
        pass
    assert trace == [1]
