"""Differential attention (decode and prefill forms) over paged pools against
the float64 restatement, within the error its arithmetic allows
(oracle.differential.bound): head shapes and groups, lengths of 0 and 1, page
ends inside a step, unreadable blocks, NaN in unused slots, strided rows, every
form of lambda, with and without the norm, all pool dtypes."""
import math

import pytest
import torch

from cloverinfer_amd import _native, kernels
from oracle import differential as od
from tests.helpers import make_paged_kv, padded_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"

# What a stored weight loses before its product with V: 16-bit pools split it
# into a value and its residual (two half steps multiply), fp8 pools and the
# MFMA prefill hold it in fp16. fp16 subnormals: half a step of 2^-24; the
# lazily raised maximum of the prefill keeps weights of up to 2^8, so its row
# sum is at least 1 like the decode's.
DECODE_BITS = {torch.float32: (0.0, 0.0), torch.float16: (2.0 ** -22, 2.0 ** -25),
               torch.bfloat16: (2.0 ** -16, 0.0)}
PREFILL_BITS = {torch.float32: (0.0, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25),
                torch.bfloat16: (2.0 ** -11, 2.0 ** -25)}


def _lam(kind, n, hq, g):
    if kind == "number":
        return 0.35
    t = torch.rand(n, hq, generator=g) * 0.6 + 0.2
    return t if kind == "row" else t[0].clone()


def _check(got, ref, dtype, bits, what):
    tol = od.bound(ref, dtype, *bits)
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    bad = (got - ref["out"]).abs() > tol
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, worst ratio "
        f"{((got - ref['out']).abs() / tol).max().item():.2f}, first at {bad.nonzero()[0].tolist()}")


def _gathered(pool, table, ctx, bs):
    t = torch.arange(ctx)
    blocks = torch.tensor(table, dtype=torch.long)
    return pool.flatten(0, 1)[blocks[t // bs] * bs + t % bs] if ctx else pool.flatten(0, 1)[:0]


def _decode(ctx, hq, hkv, d, dtype, bs=16, lam="head", norm=True, num_waves=0, seed=0, max_len=None,
            hole=None, strided=False, scale=None, out_scale=0.4, value_scale=1.0):
    print(f"differential decode {dtype} {hq}/{hkv} d{d} bs{bs} ctx {ctx} lam {lam} norm {norm} "
          f"waves {num_waves}", flush=True)
    k, v, tables = make_paged_kv(seed, ctx, hkv, d, bs, dtype, value_scale, spare_blocks=2)
    g = torch.Generator().manual_seed(seed + 1)
    n = len(ctx)
    q = torch.randn(n, hq, d, generator=g).to(dtype)
    lam = _lam(lam, n, hq, g)
    weight = torch.rand(d, generator=g) + 0.5 if norm else None
    shown = [list(t) for t in tables]
    limits = [min(c, max_len) if max_len is not None else c for c in ctx]
    visible = [list(range(c)) for c in limits]
    if hole is not None:  # an unreadable block in the middle of every context
        for s, t in enumerate(shown):
            i = len(t) // 2
            t[i] = hole
            visible[s] = [x for x in visible[s] if x // bs != i]
    ref = []
    for s in range(n):
        kk, vv = _gathered(k, tables[s], ctx[s], bs), _gathered(v, tables[s], ctx[s], bs)
        ls = lam[s:s + 1] if isinstance(lam, torch.Tensor) and lam.dim() == 2 else lam
        ref.append(od.rows(q[s:s + 1], kk, vv, [visible[s]], ls, weight, out_scale=out_scale,
                           scale=scale))
    ref = {key: (torch.cat([r[key] for r in ref]) if isinstance(ref[0][key], torch.Tensor)
                 and key != "weight" else ref[0][key]) for key in ref[0]}
    qg = q.to(DEV)
    out = torch.full((n, hq, d), float("nan"), dtype=dtype, device=DEV)
    if strided:  # rows of a wider buffer, heads transposed in the output
        wide = torch.zeros(n, 2, hq, d, dtype=dtype, device=DEV)
        wide[:, 1] = qg
        qg = wide[:, 1]
        out = torch.full((hq, n, d), float("nan"), dtype=dtype, device=DEV).transpose(0, 1)
    if isinstance(lam, torch.Tensor):
        lam = lam.to(DEV)
        if strided and lam.dim() == 2:
            lam = lam.t().contiguous().t()
    kernels.differential_attention(
        out, qg, k.to(DEV), v.to(DEV), padded_tables(shown).to(DEV),
        torch.tensor(ctx, dtype=torch.int32, device=DEV), bs,
        max(ctx) if max_len is None else max_len, lam, scale=scale,
        norm_weight=None if weight is None else weight.to(DEV), out_scale=out_scale,
        num_waves=num_waves)
    torch.cuda.synchronize()
    _check(out, ref, dtype, DECODE_BITS[dtype], "differential decode")
    return out


HEADS = [(6, 6, 128), (14, 2, 256), (28, 4, 128), (16, 4, 64), (3, 1, 256)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
RAGGED = [0, 1, 2, 15, 16, 17, 63, 300, 513, 1100]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("num_waves", [0, 37])
def test_decode_ragged(hq, hkv, d, dtype, num_waves):
    _decode(RAGGED, hq, hkv, d, dtype, num_waves=num_waves, lam="row")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_decode_short(hq, hkv, d, dtype):
    """At most 512 tokens: one launch."""
    _decode([1, 0, 128, 511, 512, 33], hq, hkv, d, dtype, norm=False, lam="number")


@pytest.mark.parametrize("hq,hkv", [(24, 2), (9, 1), (40, 2)])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("ctx", [[40, 0, 200], [700, 1, 0, 1500]])
def test_decode_large_groups(hq, hkv, d, ctx):
    """More rows of both maps per kv head than one 16-row chunk."""
    _decode(ctx, hq, hkv, d, torch.bfloat16)


@pytest.mark.parametrize("bs", [1, 4, 8, 32, 128])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_block_sizes(bs, d, dtype):
    _decode([5, 700, 37, 130], 8, 2, d, dtype, bs=bs)


@pytest.mark.parametrize("d", [8, 16, 32])
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_small_heads(d, dtype):
    _decode([5, 0, 700, 1], 6, 2, d, dtype, lam="row")


@pytest.mark.parametrize("hole", [-1, 1 << 30])
@pytest.mark.parametrize("ctx", [[100, 300, 33, 7], [1000, 600, 40, 7]])
@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 256)])
def test_decode_unreadable_blocks(hole, ctx, hq, hkv, d):
    """Masked tokens; the sequence of 7 tokens has no readable one: zeros."""
    out = _decode(ctx, hq, hkv, d, torch.float16, hole=hole)
    assert (out[3] == 0).all()


def test_decode_lengths_past_the_bound():
    """context_lens beyond max_context_len are cut there."""
    _decode([900, 20, 700], 6, 6, 128, torch.float16, max_len=650)
    _decode([900, 20, 300], 6, 6, 128, torch.float16, max_len=100)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx", [[40, 7, 300], [40, 7, 1300]])
def test_decode_strided_rows(dtype, ctx):
    _decode(ctx, 12, 4, 128, dtype, lam="row", strided=True)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_decode_scales(scale):
    _decode([40, 900], 6, 2, 128, torch.bfloat16, scale=scale, lam="number", out_scale=-1.5)


@pytest.mark.parametrize("kind", ["number", "head", "row"])
def test_decode_equal_maps_cancel(kind):
    """Both maps equal and lambda 1: o is 0 up to rounding, and the norm's eps
    keeps it there."""
    ctx, hq, hkv, d = [700, 40], 4, 2, 128
    k, v, tables = make_paged_kv(3, ctx, hkv, d, 16, torch.bfloat16)
    k[..., d // 2:] = k[..., :d // 2]
    q = torch.randn(2, hq, d, generator=torch.Generator().manual_seed(1)).bfloat16()
    q[..., d // 2:] = q[..., :d // 2]
    lam = {"number": 1.0, "head": torch.ones(hq, device=DEV),
           "row": torch.ones(2, hq, device=DEV)}[kind]
    out = torch.full_like(q, float("nan"), device=DEV)
    kernels.differential_attention(out, q.to(DEV), k.to(DEV), v.to(DEV),
                                   padded_tables(tables).to(DEV),
                                   torch.tensor(ctx, dtype=torch.int32, device=DEV), 16, 700, lam,
                                   norm_weight=torch.ones(d, device=DEV))
    # a context is off by at most about (64 + 6 + 2 * 108) 2^-24 of |v| <= 6, so
    # |o| < 2.1e-4 and out < 2.1e-4 / sqrt(eps) = 0.066.
    assert out.abs().max().item() < 0.066


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv", [(28, 4), (6, 6), (24, 2)])
@pytest.mark.parametrize("ctx", [[1, 0, 17, 400], [3000, 1, 700]])
@pytest.mark.parametrize("num_waves", [0, 48])  # one launch or partitions; the even split
def test_decode_fp8_pools(dtype, hq, hkv, ctx, num_waves):
    d, bs, n = 128, 16, len(ctx)
    print(f"differential decode fp8 {dtype} {hq}/{hkv} ctx {ctx} waves {num_waves}", flush=True)
    k, v, tables = make_paged_kv(5, ctx, hkv, d, bs, dtype)
    g = torch.Generator().manual_seed(6)
    ks, vs = (torch.rand(hkv, generator=g) * 0.02 + 0.01 for _ in range(2))
    k8 = torch.zeros(k.shape, dtype=torch.uint8).view(kernels.FP8).to(DEV)
    v8 = torch.zeros(k.shape, dtype=torch.uint8).view(kernels.FP8).to(DEV)
    slots = torch.tensor([t[p // bs] * bs + p % bs for t, c in zip(tables, ctx) for p in range(c)])
    kernels.reshape_and_cache(k.flatten(0, 1)[slots].to(DEV), v.flatten(0, 1)[slots].to(DEV), k8, v8,
                              slots.to(DEV), k_scale=ks, v_scale=vs)
    kd = k8.cpu().double() * ks.double().view(1, 1, -1, 1)
    vd = v8.cpu().double() * vs.double().view(1, 1, -1, 1)
    q = torch.randn(n, hq, d, generator=g).to(dtype)
    weight = torch.rand(d, generator=g) + 0.5
    out = torch.full((n, hq, d), float("nan"), dtype=dtype, device=DEV)
    kernels.differential_attention(out, q.to(DEV), k8, v8, padded_tables(tables).to(DEV),
                                   torch.tensor(ctx, dtype=torch.int32, device=DEV), bs, max(ctx),
                                   0.6, norm_weight=weight.to(DEV), k_scale=ks, v_scale=vs.to(DEV),
                                   num_waves=num_waves)
    for s in range(n):
        ref = od.rows(q[s:s + 1], _gathered(kd, tables[s], ctx[s], bs),
                      _gathered(vd, tables[s], ctx[s], bs), [ctx[s]], 0.6, weight)
        # a weight in fp16; the scales enter as one fp32 factor each
        _check(out[s:s + 1], ref, dtype, (2.0 ** -11 + 2.0 ** -22, 2.0 ** -25), f"sequence {s}")


def test_decode_offsets_past_32_bits():
    """Blocks past 2^32 bytes of a pool."""
    bs, hkv, d, hq = 16, 2, 256, 14
    blocks = (1 << 32) // (bs * hkv * d * 2) + 300
    k = torch.empty(blocks, bs, hkv, d, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(0)
    ctx = [700, 90]
    tables = [[blocks - 1 - i for i in range(44)], [blocks - 60 - i for i in range(6)]]
    kk = [torch.randn(c, hkv, d, generator=g).bfloat16() for c in ctx]
    vv = [torch.randn(c, hkv, d, generator=g).bfloat16() for c in ctx]
    slots = torch.tensor([t[p // bs] * bs + p % bs for t, c in zip(tables, ctx) for p in range(c)])
    kernels.reshape_and_cache(torch.cat(kk).to(DEV), torch.cat(vv).to(DEV), k, v, slots.to(DEV))
    q = torch.randn(2, hq, d, generator=g).bfloat16()
    out = torch.full((2, hq, d), float("nan"), dtype=torch.bfloat16, device=DEV)
    cl = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    kernels.differential_attention(out, q.to(DEV), k, v, padded_tables(tables).to(DEV), cl, bs, 700,
                                   0.5)
    rows = torch.full_like(out, float("nan"))
    kernels.differential_prefill(rows, q.to(DEV), k, v, padded_tables(tables).to(DEV), cl,
                                 torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), 1, 0.5)
    for s in range(2):
        ref = od.rows(q[s:s + 1], kk[s], vv[s], [ctx[s]], 0.5)
        _check(out[s:s + 1], ref, torch.bfloat16, DECODE_BITS[torch.bfloat16], f"decode {s}")
        _check(rows[s:s + 1], ref, torch.bfloat16, PREFILL_BITS[torch.bfloat16], f"prefill {s}")


# ------------------------------------------------------------------ prefill
def _prefill(cached, new, hq, hkv, d, dtype, bs=16, lam="head", norm=True, seed=0, max_new=None,
             hole=None, strided=False, pad=0, scale=None, width=None, value_scale=1.0):
    print(f"differential prefill {dtype} {hq}/{hkv} d{d} bs{bs} cached {cached} new {new} lam {lam} "
          f"norm {norm}", flush=True)
    ctx = [c + n for c, n in zip(cached, new)]
    k, v, tables = make_paged_kv(seed, ctx, hkv, d, bs, dtype, value_scale, spare_blocks=2)
    g = torch.Generator().manual_seed(seed + 1)
    rows = sum(new)
    q = torch.randn(rows + pad, hq, d, generator=g).to(dtype)
    lam = _lam(lam, rows + pad, hq, g)
    weight = torch.rand(d, generator=g) + 0.5 if norm else None
    shown = [list(t) for t in tables]
    holes = {}
    if hole is not None:
        for s, t in enumerate(shown):
            holes[s] = len(t) // 2
            t[holes[s]] = hole
    qsl = [0]
    for n in new:
        qsl.append(qsl[-1] + n)
    qg = q.to(DEV)
    out = torch.full((rows + pad, hq, d), float("nan"), dtype=dtype, device=DEV)
    if strided:
        wide = torch.zeros(rows + pad, 2, hq, d, dtype=dtype, device=DEV)
        wide[:, 1] = qg
        qg = wide[:, 1]
        out = torch.full((hq, rows + pad, d), float("nan"), dtype=dtype, device=DEV).transpose(0, 1)
    lg = lam.to(DEV) if isinstance(lam, torch.Tensor) else lam
    kernels.differential_prefill(
        out, qg, k.to(DEV), v.to(DEV), padded_tables(shown, width).to(DEV),
        torch.tensor(ctx, dtype=torch.int32, device=DEV),
        torch.tensor(qsl, dtype=torch.int32, device=DEV), max_new or max(new), lg, scale=scale,
        norm_weight=None if weight is None else weight.to(DEV), out_scale=0.4)
    torch.cuda.synchronize()
    for s, (c, n) in enumerate(zip(cached, new)):
        if n == 0:
            continue
        lo, hi = qsl[s], qsl[s + 1]
        limits = [c + i + 1 for i in range(n)]
        if s in holes:
            limits = [[x for x in range(m) if x // bs != holes[s]] for m in limits]
        ls = lam[lo:hi] if isinstance(lam, torch.Tensor) and lam.dim() == 2 else lam
        ref = od.rows(q[lo:hi], _gathered(k, tables[s], ctx[s], bs),
                      _gathered(v, tables[s], ctx[s], bs), limits, ls, weight, out_scale=0.4,
                      scale=scale)
        _check(out[lo:hi], ref, dtype, PREFILL_BITS[dtype], f"sequence {s}")
    if pad:  # rows behind the last sequence stay as they were
        assert torch.isnan(out[rows:]).all()
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_prefill_ragged(hq, hkv, d, dtype):
    _prefill([0, 5, 0, 100, 17, 63], [1, 40, 0, 7, 130, 1], hq, hkv, d, dtype, lam="row", pad=5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_prefill_long(hq, hkv, d, dtype):
    """Contexts long enough for the even split."""
    _prefill([1500, 0, 2000], [20, 90, 1], hq, hkv, d, dtype, norm=hq != 6)


@pytest.mark.parametrize("hq,hkv", [(24, 2), (9, 1), (130, 1)])
def test_prefill_large_groups(hq, hkv):
    _prefill([30, 0], [9, 40], hq, hkv, 128, torch.bfloat16)


@pytest.mark.parametrize("bs", [1, 2, 4, 8, 32, 128])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prefill_block_sizes(bs, d, dtype):
    _prefill([5, 70], [33, 20], 8, 2, d, dtype, bs=bs)


@pytest.mark.parametrize("d", [8, 16, 32])
def test_prefill_small_heads(d):
    _prefill([5, 0], [3, 40], 6, 2, d, torch.float16, lam="row")


@pytest.mark.parametrize("hole", [-1, 1 << 30])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [128, 256])
def test_prefill_unreadable_blocks(hole, dtype, d):
    """The last sequence has a single, unreadable block: zeros."""
    out = _prefill([100, 0, 4], [20, 60, 3], 8, 2, d, dtype, hole=hole)
    assert (out[80:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_strided_rows(dtype):
    _prefill([0, 60], [50, 3], 12, 4, 128, dtype, lam="row", strided=True)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_prefill_scales(scale):
    _prefill([0, 60], [50, 3], 6, 2, 128, torch.bfloat16, scale=scale, lam="number")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("cached", [[0, 0], [1500, 0]])
def test_prefill_rows_past_the_bound_are_nan(dtype, d, cached):
    """A chunk longer than max_query_len marks its rows past it."""
    new, hq, hkv = [30, 5], 4, 2
    ctx = [c + n for c, n in zip(cached, new)]
    k, v, tables = make_paged_kv(1, ctx, hkv, d, 16, dtype)
    q = torch.randn(35, hq, d, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    out = torch.zeros_like(q)
    kernels.differential_prefill(out, q, k.to(DEV), v.to(DEV), padded_tables(tables).to(DEV),
                                 torch.tensor(ctx, dtype=torch.int32, device=DEV),
                                 torch.tensor([0, 30, 35], dtype=torch.int32, device=DEV), 9, 0.3)
    assert torch.isnan(out[9:30]).all()
    assert torch.isfinite(out[:9]).all() and torch.isfinite(out[30:]).all()


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("cached", [0, 1500])
def test_prefill_large_bf16_values(d, cached):
    """bf16 values that fp16 does not hold."""
    _prefill([cached, 20], [40, 30], 8, 2, d, torch.bfloat16, value_scale=1e5)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("pool", ["k", "v"])
@pytest.mark.parametrize("cached", [0, 1500])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_hidden_values_stay_hidden(dtype, d, cached, pool, value):
    """A key or value that is not finite reaches no row that does not see its
    token; in V it reaches only its own column of those that do."""
    hq, hkv, n, bad = 4, 2, 40, 13
    ctx = [cached + n, 20]
    k, v, tables = make_paged_kv(2, ctx, hkv, d, 16, dtype)
    q = torch.randn(n + 20, hq, d, generator=torch.Generator().manual_seed(2)).to(dtype)
    kk = [_gathered(k, tables[s], ctx[s], 16) for s in range(2)]
    vv = [_gathered(v, tables[s], ctx[s], 16) for s in range(2)]
    pos, col = cached + bad, d - 3
    block, offset = tables[0][pos // 16], pos % 16
    (k if pool == "k" else v)[block, offset, 1, col] = value
    out = torch.zeros_like(q, device=DEV)
    kernels.differential_prefill(out, q.to(DEV), k.to(DEV), v.to(DEV), padded_tables(tables).to(DEV),
                                 torch.tensor(ctx, dtype=torch.int32, device=DEV),
                                 torch.tensor([0, n, n + 20], dtype=torch.int32, device=DEV), n, 0.3)
    out = out.cpu()
    clean = od.rows(q[:n], kk[0], vv[0], [cached + i + 1 for i in range(n)], 0.3)
    if pool == "v":
        assert not torch.isfinite(out[bad:n, 2:, col]).any()
        out[bad:n, 2:, col] = clean["out"][bad:, 2:, col].to(dtype)
    else:  # those rows' heads are all not finite, or all the value's limit
        out[bad:n, 2:] = clean["out"][bad:, 2:].to(dtype)
    _check(out[:n], clean, dtype, PREFILL_BITS[dtype], "rows of the sequence")
    other = od.rows(q[n:], kk[1], vv[1], [i + 1 for i in range(20)], 0.3)
    _check(out[n:], other, dtype, PREFILL_BITS[dtype], "the other sequence")


def test_prefill_one_row_equals_decode():
    """A chunk of one row per sequence is the decode's call."""
    ctx, hq, hkv, d, dtype = [1, 700, 33, 2000], 14, 2, 256, torch.float32
    k, v, tables = make_paged_kv(9, ctx, hkv, d, 16, dtype)
    k, v, bt = k.to(DEV), v.to(DEV), padded_tables(tables).to(DEV)
    q = torch.randn(4, hq, d, generator=torch.Generator().manual_seed(3)).to(DEV)
    cl = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    a, b = torch.empty_like(q), torch.empty_like(q)
    kernels.differential_attention(a, q, k, v, bt, cl, 16, 2000, 0.4)
    kernels.differential_prefill(b, q, k, v, bt, cl, torch.arange(5, dtype=torch.int32, device=DEV),
                                 None, 0.4)
    # two fp32 results, each within its bound of the same number
    for s in range(4):
        ref = od.rows(q[s:s + 1].cpu(), _gathered(k.cpu(), tables[s], ctx[s], 16),
                      _gathered(v.cpu(), tables[s], ctx[s], 16), [ctx[s]], 0.4)
        assert ((a[s] - b[s]).double().cpu().abs() <= 2 * od.bound(ref, dtype)[0]).all()


@pytest.mark.parametrize("form", ["decode", "decode_short", "prefill"])
def test_graph_replays(form):
    """Captured and replayed over changed inputs, with eager calls between."""
    hq, hkv, d, dtype = 14, 2, 256, torch.bfloat16
    ctx = [300, 40, 0, 511] if form == "decode_short" else [1300, 40, 0, 2000]
    k, v, tables = make_paged_kv(4, ctx, hkv, d, 16, dtype)
    k, v, bt = k.to(DEV), v.to(DEV), padded_tables(tables).to(DEV)
    cl = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    new = [5, 2, 0, 30]
    rows = sum(new) if form == "prefill" else 4
    qsl = torch.tensor([0, 5, 7, 7, 37], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(rows, hq, d, generator=g, device=DEV).to(dtype)
    lam = torch.rand(rows, hq, generator=g, device=DEV)
    w = torch.rand(d, generator=g, device=DEV)

    def call(out, q):
        if form == "prefill":
            kernels.differential_prefill(out, q, k, v, bt, cl, qsl, 30, lam, norm_weight=w)
        else:
            kernels.differential_attention(out, q, k, v, bt, cl, 16, max(ctx), lam, norm_weight=w)

    out, eager = torch.empty_like(q), torch.empty_like(q)
    call(out, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, q)
    for i in range(5):
        q.copy_(torch.randn(rows, hq, d, generator=g, device=DEV).to(dtype))
        out.fill_(float("nan"))
        graph.replay()
        call(eager, q)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {i}"


def test_repeated_calls_are_bit_equal_and_streams_do_not_share():
    """The same call gives the same bits; calls on two streams at once keep to
    their own workspaces."""
    hq, hkv, d, dtype = 28, 4, 128, torch.bfloat16
    ctx = [3000, 100, 1700, 5]
    k, v, tables = make_paged_kv(8, ctx, hkv, d, 16, dtype)
    k, v, bt = k.to(DEV), v.to(DEV), padded_tables(tables).to(DEV)
    cl = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    qs = [torch.randn(4, hq, d, generator=g, device=DEV).to(dtype) for _ in range(2)]
    want = [torch.empty_like(q) for q in qs]
    for q, o in zip(qs, want):
        kernels.differential_attention(o, q, k, v, bt, cl, 16, 3000, 0.4)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[torch.empty_like(q) for _ in range(4)] for q in qs]
    for i in range(4):
        for q, o, st in zip(qs, got, streams):
            with torch.cuda.stream(st):
                kernels.differential_attention(o[i], q, k, v, bt, cl, 16, 3000, 0.4)
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


@pytest.mark.parametrize("hq,hkv,d,dtype,cached,new", [
    (6, 6, 128, torch.float32, [100, 0], [200, 30]),
    (6, 2, 128, torch.bfloat16, [50, 300], [1000, 40]),
    (3, 1, 256, torch.float16, [0, 300], [1030, 7]),
])
def test_prefill_without_a_workspace(monkeypatch, hq, hkv, d, dtype, cached, new):
    """Where the device has no room for a split prefill's partials, the form
    that needs none answers."""
    real, refused = torch.empty, []

    def empty(*size, **kw):
        if kw.get("dtype") is torch.uint8:
            refused.append(size[0])
            raise torch.cuda.OutOfMemoryError("no room")
        return real(*size, **kw)

    split = _prefill(cached, new, hq, hkv, d, dtype)
    monkeypatch.setattr(torch, "empty", empty)
    whole = _prefill(cached, new, hq, hkv, d, dtype)
    monkeypatch.undo()
    assert len(refused) == 1 and refused[0] > 0
    assert whole.shape == split.shape


def test_decode_many_short_wide_rows():
    """head_dim 256 past the segments that one launch takes."""
    _decode([(i * 7) % 40 for i in range(130)], 4, 4, 256, torch.float16)


def test_native_argument_block_is_the_python_one(monkeypatch):
    """The native host code fills the block that the Python checks fill, and
    leaves what they refuse, or take in another form, to them."""
    q = torch.zeros(3, 8, 64, dtype=torch.float16, device=DEV)
    lam = torch.rand(3, 8, device=DEV)
    weight = torch.rand(64, device=DEV)
    real = kernels._filled
    for x in (0.25, lam, lam[0], torch.rand(8, 3, device=DEV).t(), torch.rand(16, device=DEV)[::2]):
        for w in (None, weight):
            assert real("fill_diff_args", _native.DiffArgs(), q, x, w, 1e-6, 0.2) is not None
            native = bytes(kernels._diff_args(q, x, w, 1e-6, 0.2))
            monkeypatch.setattr(kernels, "_filled", lambda *a: None)
            assert bytes(kernels._diff_args(q, x, w, 1e-6, 0.2)) == native
            monkeypatch.setattr(kernels, "_filled", real)
    assert kernels._diff_args(q, 1, None, 1e-6, 0.2).lambda_value == 1.0
    for x, w in ((lam.double(), None), (lam[:2], None), (lam[:, :7], None), (lam.cpu(), None),
                 (lam[None], None), (0.2, weight.half()), (0.2, weight[:32]), (0.2, weight.cpu()),
                 (0.2, torch.rand(128, device=DEV)[::2]), (lam[0, 0], None)):
        assert real("fill_diff_args", _native.DiffArgs(), q, x, w, 1e-6, 0.2) is None
        with pytest.raises(ValueError):
            kernels._diff_args(q, x, w, 1e-6, 0.2)


def test_decode_more_segments_than_the_split_takes():
    """Past 4096 segments a workgroup each, at any length."""
    _decode([3 + (i * 13) % 40 for i in range(1030)] + [700], 4, 4, 64, torch.bfloat16)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(14, 2, 256, torch.bfloat16), (28, 4, 128, torch.float16),
                                            (6, 6, 128, torch.float32), (16, 4, 64, torch.bfloat16)])
@pytest.mark.parametrize("num_waves", [0, 48])  # partitions of a small batch; the even split
@pytest.mark.parametrize("form", ["ends", "hole", "strided", "bound", "one"])
def test_decode_splits(hq, hkv, d, dtype, num_waves, form):
    """Both ways of splitting a small batch: contexts that end on and beside a
    partition, unreadable blocks, strided rows, lengths past the bound."""
    ctx = {"ends": [64, 63, 65, 128, 127, 129, 0, 1, 192, 1025], "hole": [1000, 600, 40, 7],
           "strided": [40, 7, 1300], "bound": [3000, 20, 700], "one": [2111]}[form]
    _decode(ctx, hq, hkv, d, dtype, num_waves=num_waves, hole=-1 if form == "hole" else None,
            strided=form == "strided", max_len=900 if form == "bound" else None, lam="row")
