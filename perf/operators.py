"""Differential attention over the paged cache, and the block tables and slot maps it reads.

Three operators, each called as a serving program calls it, on tensors that already lie on the GPU:

* ``decode`` (``kernels.differential_attention``): one query row per sequence over its paged context.
  Query head h has two halves q1 | q2 of head_dim / 2, its kv head's key row is k1 | k2, its value row v
  has the whole head_dim:
      a_m = softmax(scale * q_m . K_m^T) V  (m = 1, 2),   o = a_1 - lambda a_2,
      out = out_scale * weight * o / sqrt(mean(o^2) + eps)   (without a norm: out_scale * o);
* ``prefill`` (``kernels.differential_prefill``): the same for each sequence's new rows, causal over its
  paged context;
* ``tables`` (``kernels.advance_block_tables``): one scheduling step of the cache: rows of the block table
  grow by their new tokens (blocks popped from a free stack), finished rows give their blocks back, every
  new token gets its cache slot.

Head shapes are the pairs of the benchmark's heads (6/6 pairs of 64 for OPT-125m, 16/16, 14/2 and 16/4
pairs of 128), and pairs of 32 and 64 in 32/8, 28/4 and 16/4 heads. A case holds plain values only; its lengths
follow from them, its tensors' contents from the seed.
"""
import math
import random

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_FP8 = torch.float8_e4m3fn
_DEV = "cuda"
_EPS = 1e-5
_OUT_SCALE = 0.2  # 1 - lambda_init of a deep layer

# (query heads, kv heads, head_dim = both halves)
_HEADS = [(6, 6, 128), (16, 16, 256), (14, 2, 256), (16, 4, 256), (28, 4, 128), (32, 8, 128), (16, 4, 64)]

# Most work of one drawn case: those of the largest listed ones.
_MAX_BYTES = 2.2e9
_MAX_FLOPS = {"float32": 2.5e10, "float16": 4.4e11, "bfloat16": 4.4e11}


# ------------------------------------------------------------------ cases
def _attn(name, op, heads, dtype, seqs, cached, new=(1, 1), block=16, pool="", lens=0, ones=0.0,
          lam="head", norm=True):
    """cached / new: the range of each sequence's cached and new tokens (uniform, drawn from ``lens``);
    ones: share of the sequences that bring a single new token instead. pool "fp8": e4m3 pools with a
    scale per kv head. lam: one number, one value per head, or one per row and head."""
    c = {"op": op, "hq": heads[0], "hkv": heads[1], "d": heads[2], "dtype": dtype, "pool": pool,
         "seqs": seqs, "cached_lo": cached[0], "cached_hi": cached[1], "new_lo": new[0], "new_hi": new[1],
         "block": block, "lens": lens, "ones": ones, "lam": lam, "norm": norm}
    if name:
        c["name"] = name
    return c


def _tab(name, rows, cached, new, width, block=16, ones=0.0, idle=0.0, done=0.0, fresh=0.0, spare=1.0,
         lens=0):
    """A step of ``rows`` table rows: a share ``done`` finishes, ``idle`` brings nothing, ``ones`` one
    token, the rest ``new`` tokens; a share ``fresh`` of the rows that bring tokens are requests that hold
    nothing yet. spare: free blocks, as a multiple of what the step takes (below 1 it cannot be served)."""
    c = {"op": "tables", "rows": rows, "cached_lo": cached[0], "cached_hi": cached[1], "new_lo": new[0],
         "new_hi": new[1], "width": width, "block": block, "ones": ones, "idle": idle, "done": done,
         "fresh": fresh, "spare": spare, "lens": lens}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # The smallest step: eight short chats of OPT-125m's heads as pairs, fp32. Launch latency.
        _attn("decode_short_f32", "decode", (6, 6, 128), "float32", 8, (128, 128)),
        # A few interactive chats on a GQA model of 14/2 pairs of 128: split over the contexts.
        _attn("decode_few_bf16", "decode", (14, 2, 256), "bfloat16", 4, (150, 3900), lens=11),
        # A full ragged batch, one lambda per row (a gate computed from the token).
        _attn("decode_ragged_bf16", "decode", (14, 2, 256), "bfloat16", 128, (256, 8192), lens=3,
              lam="row"),
        # A ragged batch over fp8 pools, heads in pairs of 64.
        _attn("decode_ragged_fp8", "decode", (28, 4, 128), "bfloat16", 128, (256, 8192), lens=3,
              pool="fp8", lam="number"),
        # No sharing of kv heads, a fixed context, fp16: the most bytes per token.
        _attn("decode_mha_f16", "decode", (16, 16, 256), "float16", 64, (2048, 2048)),
        # 512-token chunks of eight long prompts over 4096 cached tokens.
        _attn("prefill_chunks_bf16", "prefill", (32, 8, 128), "bfloat16", 8, (4096, 4096), (512, 512)),
        # A mixed step: ragged prompt chunks beside sequences that bring one token each.
        _attn("prefill_mixed_bf16", "prefill", (14, 2, 256), "bfloat16", 24, (0, 6000), (1, 300), lens=7,
              ones=0.6, lam="row"),
        # One user's new prompt, no sharing of kv heads: time to the first token.
        _attn("prefill_prompt_f16", "prefill", (16, 16, 256), "float16", 1, (0, 0), (777, 777), norm=False,
              lam="number"),
        # Prompts of OPT-125m's heads as pairs, fp32.
        _attn("prefill_short_f32", "prefill", (6, 6, 128), "float32", 8, (0, 0), (17, 512), lens=9),
        # The tables of a decode step: every row one token. Launch latency.
        _tab("tables_step", 128, (256, 8192), (1, 1), 640, ones=1.0, lens=3, spare=4.0),
        # A mixed step: rows that end, idle ones, one-token rows, prompt chunks, new requests.
        _tab("tables_mixed", 256, (0, 6000), (17, 512), 512, ones=0.5, idle=0.1, done=0.1, fresh=0.3,
             lens=7),
        # A batch of long prompts admitted at once: a million slots.
        _tab("tables_admit", 512, (0, 0), (512, 3584), 256, fresh=1.0, lens=5),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    while True:
        op = rng.choice(["decode", "decode", "prefill", "prefill", "tables"])
        block = rng.choice([16, 16, 16, 32])
        lens = rng.randrange(1 << 20)
        if op == "tables":
            rows = _log_int(rng, 1, 1024)
            hi = _log_int(rng, 1, 4096)
            new = (max(1, int(hi * rng.uniform(0.01, 1.0))), hi)
            chi = rng.choice([0, _log_int(rng, 16, 8192)])
            cached = (int(chi * rng.uniform(0.0, 1.0)), chi)
            c = _tab("", rows, cached, new, math.ceil((chi + hi + 1) / block) + rng.randrange(0, 9), block,
                     ones=rng.choice([0.0, 1.0, round(rng.random(), 2)]),
                     idle=rng.choice([0.0, round(0.3 * rng.random(), 2)]),
                     done=rng.choice([0.0, round(0.5 * rng.random(), 2)]),
                     fresh=rng.choice([0.0, 1.0, round(rng.random(), 2)]),
                     spare=rng.choice([1.0, 1.0, 2.5, 0.9]), lens=lens)
            if sum(max(0, n) for n in _steps(c)[2]) <= 1_200_000:
                return c
            continue
        heads = rng.choice(_HEADS)
        dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
        lam = rng.choice(["number", "head", "row"])
        norm = rng.random() < 0.75
        pool, new, ones = "", (1, 1), 0.0
        if op == "decode":
            seqs = _log_int(rng, 1, 128)
            hi = _log_int(rng, 1, 32768 if seqs <= 16 else 8192)
            cached = (max(1, int(hi * rng.uniform(0.03, 1.0))), hi)
            if dtype != "float32" and heads[2] == 128 and rng.random() < 0.4:
                pool = "fp8"
        else:
            seqs = _log_int(rng, 1, 16)
            hi = _log_int(rng, 1, 1024)
            new = (max(1, int(hi * rng.uniform(0.01, 1.0))), hi)
            hi = rng.choice([0, _log_int(rng, 1, 8192)])
            cached = (int(hi * rng.uniform(0.0, 1.0)), hi)
            ones = rng.choice([0.0, 0.0, round(rng.random(), 2)])
        c = _attn("", op, heads, dtype, seqs, cached, new, block, pool, lens, ones, lam, norm)
        w = work(c)
        if w["bytes"] <= _MAX_BYTES and w["flops"] <= _MAX_FLOPS[dtype] and _pool_bytes(c) <= 6e9:
            return c


# ------------------------------------------------------------------ lengths and work
def _lens(case):
    """(cached tokens, new tokens) of every sequence; decode attends to ``cached`` tokens."""
    r = random.Random(case["lens"] * 1000003 + case["seqs"])
    cached = [r.randint(case["cached_lo"], case["cached_hi"]) for _ in range(case["seqs"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    new = [1 if r.random() < case["ones"] else n for n in new]
    if case["op"] == "decode":
        new = [0] * case["seqs"]
    return cached, new


def _steps(case):
    """(tokens, blocks held, new tokens) of every table row; new < 0: the row ends."""
    r = random.Random(case["lens"] * 1000003 + case["rows"])
    lens, held, new = [], [], []
    for _ in range(case["rows"]):
        c, n = r.randint(case["cached_lo"], case["cached_hi"]), r.randint(case["new_lo"], case["new_hi"])
        if r.random() < case["ones"]:
            n = 1
        u = r.random()
        if u < case["done"]:
            n = -1
        elif u < case["done"] + case["idle"]:
            n = 0
        elif r.random() < case["fresh"]:
            c = 0
        lens.append(c)
        held.append(-(-(c + 1) // case["block"]) if c else 0)
        new.append(n)
    return lens, held, new


def _takes(case):
    lens, held, new = _steps(case)
    return [max(h, -(-(c + n + (1 if h == 0 else 0)) // case["block"])) - h if n > 0 else 0
            for c, h, n in zip(lens, held, new)]


def _contexts(case):
    return [c + n for c, n in zip(*_lens(case))]


def _eb(case):
    return 1 if case["pool"] == "fp8" else 4 if case["dtype"] == "float32" else 2


def _num_blocks(case):
    return math.ceil(1.1 * sum(max(1, math.ceil(c / case["block"])) for c in _contexts(case))) + 1


def _pool_bytes(case):
    return 2 * _num_blocks(case) * case["block"] * case["hkv"] * case["d"] * _eb(case)


def work(case):
    """K and V once per kv head, q and out once; two score products over half the head and two value
    products over all of it per visible (row, key). Tables: the rows' state read and written, one entry
    read per block that new tokens lie in, the entries, slots and free blocks that change."""
    if case["op"] == "tables":
        lens, held, new = _steps(case)
        grow = [max(0, n) for n in new]
        touched = sum(-(-(c + n) // case["block"]) - c // case["block"] for c, n in zip(lens, grow) if n)
        taken, freed = sum(_takes(case)), sum(h for h, n in zip(held, new) if n < 0)
        return {"bytes": 8 * sum(grow) + 4 * (touched + 2 * taken + 2 * max(0, freed - taken))
                + 4 * 6 * len(lens), "flops": 0}
    cached, new = _lens(case)
    ctx = _contexts(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    eb, qb = _eb(case), 4 if case["dtype"] == "float32" else 2
    b = 2 * sum(ctx) * hkv * d * eb + 4 * sum(math.ceil(c / case["block"]) for c in ctx) + 4 * len(ctx)
    if case["op"] == "prefill":
        keys = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, new))
        rows = sum(new)
    else:
        keys, rows = sum(ctx), len(ctx)
    return {"bytes": b + 2 * rows * hq * d * qb, "flops": 6 * keys * hq * d}


# ------------------------------------------------------------------ tensors
def _randn(shape, dtype, gen):
    return torch.randn(shape, generator=gen, device=_DEV, dtype=dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).to(_DEV)


def _block_lists(needs, total, seed, width):
    """A padded table of physical blocks in no order, as a pool in use has them, and the blocks left."""
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(needs), width), -1, dtype=torch.int32)
    pos = 0
    for i, n in enumerate(needs):
        table[i, :n] = perm[pos:pos + n]
        pos += n
    return table, perm[pos:]


def prepare(case, seed):
    if case["op"] == "tables":
        return _prepare_tables(case, seed)
    dtype = _DTYPES[case["dtype"]]
    hq, hkv, d, op = case["hq"], case["hkv"], case["d"], case["op"]
    cached, new = _lens(case)
    ctx = _contexts(case)
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    needs = [max(1, math.ceil(c / case["block"])) for c in ctx]
    table, _ = _block_lists(needs, _num_blocks(case), seed, max(needs))
    st = {"case": case, "table": table.to(_DEV), "ctx": _i32(ctx), "max_ctx": max(ctx), "lens": ctx,
          "new": new, "k_scale": None, "v_scale": None}
    shape = (_num_blocks(case), case["block"], hkv, d)
    for name in ("k", "v"):
        if case["pool"] == "fp8":
            scale = torch.rand(hkv, generator=gen, device=_DEV) * 0.01 + 0.01
            x = _randn(shape, torch.bfloat16, gen) / scale.to(torch.bfloat16).view(1, 1, -1, 1)
            st[name + "_scale"], st[name] = scale, x.clamp(-448, 448).to(_FP8)
        else:
            st[name] = _randn(shape, dtype, gen)
    rows = sum(new) if op == "prefill" else case["seqs"]
    st["q"] = _randn((rows, hq, d), dtype, gen)
    st["out"] = torch.empty_like(st["q"])
    r = random.Random(seed)
    lam_shape = {"head": (hq,), "row": (rows, hq)}
    st["lam"] = round(r.uniform(0.2, 0.8), 6) if case["lam"] == "number" else \
        torch.rand(lam_shape[case["lam"]], generator=gen, device=_DEV) * 0.6 + 0.2
    st["weight"] = torch.rand(d, generator=gen, device=_DEV) + 0.5 if case["norm"] else None
    if op == "prefill":
        qsl = [0]
        for n in new:
            qsl.append(qsl[-1] + n)
        st["qsl"], st["max_new"] = _i32(qsl), max(new)
    return st


def _prepare_tables(case, seed):
    lens, held, new = _steps(case)
    grow = [max(0, n) for n in new]
    freed = sum(h for h, n in zip(held, new) if n < 0)
    spare = max(0, math.ceil(case["spare"] * sum(_takes(case))) - freed)
    total = sum(held) + spare
    table, left = _block_lists(held, max(1, total), seed, case["width"])
    free = torch.zeros(max(1, total), dtype=torch.int32)
    free[:spare] = left[:spare]
    rows = len(lens)
    return {"case": case, "table": table.to(_DEV), "held": _i32(held), "lens": _i32(lens), "new": _i32(new),
            "free": free.to(_DEV), "num_free": _i32([spare]),
            "slots": torch.empty(max(1, sum(grow)), dtype=torch.int64, device=_DEV),
            "qsl": torch.empty(rows + 1, dtype=torch.int32, device=_DEV),
            "status": torch.empty(1, dtype=torch.int32, device=_DEV),
            # The state after the step goes to a second set of buffers (a program that keeps the state
            # before the step, to undo it), so a pass can be made again.
            "held_out": torch.empty(rows, dtype=torch.int32, device=_DEV),
            "lens_out": torch.empty(rows, dtype=torch.int32, device=_DEV),
            "num_free_out": torch.empty(1, dtype=torch.int32, device=_DEV)}


# ------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    if not own:
        return _PLAIN[case["op"]](st)
    from cloverinfer_amd import kernels
    if case["op"] == "decode":
        kernels.differential_attention(st["out"], st["q"], st["k"], st["v"], st["table"], st["ctx"],
                                       case["block"], st["max_ctx"], st["lam"], norm_weight=st["weight"],
                                       norm_eps=_EPS, out_scale=_OUT_SCALE, k_scale=st["k_scale"],
                                       v_scale=st["v_scale"])
        return st["out"]
    if case["op"] == "prefill":
        kernels.differential_prefill(st["out"], st["q"], st["k"], st["v"], st["table"], st["ctx"],
                                     st["qsl"], st["max_new"], st["lam"], norm_weight=st["weight"],
                                     norm_eps=_EPS, out_scale=_OUT_SCALE)
        return st["out"]
    kernels.advance_block_tables(st["table"], st["held"], st["lens"], st["new"], st["free"],
                                 st["num_free"], case["block"], st["slots"], st["qsl"], st["status"],
                                 reserve=1, blocks_held_out=st["held_out"], context_lens_out=st["lens_out"],
                                 num_free_out=st["num_free_out"])
    return _tables_out(st["table"], st["held_out"], st["lens_out"], st["free"], st["num_free_out"],
                       st["slots"], st["qsl"], st["status"])


def _tables_out(table, held, lens, free, num_free, slots, qsl, status):
    return {"table": table, "held": held, "lens": lens, "free": free, "num_free": num_free, "slots": slots,
            "qsl": qsl, "status": status}


# ------------------------------------------------------------------ plain forms
def _softmax(x):
    e = torch.exp(x - x.amax(dim=-1, keepdim=True))
    return e / e.sum(dim=-1, keepdim=True)


def _finish(a1, a2, lam, weight, dtype):
    """a1, a2 [rows, hq, d] in 32 bits, lam [rows or 1, hq] or a number."""
    o = a1 - (lam if isinstance(lam, float) else lam.unsqueeze(-1)) * a2
    if weight is not None:
        o = o * torch.rsqrt((o * o).mean(dim=-1, keepdim=True) + _EPS) * weight
    return (o * _OUT_SCALE).to(dtype)


def _gather(st, name, lo, hi, width):
    """Rows [hkv, tokens, d] of sequences lo..hi in 32 bits: [seqs, hkv, tokens, d]."""
    case = st["case"]
    blocks = st["table"][lo:hi, :width].clamp(min=0).long()
    x = st[name][blocks].float()
    if case["pool"] == "fp8":
        x = x * st[name + "_scale"].view(1, 1, 1, -1, 1)
    return x.view(hi - lo, width * case["block"], case["hkv"], case["d"]).transpose(1, 2).contiguous()


def _plain_decode(st):
    case = st["case"]
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["block"]
    half, group, lens = d // 2, hq // hkv, st["lens"]
    scale = 1.0 / math.sqrt(half)
    a = [[], []]
    lo = 0
    while lo < len(lens):  # sequences together, up to 2^29 gathered elements
        hi, longest = lo, 0
        while hi < len(lens) and (hi == lo or (hi + 1 - lo) * max(longest, lens[hi]) * hkv * d <= 1 << 29):
            longest = max(longest, lens[hi])
            hi += 1
        width = -(-longest // bs)
        k, v = _gather(st, "k", lo, hi, width), _gather(st, "v", lo, hi, width)
        q = st["q"][lo:hi].float().view(hi - lo, hkv, group, d)
        hidden = torch.arange(width * bs, device=_DEV).view(1, 1, 1, -1) >= st["ctx"][lo:hi].view(-1, 1, 1, 1)
        for m in range(2):
            km = k[..., m * half:(m + 1) * half].transpose(2, 3).contiguous()
            x = torch.matmul(q[..., m * half:(m + 1) * half].contiguous(), km) * scale
            w = _softmax(x.masked_fill(hidden, -math.inf))
            a[m].append(torch.matmul(w, v).view(hi - lo, hq, d))
        lo = hi
    return _finish(torch.cat(a[0]), torch.cat(a[1]), st["lam"], st["weight"], _DTYPES[case["dtype"]])


def _plain_prefill(st):
    case = st["case"]
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["block"]
    half, group = d // 2, hq // hkv
    scale = 1.0 / math.sqrt(half)
    out = [[], []]
    row = 0
    for s, (c, n) in enumerate(zip(st["lens"], st["new"])):
        width = -(-c // bs)
        k, v = _gather(st, "k", s, s + 1, width)[0], _gather(st, "v", s, s + 1, width)[0]
        q = st["q"][row:row + n].float().view(n, hkv, group, d).permute(1, 2, 0, 3).contiguous()
        q = q.view(hkv, group * n, d)
        last = torch.arange(c - n, c, device=_DEV).repeat(group).view(1, -1, 1)
        hidden = torch.arange(width * bs, device=_DEV).view(1, 1, -1) > last
        for m in range(2):
            km = k[..., m * half:(m + 1) * half].transpose(1, 2).contiguous()
            x = torch.matmul(q[..., m * half:(m + 1) * half].contiguous(), km) * scale
            w = _softmax(x.masked_fill(hidden, -math.inf))
            a = torch.matmul(w, v).view(hkv, group, n, d).permute(2, 0, 1, 3)
            out[m].append(a.reshape(n, hq, d))
        row += n
    return _finish(torch.cat(out[0]), torch.cat(out[1]), st["lam"], st["weight"], _DTYPES[case["dtype"]])


def _plain_tables(st):
    bs = st["case"]["block"]
    table, held, lens, new = st["table"], st["held"].long(), st["lens"].long(), st["new"].long()
    rows, width = table.shape
    free, n_slots = st["free"], st["slots"].numel()
    have = st["num_free"].long()
    zero = torch.zeros(1, dtype=torch.int64, device=_DEV)
    grow = new.clamp(min=0)
    after = lens + grow
    need = torch.where(new > 0, torch.maximum(held, (after + (held == 0).long() + bs - 1) // bs), held)
    take, gone = need - held, torch.where(new < 0, held, torch.zeros_like(held))
    tok = torch.cat([zero, torch.cumsum(grow, 0)])
    taken = torch.cat([zero, torch.cumsum(take, 0)])
    freed = torch.cat([zero, torch.cumsum(gone, 0)])
    total, returned = taken[-1:], freed[-1:]
    status = torch.where(total > have + returned, 1, 0)
    status = torch.where((need.max() > width) & (status == 0), 2, status)
    status = torch.where((tok[-1:] > n_slots) & (status == 0), 3, status)
    ok = status == 0
    cols = torch.arange(width, device=_DEV).view(1, -1)
    # The stack with the returned blocks on top; what a step takes comes from its end.
    size = free.numel() + rows * width
    stack = torch.cat([free, free.new_zeros(rows * width + 1)])
    back = cols < gone.view(-1, 1)
    where = torch.where(back, have + freed[:-1].view(-1, 1) + cols, size)
    stack = stack.scatter(0, where.flatten(), table.flatten())
    fresh = (cols >= held.view(-1, 1)) & (cols < need.view(-1, 1)) & ok
    at = have + returned - 1 - (taken[:-1].view(-1, 1) + cols - held.view(-1, 1))
    table = torch.where(fresh, stack[at.clamp(0, size)], table)
    left = torch.where(ok, have + returned - total, have)
    i = torch.arange(free.numel(), device=_DEV)
    free = torch.where((i >= have) & (i < left), stack[:free.numel()], free)
    t = torch.arange(n_slots, device=_DEV)
    row = torch.searchsorted(tok[1:], t, right=True).clamp(max=rows - 1)
    pos = lens[row] + t - tok[row]
    block = table[row, (pos // bs).clamp(0, width - 1)].long()
    slots = torch.where((t < tok[-1:]) & ok, block * bs + pos % bs, -1)
    live = (new >= 0).long()
    return _tables_out(table, torch.where(ok, need * live, held).int(),
                       torch.where(ok, after * live, lens).int(), free, left.int(), slots,
                       torch.where(ok, tok, 0).int(), status.int())


_PLAIN = {"decode": _plain_decode, "prefill": _plain_prefill, "tables": _plain_tables}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    st = prepare(case, seed)
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["block"]
    cached, new = _lens(case)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=_DEV)
    row = 0
    for s, c in enumerate(_contexts(case)):
        n = new[s] if case["op"] == "prefill" else 1
        pages = st["table"][s, :-(-c // bs)].long()
        kv = []
        for name in ("k", "v"):
            x = st[name].index_select(0, pages).flatten(0, 1)[:c].double()
            kv.append(x if st[name + "_scale"] is None else x * st[name + "_scale"].double()[:, None])
        first = c - n  # position of the first row
        for h in range(hq):
            key, value = kv[0][:, h // (hq // hkv)], kv[1][:, h // (hq // hkv)]
            q = st["q"][row:row + n, h].double()
            lam = st["lam"]
            if not isinstance(lam, float):
                lam = (lam[h].expand(n) if lam.dim() == 1 else lam[row:row + n, h]).double().view(n, 1)
            o = torch.zeros(n, d, dtype=torch.float64, device=_DEV)
            for part, sign in ((slice(0, d // 2), None), (slice(d // 2, d), lam)):
                score = q[:, part].contiguous() @ key[:, part].t().contiguous() * (d // 2) ** -0.5
                if n > 1:
                    score += torch.full((n, c), -math.inf, dtype=torch.float64, device=_DEV).triu(first + 1)
                a = torch.softmax(score, dim=1) @ value.contiguous()
                o = a if sign is None else o - sign * a
            if st["weight"] is not None:
                o = o / torch.sqrt(o.square().mean(dim=1, keepdim=True) + _EPS) * st["weight"].double()
            out[row:row + n, h] = o * _OUT_SCALE
        row += n
    return out
