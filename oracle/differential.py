"""Differential attention and the block tables' step, restated on the CPU.

``rows`` is plain float64 torch from the definition: two softmax maps of half
heads over one value, their difference, the per-head norm. ``bound`` is the
error a correct kernel may have on those rows, by arithmetic. ``advance`` runs
the reference's allocator (``oracle.blocks.KVCacheManager`` semantics: a LIFO
list popped from its end) call by call, as a step of the device tables does it
at once. Nothing here is used by the product.
"""
from __future__ import annotations

import math

import torch

TABLES_OK, TABLES_NO_BLOCKS, TABLES_ROW_FULL, TABLES_NO_SLOTS, TABLES_BAD_STATE = range(5)


def rows(q, k, v, limits, lam, weight=None, eps=1e-5, out_scale=1.0, scale=None):
    """q [n, H, D], k/v [L, Hkv, D] (any dtype), limits [n]: row i sees tokens
    < limits[i] (an iterable of visible token indices instead of a number is
    taken as it is). lam [n, H] or [H] or a number. Returns a dict of float64
    tensors: out, o, and what ``bound`` needs."""
    n, hq, d = q.shape
    half, group = d // 2, hq // k.shape[1]
    scale = 1.0 / math.sqrt(half) if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    lam = torch.as_tensor(lam, dtype=torch.float64).expand(n, hq)
    o = torch.zeros(n, hq, d, dtype=torch.float64)
    mass = torch.zeros_like(o)      # sum of weights times |v|, both maps
    peak = torch.zeros(n, hq, 1, dtype=torch.float64)   # largest sum |q_i k_i| * scale
    loose = torch.zeros_like(o)     # sum of |v| over the visible tokens, both maps
    seen = torch.zeros(n, 1, 1, dtype=torch.float64)
    for i in range(n):
        idx = torch.arange(limits[i]) if isinstance(limits[i], int) else torch.as_tensor(limits[i])
        seen[i] = len(idx)
        if len(idx) == 0:
            continue
        ki = k[idx].repeat_interleave(group, dim=1).transpose(0, 1)  # [H, L, D]
        vi = v[idx].repeat_interleave(group, dim=1).transpose(0, 1)
        for m in range(2):
            part = slice(m * half, (m + 1) * half)
            s = torch.matmul(ki[..., part], q[i, :, part].unsqueeze(-1)).squeeze(-1) * scale
            big = torch.matmul(ki[..., part].abs(), q[i, :, part].abs().unsqueeze(-1))
            w = torch.softmax(s, dim=-1)
            a = torch.matmul(w.unsqueeze(1), vi).squeeze(1)
            sign = 1.0 if m == 0 else -lam[i].unsqueeze(-1)
            o[i] += sign * a
            size = 1.0 if m == 0 else lam[i].abs().unsqueeze(-1)
            mass[i] += size * torch.matmul(w.unsqueeze(1), vi.abs()).squeeze(1)
            loose[i] += size * vi.abs().sum(dim=1)
            peak[i] = torch.maximum(peak[i], big.amax(dim=1) * abs(scale))
    out, norm = o * out_scale, None
    if weight is not None:
        norm = torch.sqrt(o.square().mean(dim=-1, keepdim=True) + eps)
        out = out / norm * weight.double()
    return {"out": out, "o": o, "mass": mass, "peak": peak, "loose": loose, "seen": seen,
            "norm": norm, "weight": weight, "out_scale": out_scale, "half": half}


def bound(r, dtype, weight_bits=0.0, loose_step=0.0):
    """Largest error of a kernel that holds scores, weights and sums in fp32.

    u = 2^-24 is half a step of fp32. A score is a sum of ``half`` products
    (error <= (half + 2) u times the sum of their magnitudes, ``peak``), and its
    exponent takes two more roundings of its own size and the exponential one
    step: a weight is off by the factor 1 + e with e <= (half + 6) u peak + 4 u.
    The sums over ``seen`` tokens run over at most seen / 16 + 64 additions in
    a row (16 tokens a step, then the merges), for the row sum and for the
    context, so a context is off by at most (2 e + 2 (seen / 16 + 64) u) times
    ``mass``. ``weight_bits``: the relative error of a weight that is stored in
    fewer bits for the product with V; ``loose_step``: the absolute one (half a
    subnormal step), which every token's |v| takes: ``loose``.
    The norm divides by sqrt(mean(o^2) + eps), which moves by at most the root
    mean square of the error. The rounding of out is half a step of its type.
    """
    u = 2.0 ** -24
    e = (r["half"] + 6) * u * r["peak"] + 4 * u
    err = (2 * e + 2 * (r["seen"] / 16 + 64) * u + weight_bits) * r["mass"] + loose_step * r["loose"]
    scale = abs(r["out_scale"])
    if r["norm"] is not None:
        rms = err.square().mean(dim=-1, keepdim=True).sqrt()
        err = (err + r["o"].abs() * (rms / r["norm"])) / r["norm"] * r["weight"].double().abs()
        # where the error is not small against the norm, the second order too
        err = err * (1 + 2 * rms / r["norm"])
    err = err * scale + 8 * u * r["out"].abs()
    half_step = {torch.float32: u, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    tiny = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}[dtype]
    return err + half_step * (r["out"].abs() + err) + tiny


def advance(table, held, lens, new, stack, block_size, num_slots, width, capacity, reserve=1):
    """One step, sequentially: (status, table, held, lens, stack, slots, qsl) as
    lists; ``table`` is a list of rows of ``width`` entries."""
    table, held, lens, free = [list(r) for r in table], list(held), list(lens), list(stack)
    kept = (TABLES_OK, [list(r) for r in table], list(held), list(lens), list(stack),
            [-1] * num_slots, [0] * (len(held) + 1))

    def refuse(status):
        return (status,) + kept[1:]

    for h, n in zip(held, lens):
        if h < 0 or h > width or n < 0 or n > h * block_size:
            return refuse(TABLES_BAD_STATE)
    for r, n in enumerate(new):
        if n < 0:
            free += table[r][:held[r]]
    if len(free) > capacity:
        return refuse(TABLES_BAD_STATE)
    need = [max(h, -(-(c + n + (reserve if h == 0 else 0)) // block_size)) if n > 0 else h
            for h, c, n in zip(held, lens, new)]
    if sum(need) - sum(held) > len(free):
        return refuse(TABLES_NO_BLOCKS)
    if any(x > width for x in need):
        return refuse(TABLES_ROW_FULL)
    if sum(max(0, n) for n in new) > num_slots:
        return refuse(TABLES_NO_SLOTS)
    slots, qsl = [], [0]
    for r, n in enumerate(new):
        if n < 0:
            held[r] = lens[r] = 0
        elif n > 0:
            while held[r] < need[r]:
                table[r][held[r]] = free.pop()
                held[r] += 1
            for p in range(lens[r], lens[r] + n):
                slots.append(table[r][p // block_size] * block_size + p % block_size)
            lens[r] += n
        qsl.append(qsl[-1] + max(0, n))
    return (TABLES_OK, table, held, lens, free, slots + [-1] * (num_slots - len(slots)), qsl)
