"""A paged cache held in 4 bits, attention over it, a step's tables and the verification of drafted tokens, stated
plainly in 64 bits on the CPU: what the kernels are tested against."""
from __future__ import annotations

import math
from typing import List, Sequence

import torch

GROUP = 32


def quantize(rows: torch.Tensor):
    """(codes [..., d], step [..., groups], middle [..., groups]) of rows in exact arithmetic; step and middle as
    bfloat16 holds them."""
    codes, steps, middles = [], [], []
    for g in rows.double().split(GROUP, -1):
        low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        step = ((high - low) / 15).float().bfloat16().double()
        step = torch.where(step < 2.0 ** -126, torch.zeros_like(step), step)
        middle = (low + 8 * step).float().bfloat16().double()
        # the nearest whole number to (g - middle) / step: where 64 bits say a border between two, what g - middle lost
        # in its rounding (a g of 2^-60 of the middle, say) still speaks, and only a true border goes to the even one
        size = torch.where(step > 0, step, torch.ones_like(step))
        far = g - middle
        lost = (g - (far - (far - g))) + (-middle - (far - g))
        low_side = torch.floor(far / size)
        over = (far - (low_side + 0.5) * size) + lost
        even = torch.remainder(low_side, 2) == 0
        nearest = torch.where((over > 0) | ((over == 0) & ~even), low_side + 1, low_side)
        code = torch.where(step > 0, nearest + 8, torch.full_like(g, 8.0)).clamp(0, 15)
        bad = ~torch.isfinite(g).all(-1, keepdim=True)
        codes.append(torch.where(bad, torch.zeros_like(code), code))
        nan = torch.full_like(step, float("nan"))
        steps.append(torch.where(bad, nan, step))
        middles.append(torch.where(bad, nan, middle))
    return torch.cat(codes, -1), torch.cat(steps, -1), torch.cat(middles, -1)


def values(codes, step, middle):
    """(step * (code - 8), middle) per channel: their sum is what the cache stands for."""
    d = codes.shape[-1]
    wide = lambda t: t.repeat_interleave(GROUP, -1)[..., :d]  # noqa: E731
    return wide(step) * (codes.double() - 8), wide(middle)


def tile_bytes(page: int, d: int) -> int:
    return page * (d // 2 + 4 * -(-d // GROUP))


def pack(codes, step, middle) -> torch.Tensor:
    """uint8 tiles [..., tile_bytes] of pages [..., page, d]."""
    page, d = codes.shape[-2:]
    c = codes.to(torch.uint8)
    byte = c[..., 0::2] | (c[..., 1::2] << 4)
    parts = [byte[..., g // 2:min(g + GROUP, d) // 2].flatten(-2) for g in range(0, d, GROUP)]
    pairs = torch.stack([step, middle], -1).to(torch.bfloat16).contiguous()
    return torch.cat(parts + [pairs.view(torch.uint8).flatten(-3)], -1)


def unpack(tiles, page: int, d: int):
    at, parts = 0, []
    for g in range(0, d, GROUP):
        wide = min(GROUP, d - g) // 2
        byte = tiles[..., at:at + page * wide].unflatten(-1, (page, wide))
        parts.append(torch.stack([byte & 15, byte >> 4], -1).flatten(-2))
        at += page * wide
    pairs = tiles[..., at:].contiguous().view(torch.bfloat16).unflatten(-1, (page, -1, 2)).double()
    return torch.cat(parts, -1), pairs[..., 0], pairs[..., 1]


def attention(q, k_tiles, v_tiles, table, positions, requests, heads: int, d: int, page: int, scale: float, window):
    """(results [T, heads * d], their bound terms) of tokens one by one: ``requests[t]`` is token t's row of the block
    table.  Bound terms: (A, B, E), A the sum of p |step (c - 8)|, B that plus p |middle|, E an upper bound of what 32-bit
    arithmetic (products added one after the other) may move a score by, all of the token's own row."""
    kv = k_tiles.shape[1]
    out = torch.zeros(q.shape[0], heads, d, dtype=torch.float64)
    a, b, e = torch.zeros_like(out), torch.zeros_like(out), torch.zeros(q.shape[0], heads, 1, dtype=torch.float64)
    for t, r in enumerate(requests):
        if r < 0:
            continue
        pos = int(positions[t])
        lo = 0 if not window else max(0, pos - window + 1)
        pages = [int(p) for p in table[r][:pos // page + 1]]
        k1, k0 = values(*unpack(k_tiles[pages], page, d))
        v1, v0 = values(*unpack(v_tiles[pages], page, d))
        flat = lambda x: x.transpose(0, 1).flatten(1, 2)[:, lo:pos + 1]  # noqa: E731
        k1, k0, v1, v0 = flat(k1), flat(k0), flat(v1), flat(v0)
        for h in range(heads):
            x = q[t].view(heads, d)[h].double()
            g = h // (heads // kv)
            p = torch.softmax(scale * ((k1[g] + k0[g]) @ x), 0)
            out[t, h] = p @ (v1[g] + v0[g])
            a[t, h] = p @ v1[g].abs()
            b[t, h] = p @ (v1[g].abs() + v0[g].abs())
            size = scale * ((k1[g].abs() + k0[g].abs()) @ x.abs()).max()
            e[t, h] = (d + 16) * 2.0 ** -23 * size
    return out.flatten(1), (a.flatten(1), b.flatten(1), e.expand_as(out).flatten(1))


def tables(rows: Sequence[int], held, brought, table, page: int, cap: int, free: Sequence[int] = (), start: int = 0):
    """A step's arrays in plain Python: (q_start, kv_len, positions, requests, slots, block table, table after, next)."""
    wide, n = len(table[0]), len(rows)
    table = [list(r) for r in table]
    block = [[-1] * wide for _ in range(n)]
    q_start, kv_len, positions, requests, slots = [0], [], [], [], []
    for b, (row, h, k) in enumerate(zip(rows, held, brought)):
        for i in range(-(-h // page), -(-(h + k) // page)):
            table[row][i] = free[start]
            start += 1
        pages = -(-(h + k) // page)
        block[b][:pages] = table[row][:pages]
        for pos in range(h, h + k):
            positions.append(pos)
            requests.append(b)
            slots.append(block[b][pos // page] * page + pos % page)
        q_start.append(q_start[-1] + k)
        kv_len.append(h + k)
    rest = cap - len(slots)
    return (q_start, kv_len, positions + [0] * rest, requests + [-1] * rest, slots + [-1] * rest, block, table, start)


def verify(logits, row_start, drafted, uniforms, temperature, draft_probs=None):
    """(tokens, accepted): drafted tokens against the target, request by request."""
    tokens: List[int] = [-1] * logits.shape[0]
    accepted = []
    for b, t in enumerate(temperature):
        first, last = row_start[b], row_start[b + 1] - 1
        r = first
        while True:
            x = logits[r].double()
            if t <= 0:
                best = int(torch.argmax(x))
                if r < last and drafted[r] == best:
                    tokens[r] = drafted[r]
                    r += 1
                    continue
                tokens[r] = best
                break
            p = torch.softmax(x / t, -1)
            if r < last:
                q = torch.zeros_like(p)
                if draft_probs is None:
                    q[drafted[r]] = 1.0
                else:
                    q = draft_probs[r].double()
                if float(uniforms[r][0]) * float(q[drafted[r]]) < float(p[drafted[r]]):
                    tokens[r] = drafted[r]
                    r += 1
                    continue
                less = (p - q).clamp(min=0)
                p = less if float(less.sum()) > 0 else p
            sums = torch.cumsum(p, 0)
            over = (sums > float(uniforms[r][1]) * float(sums[-1])).nonzero()
            tokens[r] = int(over[0]) if len(over) else int((p > 0).nonzero()[-1])
            break
        accepted.append(r - first)
    return tokens, accepted


def tiles_of(lengths: Sequence[int], most: int):
    """(request, first token row, tokens) of tiles of up to ``most`` neighbouring tokens."""
    out, row = [], 0
    for b, n in enumerate(lengths):
        out += [(b, row + i, min(most, n - i)) for i in range(0, n, most)]
        row += n
    return out


def attention_bound(ref, terms, keys: int, dtype) -> torch.Tensor:
    """How far a result may be from the 64-bit one.  bfloat16: half a step of the result (2^-8), of every probability
    times its step (2^-8 of A) and of every probability that goes with a middle (2^-8 of B - A), so 2^-8 of B.  Both
    types: a score that 32-bit sums moved by E moves a probability by up to 2 E of itself (once by itself, once by the sum
    of all; e^x - 1 <= 1.01 x here), the exponential is good for 2^-21 with its argument's rounding (2^-24 of up to 64 log2
    units), and sums over the keys one after the other lose up to 2^-23 a key.  (Portions of prompts round values too,
    another 2^-8 of p |value|: they are held to the same bound, which the roundings' signs leave room for.)"""
    _a, b, e = terms
    assert float(e.max()) < 0.01
    wide = 2 * (1.01 * e + 2.0 ** -21 + 2.0 ** -17) + (keys + 16) * 2.0 ** -23
    if dtype == torch.float32:
        return wide * b + 2.0 ** -23 * ref.abs() + 1e-30
    return 1.01 * 2.0 ** -8 * (ref.abs() + b) + wide * b + 1e-30
