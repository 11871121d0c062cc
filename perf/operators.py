"""Operators of a step over a paged cache held in 4 bits, with drafted tokens, as a user's program calls
them, beside their plain forms in elementary tensor operations.

``append``     the step's keys and values are rounded to 4 bits at their slots of the paged cache and read
               back as the values they stand for;
``attention``  causal attention (a window, too) of the step's tokens over their requests' pages: single
               tokens, a few drafted tokens each, portions of prompts;
``tables``     positions, requests, slots and block tables of a step from the requests' lengths, with new
               pages taken from a list of free ones;
``verify``     drafted tokens against the target's probabilities: how many stay, and the token behind them.

The cache: a page of one key/value head is one tile of bytes: for every group of 32 channels (the last may
be shorter) the codes of ``page_size`` rows (two channels a byte, channel 2i in the low half of byte i), then
for every row its groups' two bfloat16 numbers (step, middle).  A code c stands for middle + step * (c - 8).
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
GROUP = 32                       # channels that share a step and a middle
SMALLEST = 2.0 ** -126           # a step below the smallest normal number counts as none


# ------------------------------------------------------------------------------------- the cases
def _append(name, tokens, heads, head_dim, dtype="bfloat16", page=64, skipped=0):
    return dict(name=name, op="append", tokens=tokens, heads=heads, head_dim=head_dim, dtype=dtype, page=page,
                skipped=skipped)


def _attention(name, requests, new, context, heads, kv_heads, head_dim, dtype="bfloat16", page=64, window=0,
               ragged=True):
    return dict(name=name, op="attention", requests=requests, new=new, context=context, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, page=page, window=window, ragged=ragged)


def _tables(name, requests, new, context, page, positions):
    return dict(name=name, op="tables", requests=requests, new=new, context=context, page=page, positions=positions)


def _verify(name, requests, drafts, vocab, temperature, draft="probabilities"):
    return dict(name=name, op="verify", requests=requests, drafts=drafts, vocab=vocab, temperature=temperature,
                draft=draft)


def listed():
    return [
        # a decode step of 64 requests at GPT-2 small's heads: a token each, some rows are padding
        _append("append_step", 64, 12, 64, skipped=3),
        # a full prompt step at GPT-2 XL's heads
        _append("append_prompts", 2048, 25, 64),
        # one user at a chat, GPT-2 small's heads: the smallest call, latency counts
        _attention("one_user", 1, 1, 1000, 12, 12, 64),
        # a loaded server near the longest contexts, GPT-2 XL's heads
        _attention("batch_64", 64, 1, 1000, 25, 25, 64),
        # long documents with grouped heads
        _attention("long_documents", 8, 1, 32749, 32, 8, 128),
        # five tokens a request (four drafted ones and the one before them), GPT-2 medium's heads
        _attention("drafted", 24, 5, 777, 16, 16, 64),
        # portions of long prompts, each behind what its request holds already
        _attention("portions", 4, 512, 4000, 16, 16, 64),
        # evaluation of texts in 32 bits
        _attention("texts_float32", 3, 301, 301, 12, 12, 64, dtype="float32"),
        # what a loaded server's decode step needs in tables
        _tables("tables_step", 64, 1, 1000, 64, 1024),
        # prompts of hundreds of requests with small pages and long contexts
        _tables("tables_prompts", 250, 250, 20000, 16, 32768),
        # one user with three drafted tokens, the largest logit wins
        _verify("verify_one", 1, 3, 50257, 0.0),
        # a loaded server, four drafted tokens each, at temperature
        _verify("verify_64", 64, 4, 50257, 0.8),
    ]


def _between(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


HEADS = [(4, 4, 16), (3, 3, 32), (12, 12, 64), (16, 16, 64), (25, 25, 64), (32, 8, 128), (16, 2, 64), (8, 1, 128),
         (10, 5, 96), (6, 3, 80), (40, 8, 128), (9, 9, 112)]


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "tables", "verify"])
    page = rng.choice([16, 32, 48, 64, 64, 128])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    dtype = "float32" if rng.random() < 0.25 else "bfloat16"
    if op == "append":
        tokens = _between(rng, 1, 2048)
        case = _append("", tokens, kv_heads, head_dim, dtype, page, skipped=rng.choice([0, 0, tokens // 9]))
    elif op == "attention":
        kind = rng.choice(["single", "single", "few", "prompt"])
        new = 1 if kind == "single" else rng.randint(2, 9) if kind == "few" else _between(rng, 10, 1000)
        requests = _between(rng, 1, 100 if kind == "single" else 40 if kind == "few" else 6)
        # no more cached numbers than the largest listed case has, no more scores than the prompts' one
        most = 1.2e8 / (requests * kv_heads * head_dim)
        most = min(most, (1.2e8 if dtype == "bfloat16" else 1.2e7) / (requests * heads * new), 40000)
        context = _between(rng, new, max(new, int(most)))
        window = _between(rng, 1, context) if rng.random() < 0.2 else 0
        case = _attention("", requests, new, context, heads, kv_heads, head_dim, dtype, page, window,
                          rng.random() < 0.8)
    elif op == "tables":
        new = _between(rng, 1, 500)
        positions = _between(rng, max(600, new), 32768)
        case = _tables("", _between(rng, 1, 250), new, _between(rng, 1, positions - new) if positions > new else 0,
                       page, positions)
    else:
        requests = _between(rng, 1, 64)
        case = _verify("", requests, rng.randint(1, 4 if requests > 30 else 8), _between(rng, 500, 50257),
                       rng.choice([0.0, 0.6, 1.0, 1.3]), rng.choice(["probabilities", "probabilities", "tokens"]))
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------- the work
def _spread(n, count, ragged, low=1):
    """Lengths of a batch: all ``n``, or spread between half and all of it (the first is whole)."""
    return [n if not ragged else max(low, n - (i * 7919) % (n // 2 + 1)) for i in range(count)]


def _lengths(case):
    """(tokens held, tokens brought) of each request."""
    if case["op"] == "tables":
        new = _spread(case["new"], case["requests"], case["new"] > 1, low=0)
        return _spread(case["context"], case["requests"], True, low=0), new
    new = _spread(case["new"], case["requests"], case["ragged"])
    total = _spread(case["context"], case["requests"], case["ragged"])
    return [max(0, t - n) for t, n in zip(total, new)], new


def _row_bytes(head_dim):
    return head_dim // 2 + 4 * -(-head_dim // GROUP)


def work(case):
    op = case["op"]
    if op == "append":
        n, h, d = case["tokens"] - case["skipped"], case["heads"], case["head_dim"]
        size = 2 if case["dtype"] == "bfloat16" else 4
        # keys and values in, their 4-bit rows out, and back as 32-bit numbers
        return {"bytes": 2 * n * h * (d * size + _row_bytes(d) + 4 * d) + 4 * case["tokens"], "flops": 2 * n * h * d * 7}
    if op == "attention":
        held, new = _lengths(case)
        d, window = case["head_dim"], case["window"]
        size = 2 if case["dtype"] == "bfloat16" else 4
        keys = pairs = 0
        for a, n in zip(held, new):
            keys += a + n if not window else min(a + n, n + window - 1)
            # token i sees a + i + 1 keys, or the window's
            short = n if not window else max(0, min(n, window - a - 1))
            pairs += short * a + short * (short + 1) // 2 + (n - short) * window
        rows = sum(new) * case["heads"] * d
        return {"bytes": 2 * keys * case["kv_heads"] * _row_bytes(d) + 2 * rows * size,
                "flops": 4 * pairs * case["heads"] * d}
    if op == "tables":
        held, new = _lengths(case)
        b, t, wide = len(held), sum(new), -(-case["positions"] // case["page"])
        pages = sum(-(-(a + n) // case["page"]) for a, n in zip(held, new))
        return {"bytes": 4 * (3 * b + pages + b * wide + 3 * t + 2 * b), "flops": 4 * t}
    rows = case["requests"] * (case["drafts"] + 1)
    # every logit once; of the draft, the row of each request that is drawn from and a number a token
    sampled = case["temperature"] > 0 and case["draft"] == "probabilities"
    return {"bytes": 4 * case["vocab"] * (rows + (case["requests"] if sampled else 0)) + 16 * rows,
            "flops": 4 * rows * case["vocab"]}


# ------------------------------------------------------------------------------------- plain forms
def _groups(x):
    """Rows [..., head_dim] in groups of 32 channels [..., groups, 32]; a short last group is filled with
    its first channel (which changes neither its smallest nor its largest number)."""
    d = x.shape[-1]
    short = -d % GROUP
    if short:
        first = x[..., d - d % GROUP:d - d % GROUP + 1]
        x = torch.cat([x, first.expand(*first.shape[:-1], short)], -1)
    return x.reshape(*x.shape[:-1], -1, GROUP)


def _quantize(x):
    """Codes [..., head_dim] and (step, middle) [..., groups, 2] (bfloat16) of rows; in 64 bits, since a
    quotient next to the border of two codes goes to one of them."""
    g = _groups(x.double())
    low, high = g.amin(-1), g.amax(-1)
    step = ((high - low) / torch.full_like(low, 15.0)).to(torch.bfloat16).double()
    step = torch.where(step < SMALLEST, torch.zeros_like(step), step)
    middle = (low + 8.0 * step).to(torch.bfloat16).double()
    size = torch.where(step > 0, step, torch.full_like(step, math.inf))
    code = (torch.round((g - middle[..., None]) / size[..., None]) + 8.0).clamp(0.0, 15.0)
    return code.flatten(-2)[..., :x.shape[-1]], torch.stack([step, middle], -1).to(torch.bfloat16)


def _values(code, params):
    """What codes [..., head_dim] stand for, in 32 bits."""
    p = params.float()
    p = p.repeat_interleave(GROUP, -2)[..., :code.shape[-1], :]
    return p[..., 1] + p[..., 0] * (code.float() - 8.0)


def _pack(code, params):
    """Tiles of bytes [pages, heads, tile] of codes [pages, heads, page, head_dim] and their parameters."""
    code = code.to(torch.uint8)
    rows = code[..., 0::2] | (code[..., 1::2] << 4)
    whole = code.shape[-1] // GROUP * (GROUP // 2)               # bytes of a row's whole groups
    parts = [rows[..., :whole].unflatten(-1, (-1, GROUP // 2)).transpose(-2, -3).flatten(2),
             rows[..., whole:].flatten(2), params.contiguous().view(torch.uint8).flatten(2)]
    return torch.cat(parts, -1).contiguous()


def _tile_parts(tiles, page, head_dim):
    """Views of tiles [..., tile]: codes of the whole groups [..., groups, page, 16], of the short one [..., page,
    bytes] and the parameters' bytes [..., page, 4 * groups]."""
    whole = head_dim // GROUP * page * (GROUP // 2)
    codes = page * head_dim // 2
    return (tiles[..., :whole].unflatten(-1, (head_dim // GROUP, page, GROUP // 2)),
            tiles[..., whole:codes].unflatten(-1, (page, head_dim % GROUP // 2)),
            tiles[..., codes:].unflatten(-1, (page, -1)))


def _unpack(tiles, page, head_dim):
    """Codes and parameters of tiles [..., tile]."""
    whole, short, params = _tile_parts(tiles, page, head_dim)
    rows = torch.cat([whole.transpose(-2, -3).flatten(-2), short], -1)
    code = torch.stack([rows & 15, rows >> 4], -1).flatten(-2)
    return code, params.contiguous().view(torch.bfloat16).unflatten(-1, (-1, 2))


def _plain_append(s):
    page, d, h = s["page"], s["head_dim"], s["heads"]
    live = s["slots"] >= 0
    rows = torch.where(live)[0]
    slots = s["slots"][rows].long()
    out = []
    for x, tiles, back in ((s["k"], s["k_tiles"], s["k_back"]), (s["v"], s["v_tiles"], s["v_back"])):
        code, params = _quantize(x[rows].unflatten(1, (h, d)))
        c = code.to(torch.uint8)
        at = (slots // page, slots % page)
        byte = c[..., 0::2] | (c[..., 1::2] << 4)
        whole, short, pairs = _tile_parts(tiles, page, d)
        cut = d // GROUP * (GROUP // 2)
        whole[at[0], :, :, at[1]] = byte[..., :cut].unflatten(-1, (-1, GROUP // 2))
        short[at[0], :, at[1]] = byte[..., cut:]
        pairs[at[0], :, at[1]] = params.contiguous().view(torch.uint8).flatten(2)
        back[rows] = _values(code, params).flatten(1)
        out.append(back)
    return out


def _plain_attention(s):
    d, page, h, kv = s["head_dim"], s["page"], s["heads"], s["kv_heads"]
    new, total = s["new"], s["total"]
    b, most = new.shape[0], s["longest_new"]
    table = s["block_table"].long().clamp(min=0)

    def cached(tiles):                                         # [requests, kv heads, positions, head_dim]
        t = tiles[table].permute(0, 2, 1, 3)
        code, params = _unpack(t, page, d)
        return _values(code, params).flatten(2, 3)
    k, v = cached(s["k_tiles"]), cached(s["v_tiles"])
    place = torch.arange(most, device=new.device)
    row = (s["first"][:, None] + place).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().unflatten(2, (kv, h // kv, d)).permute(0, 2, 3, 1, 4)   # [b, kv, group, most, d]
    at = (total - new)[:, None] + place                                             # positions of the tokens
    key = torch.arange(k.shape[2], device=new.device)
    seen = (key[None, None] <= at[..., None])
    if s["window"]:
        seen &= key[None, None] > at[..., None] - s["window"]
    # (what lies behind a request's last position is not looked at, whatever the pages hold there)
    v = torch.where((key[None] < total[:, None])[:, None, :, None], v, torch.zeros_like(v))
    score = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)).mul_(s["scale"])
    score = torch.where(seen[:, None, None].expand(b, kv, h // kv, most, -1).flatten(2, 3), score,
                        torch.full_like(score, -math.inf))
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(score, v) / score.sum(-1, keepdim=True)
    o = o.unflatten(2, (h // kv, most)).permute(0, 3, 1, 2, 4).flatten(2)            # [b, most, heads * d]
    live = place[None] < new[:, None]
    s["out"][row[live]] = o[live].to(s["out"].dtype)
    return s["out"]


def _plain_tables(s):
    page, held, new = s["page"], s["held"], s["brought"]
    wide, b, cap = s["tables"].shape[1], held.shape[0], s["slots"].shape[0]
    have, want = (held + page - 1) // page, (held + new + page - 1) // page
    taken = want - have
    before = torch.cumsum(taken, 0) - taken
    place = torch.arange(wide, device=held.device)[None]
    rows = s["tables"][s["rows"].long()]
    fresh = (place >= have[:, None]) & (place < want[:, None])
    index = (s["free_start"] + before[:, None] + place - have[:, None]).clamp(0, s["free_pages"].shape[0] - 1)
    rows = torch.where(fresh, s["free_pages"][index.long()], rows)
    s["tables"][s["rows"].long()] = rows
    s["block_table"].copy_(torch.where(place < want[:, None], rows, torch.full_like(rows, -1)))
    ends = torch.cumsum(new, 0)
    s["q_start"][0] = 0
    s["q_start"][1:] = ends
    s["kv_len"].copy_(held + new)
    token = torch.arange(cap, device=held.device)
    live = token < ends[-1]
    request = torch.searchsorted(ends, token, right=True).clamp(max=b - 1)
    at = held[request] + token - (ends - new)[request]
    zero = torch.zeros_like(at)
    at = torch.where(live, at, zero)
    slot = s["block_table"][request, (at // page).clamp(max=wide - 1).long()] * page + at % page
    s["positions"].copy_(at)
    s["seq_of_token"].copy_(torch.where(live, request, zero - 1))
    s["slots"].copy_(torch.where(live, slot, zero - 1))
    s["free_next"].copy_(s["free_start"] + taken.sum())
    return _tables_out(s)


def _tables_out(s):
    return [s[n] for n in ("q_start", "kv_len", "positions", "seq_of_token", "slots", "block_table", "tables",
                           "free_next")]


def _plain_verify(s):
    rows, vocab = s["logits"].shape
    b = s["temperature"].shape[0]
    n = s["row_start"][1:] - s["row_start"][:-1] - 1                        # drafted tokens of each request
    request = torch.repeat_interleave(torch.arange(b, device=n.device), n.long() + 1, output_size=rows)
    t = s["temperature"][request].double()
    greedy = t <= 0
    best = s["logits"].argmax(-1)                                           # (ties: the lowest index)
    x = s["logits"].double() / torch.where(greedy, torch.ones_like(t), t)[:, None]
    p = (x - x.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    drafted = s["drafted"].long().clamp(min=0)
    mine = p.gather(1, drafted[:, None])[:, 0]
    theirs = torch.ones_like(mine) if s["draft_probs"] is None else \
        s["draft_probs"].gather(1, drafted[:, None])[:, 0].double()
    u = s["uniforms"].double()
    last = s["row_start"][1:][request] - 1 == torch.arange(rows, device=n.device)
    stays = torch.where(greedy, drafted == best, u[:, 0] * theirs < mine) & ~last
    # a token stays when it and all before it do
    place = torch.arange(rows, device=n.device) - s["row_start"][request]
    gone = torch.where(stays, rows, place)
    accepted = torch.full((b,), rows, device=n.device).scatter_reduce(0, request, gone.long(), "amin")
    final = (s["row_start"][:-1] + accepted).long()
    w = p[final]
    rejected = (accepted < n)[:, None]
    if s["draft_probs"] is None:
        less = w.scatter(1, drafted[final][:, None], 0.0)
    else:
        less = (w - s["draft_probs"][final].double()).clamp(min=0.0)
    left = torch.where(rejected, less, w)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, w)
    sums = torch.cumsum(left, -1)
    drawn = (sums > u[final, 1:] * sums[:, -1:]).to(torch.uint8).argmax(-1)
    chosen = torch.where(greedy[final], best[final], drawn)
    tokens = torch.where(place < accepted[request], s["drafted"].long(), torch.full_like(drafted, -1))
    tokens[final] = chosen
    s["tokens"].copy_(tokens)
    s["accepted"].copy_(accepted)
    return [s["tokens"], s["accepted"]]


# ------------------------------------------------------------------------------------ 64-bit forms
def _exact_rows(x):
    """What rows [..., head_dim] are worth once they have been through 4 bits, in 64 bits but for the step
    and the middle, which the cache holds in bfloat16."""
    parts = []
    for g in x.split(GROUP, -1):
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        step = ((high - low) / 15).bfloat16().double()     # (by way of 32 bits, as a conversion goes)
        step[step < SMALLEST] = 0
        middle = (low + 8 * step).bfloat16().double()
        code = torch.where(step > 0, ((g - middle) / step).round() + 8, torch.full_like(g, 8.0))
        parts.append(middle + step * (code.clamp(0, 15) - 8))
    return torch.cat(parts, -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        out = []
        for x, back in ((s["k"], s["k_back"]), (s["v"], s["v_back"])):
            back = back.double()
            for i, slot in enumerate(s["slots"].tolist()):
                if slot >= 0:
                    back[i] = _exact_rows(x[i].double().view(s["heads"], s["head_dim"])).view(-1)
            out.append(back)
        return out
    if case["op"] != "attention":
        return None                                            # whole numbers
    d, page, h, kv = s["head_dim"], s["page"], s["heads"], s["kv_heads"]
    out = s["out"].double()
    group = h // kv
    row = 0
    for b, (n, total) in enumerate(zip(s["new"].tolist(), s["total"].tolist())):
        pages = s["block_table"][b, :-(-total // page)].long()
        cached = []
        for tiles in (s["k_tiles"][pages], s["v_tiles"][pages]):
            raw = tiles.permute(1, 0, 2)                                        # [kv, pages, tile]
            edge = [page * min(g * GROUP, d) // 2 for g in range(-(-d // GROUP) + 1)]
            byte = torch.cat([raw[..., i:j].reshape(kv, raw.shape[1] * page, -1) for i, j in zip(edge, edge[1:])], -1)
            byte = byte[:, :total]
            par = raw[..., page * d // 2:].contiguous().view(torch.bfloat16).reshape(kv, -1, -(-d // GROUP), 2)
            par = par[:, :total].double()
            value = torch.empty(kv, total, d, dtype=torch.float64, device=raw.device)
            value[..., 0::2], value[..., 1::2] = byte % 16, byte // 16
            for g in range(par.shape[2]):
                part = value[..., g * GROUP:(g + 1) * GROUP]
                part.sub_(8).mul_(par[:, :, g, :1]).add_(par[:, :, g, 1:])
            cached.append(value)
        k, v = cached
        at = torch.arange(total - n, total, device=k.device)
        key = torch.arange(total, device=k.device)
        hidden = key[None] > at[:, None]
        if s["window"]:
            hidden |= key[None] <= at[:, None] - s["window"]
        for head in range(h):
            q = s["q"][row:row + n, head * d:(head + 1) * d].double()
            w = (q @ k[head // group].T * s["scale"]).masked_fill(hidden, -math.inf)
            out[row:row + n, head * d:(head + 1) * d] = torch.softmax(w, -1) @ v[head // group]
        row += n
    return out


# ------------------------------------------------------------------------------------------ inputs
def _rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _rows(g, n, heads, d):
    """Keys or values as projections make them: each head has channels of its own size and offset."""
    x = torch.randn(n, heads, d, generator=g, device="cuda")
    wide = torch.exp(0.5 * torch.randn(heads, d, generator=g, device="cuda"))
    return x * wide + 0.5 * torch.randn(heads, d, generator=g, device="cuda")


def _pages(g, count, of):
    """``count`` different pages of a pool of ``of``, in no order."""
    return torch.randperm(of, generator=g, device="cuda")[:count].to(torch.int32)


def _status():
    return torch.zeros(4, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, op = _rng(seed), case["op"]
    s = dict(case)
    s["status"] = _status()
    if op == "append":
        n, h, d, page = case["tokens"], case["heads"], case["head_dim"], case["page"]
        dtype = DTYPES[case["dtype"]]
        # (columns of a fused product: queries, keys, values side by side)
        fused = torch.cat([_rows(g, n, h, d).flatten(1) for _ in range(3)], 1).to(dtype)
        s["k"], s["v"] = fused[:, h * d:2 * h * d], fused[:, 2 * h * d:]
        pages = -(-n // page) + 3
        tile = page * _row_bytes(d)
        for name in ("k_tiles", "v_tiles"):
            s[name] = torch.zeros(pages, h, tile, dtype=torch.uint8, device="cuda")
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:n]
        if n > 256:                                            # prompts fill pages in order
            slots = (_pages(g, pages, pages).long()[:, None] * page +
                     torch.arange(page, device="cuda")[None]).flatten()[:n]
        if case["skipped"]:
            slots[torch.randperm(n, generator=g, device="cuda")[:case["skipped"]]] = -1
        s["slots"] = slots.to(torch.int32)
        s["k_back"] = torch.zeros(n, h * d, device="cuda")
        s["v_back"] = torch.zeros(n, h * d, device="cuda")
    elif op == "attention":
        held, new = _lengths(case)
        total = [a + n for a, n in zip(held, new)]
        d, kv, page = case["head_dim"], case["kv_heads"], case["page"]
        wide = -(-max(total) // page)
        count = sum(-(-t // page) for t in total)
        pool = count + 5
        for name in ("k_tiles", "v_tiles"):
            x = _rows(g, pool * page, kv, d).unflatten(0, (pool, page)).transpose(1, 2)
            s[name] = _pack(*_quantize(x))
            del x
        s["num_pages"] = pool
        order = _pages(g, count, pool).tolist()
        table, at = [], 0
        for t in total:
            n = -(-t // page)
            table.append(order[at:at + n] + [-1] * (wide - n))
            at += n
        cuda = dict(dtype=torch.int32, device="cuda")
        s["block_table"] = torch.tensor(table, **cuda)
        s["new"] = torch.tensor(new, device="cuda")
        s["total"] = torch.tensor(total, device="cuda")
        s["first"] = torch.cumsum(s["new"], 0) - s["new"]
        s["longest_new"], s["longest"] = max(new), max(total)
        s["positions"] = torch.tensor([a + i for a, n in zip(held, new) for i in range(n)], **cuda)
        # tiles: up to 128 rows (tokens times the heads that share keys and values) of one request
        most = max(1, 128 * kv // case["heads"])
        tiles, row = [], 0
        for b, n in enumerate(new):
            tiles += [(b, row + i, min(most, n - i)) for i in range(0, n, most)]
            row += n
        s["tile_req"], s["tile_row0"], s["tile_rows"] = torch.tensor(tiles, **cuda).t().contiguous().unbind(0)
        s["tile_most"] = min(most, max(new))
        dtype = DTYPES[case["dtype"]]
        x = 1.5 * torch.randn(sum(new), (case["heads"] + 2 * kv) * d, generator=g, device="cuda")
        s["q"] = x.to(dtype)[:, :case["heads"] * d]
        s["scale"] = 1.0 / math.sqrt(d)
        s["out"] = torch.zeros(sum(new), case["heads"] * d, dtype=dtype, device="cuda")
    elif op == "tables":
        held, new = _lengths(case)
        b, page = len(held), case["page"]
        wide = -(-case["positions"] // page)
        have = [-(-a // page) for a in held]
        fresh = sum(-(-(a + n) // page) for a, n in zip(held, new)) - sum(have)
        lanes = b + 3
        cuda = dict(dtype=torch.int32, device="cuda")
        pages = _pages(g, sum(have) + fresh + 8, sum(have) + fresh + 8)
        s["rows"] = _pages(g, b, lanes)                        # the requests' rows among all rows
        tables, at = torch.full((lanes, wide), -1, dtype=torch.int32), 0
        order, rows = pages.cpu(), s["rows"].tolist()
        for row, n in zip(rows, have):
            tables[row, :n] = order[at:at + n]
            at += n
        s["tables"] = tables.cuda()
        s["free_pages"] = pages[at:].contiguous()
        s["free_start"] = torch.tensor([2], **cuda)
        s["free_next"] = torch.zeros(1, **cuda)
        s["held"], s["brought"] = torch.tensor(held, **cuda), torch.tensor(new, **cuda)
        cap = sum(new) + 5                                     # (some token rows stay unused)
        for name, n in (("positions", cap), ("seq_of_token", cap), ("slots", cap), ("kv_len", b), ("q_start", b + 1)):
            s[name] = torch.zeros(n, **cuda)
        s["block_table"] = torch.zeros(b, wide, **cuda)
    else:
        n, vocab = case["drafts"], case["vocab"]
        cuda = dict(dtype=torch.int32, device="cuda")
        counts = [n if i == 0 else n - (i * 7919) % 2 for i in range(case["requests"])]
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c + 1)
        rows = starts[-1]
        s["row_start"] = torch.tensor(starts, **cuda)
        s["logits"] = 2.5 * torch.randn(rows, vocab, generator=g, device="cuda")
        t = torch.full((case["requests"],), float(case["temperature"]), device="cuda")
        s["temperature"] = t
        # the draft: the target's logits with some noise, tokens drawn from it (or its largest)
        near = s["logits"] + 0.8 * torch.randn(rows, vocab, generator=g, device="cuda")
        probs = torch.softmax(near / (case["temperature"] or 1.0), -1)
        if case["draft"] == "tokens" or case["temperature"] == 0.0:
            s["drafted"] = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.7, s["logits"].argmax(-1),
                                       near.argmax(-1)).to(torch.int32)
        else:
            s["drafted"] = torch.multinomial(probs, 1, generator=g)[:, 0].to(torch.int32)
        s["draft_probs"] = None if case["draft"] == "tokens" else probs
        s["uniforms"] = torch.rand(rows, 2, generator=g, device="cuda")
        s["tokens"] = torch.zeros(rows, **cuda)
        s["accepted"] = torch.zeros(case["requests"], **cuda)
    return s


# ------------------------------------------------------------------------------------------ a pass
def run(s):
    op = s["op"]
    if own:
        from pretrained_rstr_b200.csrc import ops
        if op == "append":
            d, page, n = s["head_dim"], s["page"], s["tokens"]
            ops.kv_append_4bit(s["k_tiles"], s["v_tiles"], s["k"], s["v"], s["slots"], n, d, page, s["status"])
            ops.kv_read_4bit(s["k_back"], s["v_back"], s["k_tiles"], s["v_tiles"], s["slots"], n, d, page, s["status"])
            return [s["k_back"], s["v_back"]]
        if op == "attention":
            ops.attention_4bit(s["out"], s["q"], s["k_tiles"], s["v_tiles"], s["block_table"], s["positions"],
                               s["tile_req"], s["tile_row0"], s["tile_rows"], s["tile_most"], s["heads"],
                               s["head_dim"], s["page"], s["scale"], s["window"] or None, s["longest"], s["status"])
            return s["out"]
        if op == "tables":
            ops.step_tables(s["rows"], s["held"], s["brought"], s["tables"], s["page"], s["q_start"], s["kv_len"],
                            s["positions"], s["seq_of_token"], s["slots"], s["block_table"], s["status"],
                            free_pages=s["free_pages"], free_start=s["free_start"], free_next=s["free_next"])
            return _tables_out(s)
        ops.verify_drafts(s["tokens"], s["accepted"], s["logits"], s["row_start"], s["drafted"], s["uniforms"],
                          s["temperature"], s["status"], draft_probs=s["draft_probs"])
        return [s["tokens"], s["accepted"]]
    if op == "append":
        return _plain_append(s)
    if op == "attention":
        return _plain_attention(s)
    if op == "tables":
        return _plain_tables(s)
    return _plain_verify(s)
