"""The kernels of a paged cache held in 4 bits, of a step's tables and of drafted tokens, each against the plain
statement in 64 bits."""
import math

import pytest
import torch

import plain_cache4 as plain

pytestmark = pytest.mark.gpu
CUDA = "cuda"


def _ops():
    from pretrained_rstr_b200.csrc import ops
    return ops


def _status():
    return torch.zeros(4, dtype=torch.int32, device=CUDA)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=CUDA)


# ------------------------------------------------------------------------------ rows in and out
def _rows(g, n, heads, d, dtype, kind="normal"):
    x = torch.randn(n, heads, d, generator=g, dtype=torch.float64)
    x = x * torch.exp(torch.randn(heads, d, generator=g, dtype=torch.float64)) + torch.randn(heads, d, generator=g)
    if kind == "equal":
        x = x[..., :1].expand_as(x).clone()
    elif kind == "halves":
        # quotients on the very border of two codes: a step of 1, numbers at odd halves
        x = torch.randint(0, 31, (n, heads, d), generator=g).double() / 2 - 8
        x[..., 0::16], x[..., 1::16] = -8.0, 7.0
    elif kind == "wide":
        x = x * 2.0 ** torch.randint(-60, 60, (n, heads, d), generator=g).double()
    elif kind == "tiny":
        x = x * 2.0 ** -128
    return x.to(dtype)


@pytest.mark.parametrize("kind", ["normal", "equal", "halves", "wide", "tiny"])
@pytest.mark.parametrize("tokens,heads,d,page,dtype", [
    (1, 1, 16, 16, torch.bfloat16), (5, 3, 32, 48, torch.float32), (64, 12, 64, 64, torch.bfloat16),
    (37, 6, 80, 16, torch.bfloat16), (130, 9, 112, 128, torch.float32), (33, 8, 128, 64, torch.bfloat16),
    (70, 2, 48, 32, torch.float32)])
def test_rows_in_and_back(tokens, heads, d, page, dtype, kind):
    ops = _ops()
    g = torch.Generator().manual_seed(tokens * 1000 + d)
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    slots[tokens // 2:tokens // 2 + tokens // 7] = -1
    k, v = (_rows(g, tokens, heads, d, dtype, kind) for _ in range(2))
    fused = torch.cat([k.flatten(1), v.flatten(1), k.flatten(1)], 1).to(CUDA)
    tiles = [torch.randint(0, 256, (pages, heads, plain.tile_bytes(page, d)), generator=g, dtype=torch.uint8)
             for _ in range(2)]
    kt, vt = (t.to(CUDA) for t in tiles)
    status = _status()
    ops.kv_append_4bit(kt, vt, fused[:, :heads * d], fused[:, heads * d:2 * heads * d], slots.to(CUDA), tokens, d, page,
                       status)
    back = [torch.full((tokens, heads * d), 7.0, device=CUDA) for _ in range(2)]
    ops.kv_read_4bit(*back, kt, vt, slots.to(CUDA), tokens, d, page, status)
    assert status.tolist() == [0] * 4
    for x, before, after, got in ((k, tiles[0], kt, back[0]), (v, tiles[1], vt, back[1])):
        codes, step, middle = plain.quantize(x)
        want = plain.unpack(before, page, d)
        for t, slot in enumerate(slots.tolist()):
            if slot >= 0:
                want[0][slot // page, :, slot % page] = codes[t].to(torch.uint8)
                want[1][slot // page, :, slot % page] = step[t]
                want[2][slot // page, :, slot % page] = middle[t]
        have = plain.unpack(after.cpu(), page, d)
        assert torch.equal(have[0], want[0].to(torch.uint8))              # every other row as it was
        for i in (1, 2):
            assert torch.equal(torch.nan_to_num(have[i], 3.0), torch.nan_to_num(want[i], 3.0))
        a, b = plain.values(codes, step, middle)
        live = slots >= 0
        assert torch.equal(got.cpu()[live], (a + b).flatten(1)[live].float())
        assert bool((got.cpu()[~live] == 7.0).all())


def test_rows_at_odd_addresses_and_back_in_bfloat16():
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    x = _rows(g, 9, 2, 32, torch.bfloat16).flatten(1)
    wide = torch.zeros(9, 131, dtype=torch.bfloat16)
    wide[:, 1:65], wide[:, 66:130] = x, x
    wide = wide.to(CUDA)
    kt, vt = (torch.zeros(1, 2, plain.tile_bytes(16, 32), dtype=torch.uint8, device=CUDA) for _ in range(2))
    slots = _ints(list(range(9)))
    ops.kv_append_4bit(kt, vt, wide[:, 1:65], wide[:, 66:130], slots, 9, 32, 16, _status())
    back = torch.zeros(9, 131, dtype=torch.bfloat16, device=CUDA)
    ops.kv_read_4bit(back[:, 1:65], back[:, 66:130], kt, vt, slots, 9, 32, 16, _status())
    a, b = plain.values(*plain.quantize(x.view(9, 2, 32)))
    assert torch.equal(back.cpu()[:, 1:65], (a + b).flatten(1).to(torch.bfloat16))
    assert torch.equal(back.cpu()[:, 66:130], (a + b).flatten(1).to(torch.bfloat16))
    assert bool((back[:, [0, 65, 130]] == 0).all())


def test_rows_that_hold_no_number():
    """A group with an infinity or a NaN reads back as NaN, its neighbours as ever; the largest numbers are numbers."""
    ops = _ops()
    x = torch.linspace(-1, 1, 2 * 64).view(2, 64)
    x[0, 3], x[1, 40] = math.inf, math.nan
    big = torch.full((2, 64), 3.0e38)
    big[:, ::2] = -3.0e38
    kt, vt = (torch.zeros(1, 1, plain.tile_bytes(16, 64), dtype=torch.uint8, device=CUDA) for _ in range(2))
    slots = _ints([4, 9])
    ops.kv_append_4bit(kt, vt, x.to(CUDA), big.to(CUDA), slots, 2, 64, 16, _status())
    kb, vb = (torch.zeros(2, 64, device=CUDA) for _ in range(2))
    ops.kv_read_4bit(kb, vb, kt, vt, slots, 2, 64, 16, _status())
    assert torch.isnan(kb[0, :32]).all() and torch.isnan(kb[1, 32:]).all()
    assert torch.isfinite(kb[0, 32:]).all() and torch.isfinite(kb[1, :32]).all()
    assert torch.isfinite(vb).all()


def test_a_slot_outside_the_pool_is_reported():
    ops = _ops()
    kt, vt = (torch.zeros(2, 1, plain.tile_bytes(16, 32), dtype=torch.uint8, device=CUDA) for _ in range(2))
    x = torch.ones(2, 32, device=CUDA)
    status = _status()
    ops.kv_append_4bit(kt, vt, x, x, _ints([32, 5]), 2, 32, 16, status)
    assert status.tolist()[:3] == [3, 0, 32]
    assert int((kt != 0).sum()) > 0 and not kt[1].any()


# ------------------------------------------------------------------------------------ attention
def _cache(g, pool, kv, page, d):
    out = []
    for _ in range(2):
        x = torch.randn(pool, kv, page, d, generator=g) * torch.exp(0.5 * torch.randn(kv, 1, d, generator=g)) \
            + 0.5 * torch.randn(kv, 1, d, generator=g)
        out.append(plain.pack(*plain.quantize(x)))
    return out


def _garbage_behind(tiles, table, total, page, d):
    """What pages hold behind their request's last position, and free pages: all kinds of bits, NaN among them."""
    codes, step, middle = plain.unpack(tiles, page, d)
    used = set()
    for pages, n in zip(table, total):
        for i in range(-(-n // page)):
            used.add(pages[i])
            keep = min(page, n - i * page)
            codes[pages[i], :, keep:] = 15
            step[pages[i], :, keep:] = math.nan
            middle[pages[i], :, keep:] = math.inf
    for p in set(range(tiles.shape[0])) - used:
        step[p], middle[p] = math.nan, -math.inf
    return plain.pack(codes, step, middle)


CASES = [
    # lengths held, tokens brought, heads, kv heads, head size, page, window
    ([0], [1], 1, 1, 16, 16, None),
    ([0, 63, 64, 200], [1, 1, 1, 1], 4, 4, 64, 64, None),
    ([999], [1], 12, 12, 64, 64, None),
    ([15, 31, 100, 0, 7], [3, 5, 1, 2, 9], 4, 2, 64, 16, None),
    ([40, 0], [70, 133], 3, 3, 32, 48, None),
    ([130, 5], [1, 1], 32, 8, 128, 128, None),
    ([257], [5], 8, 1, 128, 64, None),
    ([90], [33], 6, 3, 80, 32, None),
    ([300, 10], [1, 1], 9, 9, 112, 16, None),
    ([77], [20], 10, 5, 96, 64, None),
    ([50], [3], 2, 2, 48, 48, None),
    ([500, 30], [1, 2], 4, 4, 64, 64, 1),
    ([500, 30], [40, 20], 4, 2, 64, 64, 37),
    ([5000], [1], 2, 1, 64, 64, None),
    ([3000], [2], 4, 1, 128, 16, 2500),
    ([10], [1], 40, 1, 64, 64, None),
    # portions of prompts that go to the tensor-memory kernel
    ([0], [33], 2, 2, 64, 64, None),
    ([130, 5, 0], [70, 200, 64], 4, 4, 64, 64, None),
    ([300, 64], [40, 64], 8, 2, 128, 64, None),
    ([1000], [128], 1, 1, 64, 128, None),
    ([700, 63], [65, 129], 2, 1, 128, 192, None),
    ([0], [50], 40, 1, 64, 64, None),
    ([11, 200], [40, 70], 4, 4, 16, 16, None),
    ([100], [60], 3, 3, 32, 48, None),
    ([33, 5], [50, 34], 2, 1, 48, 32, None),
    ([90], [64], 3, 3, 80, 16, None),
    ([150], [40], 4, 2, 96, 96, None),
    ([20], [129], 2, 2, 112, 48, None),
    # more heads to a key/value head than a tile has rows
    ([20], [2], 130, 1, 16, 16, None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("parts", [0, 1, 3, 8])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_against_64_bits(case, parts, dtype):
    ops = _ops()
    held, new, heads, kv, d, page, window = CASES[case]
    if parts in (1, 3) and case not in (1, 3, 5, 13, 17, 19, 24, 27):
        pytest.skip("one or two long cases are enough for a forced number of parts")
    g = torch.Generator().manual_seed(case)
    total = [a + n for a, n in zip(held, new)]
    count = sum(-(-t // page) for t in total)
    wide = max(-(-t // page) for t in total) + 1
    order = torch.randperm(count + 3, generator=g).tolist()
    table, at = [], 0
    for t in total:
        n = -(-t // page)
        table.append(order[at:at + n] + [-1] * (wide - n))
        at += n
    kt, vt = (_garbage_behind(x, table, total, page, d) for x in _cache(g, count + 3, kv, page, d))
    tokens = sum(new) + 2                                                 # (two rows belong to no tile)
    q = (1.3 * torch.randn(tokens, heads * d + 8, generator=g)).to(dtype)[:, :heads * d]
    positions = [a + i for a, n in zip(held, new) for i in range(n)] + [0, 0]
    requests = [b for b, n in enumerate(new) for _ in range(n)] + [-1, -1]
    scale = 1.0 / math.sqrt(d)
    ref, terms = plain.attention(q, kt, vt, table, positions, requests, heads, d, page, scale, window)
    most = max(1, 128 * kv // heads)
    tiles = plain.tiles_of(new, most)
    out = torch.full((tokens, heads * d), 5.0, dtype=dtype, device=CUDA)
    status = _status()
    qd = torch.zeros(tokens, heads * d + 8, dtype=dtype, device=CUDA)
    qd[:, :heads * d] = q.to(CUDA)
    args = (kt.to(CUDA), vt.to(CUDA), _ints(table), _ints(positions), *(_ints(list(x)) for x in zip(*tiles)),
            min(most, max(new)), heads, d, page, scale, window, max(total), status)
    ops.attention_4bit(out, qd[:, :heads * d], *args, parts=parts)
    assert status.tolist() == [0] * 4
    assert bool((out[-2:] == 5.0).all())                                  # rows of no tile
    err = (out.cpu().double() - ref)[:-2].abs()
    bound = plain.attention_bound(ref, terms, max(total), dtype)[:-2]
    worst = float((err / bound).max())
    assert worst <= 1.0, f"{worst:.2f} of the bound"
    again = torch.zeros_like(out)
    ops.attention_4bit(again, qd[:, :heads * d], *args, parts=parts)
    assert torch.equal(again[:-2], out[:-2])                              # the same bits every time


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,d,page,new", [(2, 2, 64, 64, 80), (4, 1, 128, 64, 30), (2, 1, 96, 32, 40), (1, 1, 64, 64, 3),
                                                  (2, 2, 80, 16, 40)])
@pytest.mark.parametrize("parts", [0, 1, 4])
def test_a_token_that_is_no_number_reaches_those_that_see_it(heads, kv, d, page, new, dtype, parts):
    """A NaN among a token's keys makes that token's and all later results NaN in the heads that share it; one among its
    values in the channels of its group; what comes before it in the same tile stays what it was."""
    ops = _ops()
    g = torch.Generator().manual_seed(new)
    held, bad_k, bad_v = 70, 70 + new - 2, 70 + new // 2
    total = held + new
    pages = -(-total // page)
    k, v = (torch.randn(pages * page, kv, d, generator=g) for _ in range(2))
    clean = [plain.pack(*plain.quantize(x.view(pages, page, kv, d).transpose(1, 2))) for x in (k, v)]
    k[bad_k, 0, 3], v[bad_v, kv - 1, d - 1] = math.nan, math.inf
    dirty = [plain.pack(*plain.quantize(x.view(pages, page, kv, d).transpose(1, 2))) for x in (k, v)]
    q = torch.randn(new, heads * d, generator=g).to(dtype).to(CUDA)
    tiles = plain.tiles_of([new], max(1, 128 * kv // heads))
    out = []
    for kt, vt in (clean, dirty):
        o, status = torch.zeros(new, heads * d, dtype=dtype, device=CUDA), _status()
        ops.attention_4bit(o, q, kt.to(CUDA), vt.to(CUDA), _ints([list(range(pages))]), _ints(list(range(held, total))),
                           *(_ints(list(x)) for x in zip(*tiles)), min(new, max(1, 128 * kv // heads)), heads, d, page, 0.3,
                           None, total, status, parts=parts)
        assert status.tolist() == [0] * 4
        out.append(o.float().cpu().view(new, heads, d))
    nan = torch.zeros(new, heads, d, dtype=torch.bool)
    group = heads // kv
    nan[bad_k - held:, :group] = True
    nan[bad_v - held:, heads - group:, (d - 1) // 32 * 32:] = True
    assert torch.equal(torch.isnan(out[1]), nan)
    assert torch.equal(out[0][~nan], out[1][~nan])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 40])
def test_what_a_tile_may_not_name_is_reported(new, dtype):
    """A page that is none, a request, a row, a position or a tile that does not fit: recorded, and the other request's
    results are what they are without it.  ``tile_count`` leaves the tiles behind it alone."""
    ops = _ops()
    g = torch.Generator().manual_seed(new)
    kt, vt = (plain.pack(*plain.quantize(torch.randn(6, 2, 64, 64, generator=g))).to(CUDA) for _ in range(2))
    q = torch.randn(2 * new, 128, generator=g).to(dtype).to(CUDA)

    def go(table=((0, 1, -1), (2, 3, -1)), positions=None, req=(0, 1), row0=(0, new), n=(new, new), most=new, count=None):
        out, status = torch.zeros(2 * new, 128, dtype=dtype, device=CUDA), _status()
        at = list(range(85, 85 + new)) + list(range(80, 80 + new)) if positions is None else positions
        ops.attention_4bit(out, q, kt, vt, _ints([list(r) for r in table]), _ints(at), _ints(list(req)), _ints(list(row0)),
                           _ints(list(n)), most, 2, 64, 64, 0.1, None, 192, status,
                           tile_count=None if count is None else _ints([count]))
        return out, status.tolist()
    want, status = go()
    assert status == [0] * 4
    for kw, code in ((dict(table=((0, -1, -1), (2, 3, -1))), 4), (dict(table=((0, 6, -1), (2, 3, -1))), 4),
                     (dict(req=(2, 1)), 2), (dict(req=(-1, 1)), 2), (dict(row0=(-1, new)), 2), (dict(row0=(new + 1, new)), 2),
                     (dict(positions=[200] * new + list(range(80, 80 + new))), 2)):
        out, status = go(**kw)
        assert status[0] == code, (kw, status)
        assert torch.equal(out[new:], want[new:]), kw
    out, status = go(count=1)
    assert status == [0] * 4 and torch.equal(out[:new], want[:new]) and not out[new:].any()
    out, status = go(count=0)
    assert status == [0] * 4 and not out.any()
    out, status = go(n=(0, new))
    assert status == [0] * 4 and not out[:new].any() and torch.equal(out[new:], want[new:])


def _call(seed, page_offset=0, pool=None, dtype=torch.bfloat16, new=1):
    """Append, read back, attend for two requests; all inputs from ``seed``.  Pages ``page_offset`` ... of ``pool``."""
    ops = _ops()
    g = torch.Generator().manual_seed(seed)
    kv, d, page, total = 8, 128, 64, [130, 70]
    pages = [[page_offset + 3, page_offset, page_offset + 4], [page_offset + 1, page_offset + 2, -1]]
    tile = plain.tile_bytes(page, d)
    kt, vt = pool or [torch.zeros(6, kv, tile, dtype=torch.uint8, device=CUDA) for _ in range(2)]
    n = sum(total)
    x = torch.randn(n, 3 * kv * d, generator=g).to(dtype).to(CUDA)
    q, k, v = x[:, :kv * d], x[:, kv * d:2 * kv * d], x[:, 2 * kv * d:]
    slots = _ints([pages[b][i // page] * page + i % page for b, t in enumerate(total) for i in range(t)])
    status = _status()
    ops.kv_append_4bit(kt, vt, k, v, slots, n, d, page, status)
    back = [torch.zeros(n, kv * d, device=CUDA) for _ in range(2)]
    ops.kv_read_4bit(*back, kt, vt, slots, n, d, page, status)
    positions = _ints([i for t in total for i in range(t)])
    at = [129, 199] if new == 1 else [130 - new, 200 - new]
    out = torch.zeros(n, kv * d, dtype=dtype, device=CUDA)
    ops.attention_4bit(out, q, kt, vt, _ints(pages), positions, _ints([0, 1]), _ints(at), _ints([new, new]), new, kv, d, page,
                       0.1, None, 130, status)
    return back + [out, status]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 40])
def test_results_beside_the_queries_in_one_tensor(new, dtype):
    """q and out as neighbouring columns of one tensor give the bits that tensors of their own give; q stays as it was."""
    ops = _ops()
    kv, d, page = 4, 64, 64
    g = torch.Generator().manual_seed(3)
    kt, vt = [torch.zeros(2, kv, plain.tile_bytes(page, d), dtype=torch.uint8, device=CUDA) for _ in range(2)]
    k, v, q = [torch.randn(100, kv * d, generator=g).to(dtype).to(CUDA) for _ in range(3)]
    status = _status()
    ops.kv_append_4bit(kt, vt, k, v, _ints(list(range(100))), 100, d, page, status)
    both = torch.zeros(100, 2 * kv * d, dtype=dtype, device=CUDA)
    for at in (0, kv * d):
        other = kv * d - at
        both[:, at:at + kv * d] = q
        both[:, other:other + kv * d] = 0
        alone = torch.zeros(100, kv * d, dtype=dtype, device=CUDA)
        for q_in, out in ((q, alone), (both[:, at:at + kv * d], both[:, other:other + kv * d])):
            ops.attention_4bit(out, q_in, kt, vt, _ints([[0, 1]]), _ints(list(range(100))), _ints([0]), _ints([100 - new]),
                               _ints([new]), new, kv, d, page, 0.125, None, 100, status)
        assert alone[100 - new:].abs().sum() > 0 and status.tolist() == [0] * 4
        assert torch.equal(both[:, other:other + kv * d], alone) and torch.equal(both[:, at:at + kv * d], q)


@pytest.mark.parametrize("new", [1, 40])
def test_pages_beyond_four_gigabytes(new):
    """The last pages of a pool of 4.7 GB of keys (and of values) give the bits that the first ones of a small pool give."""
    tile, last = plain.tile_bytes(64, 128), 115000
    pool = [torch.empty(last + 6, 8, tile, dtype=torch.uint8, device=CUDA) for _ in range(2)]
    for a, b in zip(_call(1, new=new), _call(1, last, pool, new=new)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 40])
def test_calls_on_two_streams_at_once(dtype, new):
    """No call shares memory with another: two streams' calls give what they give alone."""
    alone = [_call(seed, dtype=dtype, new=new) for seed in (1, 2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_call(i + 1, dtype=dtype, new=new))
    torch.cuda.synchronize()
    for want, runs in zip(alone, got):
        for run in runs:
            for a, b in zip(want, run):
                assert torch.equal(a, b)


# --------------------------------------------------------------------------------------- tables
def _run_tables(rows, held, brought, table, page, cap, free=None, start=0):
    ops = _ops()
    n, wide = len(rows), len(table[0])
    t = _ints(table)
    out = dict(q_start=_ints([9] * (n + 1)), kv_len=_ints([9] * n), positions=_ints([9] * cap), seq=_ints([9] * cap),
               slots=_ints([9] * cap), block=_ints([[9] * wide] * n))
    nxt, status = _ints([-5]), _status()
    kw = {} if free is None else dict(free_pages=_ints(free), free_start=_ints([start]), free_next=nxt)
    ops.step_tables(_ints(rows), _ints(held), _ints(brought), t, page, out["q_start"], out["kv_len"], out["positions"],
                    out["seq"], out["slots"], out["block"], status, **kw)
    return [out[k].tolist() for k in ("q_start", "kv_len", "positions", "seq", "slots", "block")] + \
        [t.tolist(), nxt.tolist()[0]], status.tolist()


@pytest.mark.parametrize("n,page,wide,most,spare", [(1, 16, 4, 20, 0), (3, 64, 3, 100, 5), (64, 64, 16, 1, 3),
                                                    (257, 16, 40, 90, 1), (1000, 7, 9, 30, 0), (4096, 16, 5, 3, 2)])
def test_step_tables(n, page, wide, most, spare):
    g = torch.Generator().manual_seed(n)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    held = [r(0, wide * page - most) if wide * page > most else 0 for _ in range(n)]
    brought = [r(0, min(most, wide * page - h)) for h in held]
    if sum(brought) == 0:
        brought[0] = 1
    lanes = n + 2
    rows = torch.randperm(lanes, generator=g)[:n].tolist()
    pages = torch.randperm(n * wide + 50, generator=g).tolist()
    table = [[-1] * wide for _ in range(lanes)]
    at = 0
    for row, h in zip(rows, held):
        for i in range(-(-h // page)):
            table[row][i] = pages[at]
            at += 1
    free = pages[at:]
    want = plain.tables(rows, held, brought, table, page, sum(brought) + spare, free, 3)
    got, status = _run_tables(rows, held, brought, table, page, sum(brought) + spare, free, 3)
    assert status == [0] * 4
    for a, b in zip(got, want):
        assert a == b


def test_step_tables_report_what_does_not_fit():
    table = [[4, -1], [6, 7]]
    # request 1 names no row, request 2 holds more than a row of the table
    got, status = _run_tables([0, 5, 1], [10, 0, 33], [2, 1, 1], table, 16, 8)
    assert status[0] in (2, 6) and got[0] == [0, 2, 2, 2] and got[1] == [12, 0, 0]
    assert got[4] == [74, 75] + [-1] * 6 and got[5] == [[4, -1], [-1, -1], [-1, -1]]
    # a page that is missing, and none to take
    got, status = _run_tables([0, 1], [16, 31], [1, 1], table, 16, 3)
    assert status[0] == 4 and got[4] == [-1, 7 * 16 + 15, -1] and got[7] == -5
    got, status = _run_tables([0], [15], [18], table, 16, 30, free=[9], start=0)
    assert status[0] in (2, 4)
    got, status = _run_tables([0], [15], [3], table, 16, 30, free=[9], start=1)
    assert status[0] == 4 and got[4][:3] == [4 * 16 + 15, -1, -1] and got[5] == [[4, -1]]
    # an empty list is a list: what a request grows into is missing
    got, status = _run_tables([0], [15], [3], [[4, 9], [6, 7]], 16, 30, free=[], start=0)
    assert status[0] == 4 and got[4][:3] == [4 * 16 + 15, -1, -1] and got[7] == 1
    # more tokens than rows: those behind are left out
    got, status = _run_tables([1, 0], [0, 0], [20, 3], table, 16, 21)
    assert status[0] == 6 and got[0] == [0, 20, 21] and got[4][20] == 64


# ------------------------------------------------------------------------------------ drafted tokens
@pytest.mark.parametrize("draft", ["probabilities", "tokens"])
@pytest.mark.parametrize("requests,drafts,vocab,temperature", [
    (1, 0, 7, 1.0), (1, 3, 1, 0.7), (3, 4, 50257, 0.8), (5, 2, 501, 1.3), (2, 31, 999, 1.0), (9, 3, 50257, 0.0),
    (40, 5, 130, 0.5), (2, 2, 70001, 1.0), (3, 1, 131072, 0.9),
    (38, 2, 60001, 0.9), (75, 4, 5003, 0.0)])
def test_verify_drafts(requests, drafts, vocab, temperature, draft):
    ops = _ops()
    g = torch.Generator().manual_seed(requests * 100 + drafts)
    counts = [drafts if i % 3 == 0 else max(0, drafts - i % 4) for i in range(requests)]
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c + 1)
    rows = starts[-1]
    logits = 2.0 * torch.randn(rows, vocab, generator=g)
    if temperature == 0.0:
        logits = torch.round(logits)                                      # equals: the lowest index wins
    if vocab > 5:
        logits[:, 2] = -math.inf
    near = logits + 0.7 * torch.randn(rows, vocab, generator=g)
    probs = torch.softmax(near / (temperature or 1.0), -1)
    drafted = torch.where(torch.rand(rows, generator=g) < 0.5, near.argmax(-1), torch.multinomial(probs, 1, generator=g)[:, 0])
    temps = [temperature if i % 5 != 4 else 0.0 for i in range(requests)]
    uniforms = torch.rand(rows, 2, generator=g)
    uniforms[0] = 0.0
    q = probs if draft == "probabilities" else None
    want = plain.verify(logits, starts, drafted.tolist(), uniforms.tolist(), temps, q)
    wide = torch.zeros(rows, vocab + 3, device=CUDA)
    wide[:, 1:vocab + 1] = logits.to(CUDA)
    tokens, accepted, status = _ints([9] * rows), _ints([9] * requests), _status()
    ops.verify_drafts(tokens, accepted, wide[:, 1:vocab + 1], _ints(starts), drafted.to(torch.int32).to(CUDA),
                      uniforms.to(CUDA), torch.tensor(temps, device=CUDA), status,
                      draft_probs=None if q is None else q.to(CUDA))
    assert status.tolist() == [0] * 4
    assert accepted.tolist() == want[1]
    assert tokens.tolist() == want[0]


def test_a_draft_that_covers_the_target_draws_from_the_target():
    """Nothing left of p - q (the draft says more than the target everywhere): the token comes from p."""
    ops = _ops()
    logits = torch.zeros(2, 4, device=CUDA)
    tokens, accepted, status = _ints([9, 9]), _ints([9]), _status()
    ops.verify_drafts(tokens, accepted, logits, _ints([0, 2]), _ints([1, 0]),
                      torch.tensor([[0.9, 0.6], [0.0, 0.0]], device=CUDA), torch.ones(1, device=CUDA), status,
                      draft_probs=torch.full((2, 4), 0.5, device=CUDA))
    assert tokens.tolist() == [2, -1] and accepted.tolist() == [0] and status.tolist() == [0] * 4


def test_rows_without_a_largest_logit_and_bad_tokens_are_reported():
    ops = _ops()

    def go(logits, drafted, t=1.0, starts=(0, 2)):
        tokens, accepted, status = _ints([9, 9]), _ints([9]), _status()
        ops.verify_drafts(tokens, accepted, logits.to(CUDA), _ints(list(starts)), _ints(drafted),
                          torch.zeros(2, 2, device=CUDA), torch.full((1,), t, device=CUDA), status)
        return tokens.tolist(), accepted.tolist(), status.tolist()
    for value in (-math.inf, math.nan, math.inf):
        rows = torch.zeros(2, 40)
        rows[0] = value
        tokens, accepted, status = go(rows, [3, 0])
        assert status[0] == 7 and status[1] == 0 and accepted == [0] and 0 <= tokens[0] < 40 and tokens[1] == -1
    for bad in (-1, 40):
        tokens, accepted, status = go(torch.zeros(2, 40), [bad, 0])
        assert status[:3] == [1, 0, bad] and accepted == [0] and 0 <= tokens[0] < 40
    tokens, accepted, status = go(torch.zeros(2, 40), [0, 0], starts=(0, 3))
    assert status[0] == 6 and accepted == [0] and tokens == [9, 9]
