"""Calls of the 4-bit cache, step tables and verification at the edges of what they take, against the plain statement in
64 bits."""
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


def _verify(logits, starts, drafted, uniforms, temps, probs=None):
    ops = _ops()
    rows = logits.shape[0]
    tokens, accepted, status = _ints([9] * rows), _ints([9] * len(temps)), _status()
    ops.verify_drafts(tokens, accepted, logits.to(CUDA), _ints(starts), _ints(drafted), uniforms.to(CUDA),
                      torch.tensor(temps, dtype=torch.float32, device=CUDA), status,
                      draft_probs=None if probs is None else probs.to(CUDA))
    return (tokens.tolist(), accepted.tolist()), status.tolist()


# ------------------------------------------------------------------------------------ verification
@pytest.mark.parametrize("requests", [1, 40])
@pytest.mark.parametrize("vocab,places", [(40, [7]), (700, [699, 0]), (50257, [50000, 33001]), (50257, [6284])])
@pytest.mark.parametrize("follows", [False, True])
def test_a_nan_wins_a_greedy_row_and_is_reported(requests, vocab, places, follows):
    """As in the framework's greedy sampler: a NaN among a row's logits wins over every number, the lowest one over other
    NaN, and the row is reported, whether the draft had that token or the largest number's."""
    g = torch.Generator().manual_seed(vocab + len(places))
    logits = torch.randn(3 * requests, vocab, generator=g)
    starts = list(range(0, 3 * requests + 1, 3))
    drafted = logits.argmax(-1).tolist()
    bad = 3 * (requests - 1) + 1
    logits[bad, places] = math.nan
    if follows:
        drafted[bad] = min(places)
    want = plain.verify(logits, starts, drafted, torch.zeros(3 * requests, 2).tolist(), [0.0] * requests)
    got, status = _verify(logits, starts, drafted, torch.zeros(3 * requests, 2), [0.0] * requests)
    assert got == want and got[0][bad] == min(places)
    assert status[:3] == [7, bad, requests - 1]


@pytest.mark.parametrize("certain", [True, False])
@pytest.mark.parametrize("requests,vocab,t", [(30, 50257, 1.1), (64, 50257, 0.8), (30, 50257, 0.3), (64, 5003, 1.3), (20, 131072, 1.0)])
def test_numbers_next_to_the_border_decide_by_it(requests, vocab, t, certain):
    """u * q < p for the float32 numbers u right below and right above p / q: the border itself in 64 bits."""
    g = torch.Generator().manual_seed(vocab)
    logits = 2.5 * torch.randn(2 * requests, vocab, generator=g)
    t = float(torch.tensor(t))
    p = torch.softmax(logits.double() / t, -1)
    drafted = torch.multinomial(p, 1, generator=g)[:, 0]
    rows = torch.arange(2 * requests)
    mine = p[rows, drafted]
    q = torch.zeros(2 * requests, vocab)
    q[rows, drafted] = 1.0 if certain else (mine.float() * (1.0 + torch.rand(2 * requests, generator=g)))
    border = mine / q[rows, drafted].double()
    below = border.float()
    below = torch.where(below.double() >= border, torch.nextafter(below, torch.zeros(1)), below)
    above = torch.nextafter(below, torch.ones(1))
    starts = list(range(0, 2 * requests + 1, 2))
    for u, stays in ((below, 1), (above, 0)):
        assert bool(((u.double() * q[rows, drafted].double() < mine) == bool(stays)).all())
        uniforms = torch.stack([u, torch.full_like(u, 0.5)], 1)
        (tokens, accepted), status = _verify(logits, starts, drafted.tolist(), uniforms, [t] * requests, None if certain else q)
        assert status == [0] * 4
        assert accepted == [stays] * requests


@pytest.mark.parametrize("t", [math.inf, 1e38, 1e-42, 1e-38])
@pytest.mark.parametrize("requests", [3, 40])
def test_the_largest_and_the_smallest_temperatures(requests, t):
    """At an endless temperature all tokens are as likely, at one next to 0 only the largest logits are."""
    g = torch.Generator().manual_seed(5)
    logits = torch.round(2 * torch.randn(3 * requests, 501, generator=g))
    starts = list(range(0, 3 * requests + 1, 3))
    drafted = logits.argmax(-1)
    drafted[::2] = torch.randint(501, drafted[::2].shape, generator=g)
    uniforms = torch.rand(3 * requests, 2, generator=g)
    uniforms[::4, 0] *= 0.003
    t = float(torch.tensor(t, dtype=torch.float32))
    want = plain.verify(logits, starts, drafted.tolist(), uniforms.tolist(), [t] * requests)
    got, status = _verify(logits, starts, drafted.tolist(), uniforms, [t] * requests)
    assert status == [0] * 4 and got == want


@pytest.mark.parametrize("rows", [33, 40, 200])
def test_a_request_of_too_many_rows_has_no_tokens(rows):
    """Refused and recorded; its rows say so (-1) instead of what an earlier step left there, its neighbours are as ever."""
    g = torch.Generator().manual_seed(rows)
    logits = torch.randn(rows + 4, 50, generator=g)
    drafted = logits.argmax(-1).tolist()
    (tokens, accepted), status = _verify(logits, [0, 2, 2 + rows, rows + 4], drafted, torch.zeros(rows + 4, 2), [0.0] * 3)
    assert status[0] == 6 and accepted == [1, 0, 1]
    assert tokens == drafted[:2] + [-1] * rows + drafted[-2:]


def test_requests_of_no_rows_accept_nothing():
    """Recorded, with the others as they are; without any row at all too."""
    logits = torch.randn(3, 50, generator=torch.Generator().manual_seed(0))
    best = logits.argmax(-1).tolist()
    (tokens, accepted), status = _verify(logits, [0, 0, 3, 3], best, torch.zeros(3, 2), [0.0] * 3)
    assert status[0] == 6 and (tokens, accepted) == (best, [0, 2, 0])
    (tokens, accepted), status = _verify(logits[:0], [0, 0, 0], [], torch.zeros(0, 2), [0.0, 1.0])
    assert status[0] == 6 and (tokens, accepted) == ([], [0, 0])


# ------------------------------------------------------------------------------------ attention
def _cached(k, v, page):
    n, kv, d = k.shape
    pages = -(-n // page)

    def one(x):
        full = torch.zeros(pages * page, kv, d)
        full[:n] = x
        return plain.pack(*plain.quantize(full.view(pages, page, kv, d).transpose(1, 2))).to(CUDA)
    return one(k), one(v), _ints([list(range(pages))])


def _attend(k, v, q, held, page, scale, parts=0, window=None, status_word=0):
    """The tokens behind ``held`` positions of one request, in tiles of up to 128 rows."""
    ops = _ops()
    total, kv, d = k.shape
    new, heads = total - held, q.shape[1] // d
    kt, vt, table = _cached(k, v, page)
    most = max(1, 128 * kv // heads)
    tiles = plain.tiles_of([new], most)
    out, status = torch.full((new, heads * d), 3.0, dtype=q.dtype, device=CUDA), _status()
    ops.attention_4bit(out, q.to(CUDA), kt, vt, table, _ints(list(range(held, total))), *(_ints(list(x)) for x in zip(*tiles)),
                       min(new, most), heads, d, page, scale, window, total, status, parts=parts)
    assert status.tolist()[0] == status_word
    return out.float().cpu().view(new, heads, d)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,d,page", [(2, 2, 64, 64), (4, 1, 128, 64), (2, 1, 96, 32), (3, 3, 16, 16)])
@pytest.mark.parametrize("held,new,parts", [(64, 1, 0), (256, 1, 4), (186, 70, 0), (186, 70, 4), (250, 40, 2), (316, 6, 8)])
def test_a_key_that_is_no_number_alone_in_its_part(held, new, parts, heads, kv, d, page, dtype):
    """The first token that opens a block of 64 has keys that are no numbers: the part of the keys that holds nothing else
    for it still makes its result NaN."""
    g = torch.Generator().manual_seed(held)
    total = held + new
    bad = -(-held // 64) * 64
    k, v, q = torch.randn(total, kv, d, generator=g), torch.randn(total, kv, d, generator=g), torch.randn(new, heads * d, generator=g)
    want = _attend(k, v, q.to(dtype), held, page, 0.2, parts)
    k[bad, 0, 3] = math.nan
    got = _attend(k, v, q.to(dtype), held, page, 0.2, parts)
    nan = torch.zeros(new, heads, d, dtype=torch.bool)
    nan[bad - held:, :heads // kv] = True
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,d,page", [(2, 2, 64, 64), (4, 1, 128, 64), (2, 1, 96, 32), (3, 3, 16, 16)])
@pytest.mark.parametrize("held,new,parts", [(99, 1, 1), (99, 1, 0), (299, 1, 4), (200, 40, 1), (200, 40, 4), (200, 5, 2), (200, 12, 1)])
@pytest.mark.parametrize("bad", [3, 98])
def test_a_value_that_is_no_number_under_a_weight_of_nearly_nothing(bad, held, new, parts, heads, kv, d, page, dtype):
    """Nearly nothing times NaN is NaN, in whichever stage or part of the keys the value lies."""
    g = torch.Generator().manual_seed(new)
    total = held + new
    k, v = 0.1 * torch.randn(total, kv, d, generator=g), torch.randn(total, kv, d, generator=g)
    q = 4.0 + 0.1 * torch.randn(new, heads * d, generator=g)
    k[held - 5 if held > 104 else 90] = 6.0                               # e^-300 and less for all the others
    want = _attend(k, v, q.to(dtype), held, page, 1.0, parts)
    v[bad, kv - 1, d - 1] = math.nan
    got = _attend(k, v, q.to(dtype), held, page, 1.0, parts)
    nan = torch.zeros(new, heads, d, dtype=torch.bool)
    nan[:, heads - heads // kv:, (d - 1) // 32 * 32:] = True
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("heads,kv,d,page", [(2, 2, 64, 64), (12, 12, 64, 64), (4, 1, 128, 64), (2, 1, 96, 32), (3, 3, 16, 16)])
@pytest.mark.parametrize("held,new", [(99, 1), (1000, 1), (300, 5), (500, 12), (63, 32)])
def test_equal_values_come_back_as_they_are(held, new, heads, kv, d, page):
    """Values that are all one number: whatever the weights are, they add up to one, so the result is that number.  A weight
    rounded to bfloat16 (2^-8 of itself) would show; in 32 bits what is lost is far below half a step of the result.
    (Where the number's step is 0 there is nothing that p * step rounds.)"""
    if new * heads > 32 * kv:
        pytest.skip("a portion of a prompt: its kernel rounds weights to bfloat16")
    g = torch.Generator().manual_seed(held + new)
    total = held + new
    # scores of 0 and of ln(0.50195...): weights 1 and 0.5 + 2^-9, which lies half way between two bfloat16 numbers
    k = torch.zeros(total, kv, d)
    k[torch.rand(total, generator=g) < 0.9] = -1.0
    q = torch.full((new, heads * d), 0.5)
    scale = -math.log(0.5 + 2.0 ** -9 * 1.02) / (0.5 * d)
    for number in (8.0, -0.0078125, 1.5):
        out = _attend(k, torch.full((total, kv, d), number), q.to(torch.bfloat16), held, page, scale)
        assert bool((out == number).all()), float((out - number).abs().max() / abs(number))


@pytest.mark.parametrize("heads,kv,d,page,held,new,window", [
    (12, 12, 64, 64, 999, 1, None), (2, 2, 64, 64, 300, 5, None), (4, 1, 128, 64, 700, 6, None), (2, 1, 96, 32, 90, 12, None),
    (3, 3, 16, 16, 200, 30, None), (4, 4, 64, 64, 800, 1, 500), (1, 1, 64, 64, 3000, 8, 2000)])
def test_weights_meet_middles_unrounded(heads, kv, d, page, held, new, window):
    """Channels with an offset, as keys and values of real models have: a result is off by half a step of its own (2^-8), of
    every weight times its step (2^-8), and by what sums in 32 bits lose: no weight is rounded before it meets an offset."""
    g = torch.Generator().manual_seed(held)
    total = held + new
    k = torch.randn(total, kv, d, generator=g)
    v = 0.3 * torch.randn(total, kv, d, generator=g) + 5.0 * torch.randn(kv, d, generator=g).sign()
    q = torch.randn(new, heads * d, generator=g).to(torch.bfloat16)
    scale = 1.0 / math.sqrt(d)
    got = _attend(k, v, q, held, page, scale, window=window).flatten(1)
    kt, vt, table = _cached(k, v, page)
    ref, (a, b, e) = plain.attention(q, kt.cpu(), vt.cpu(), table.tolist(), list(range(held, total)), [0] * new, heads, d, page,
                                     scale, window)
    wide = 2 * (1.01 * e + 2.0 ** -21 + 2.0 ** -17) + (total + 16) * 2.0 ** -23
    worst = float(((got.double() - ref).abs() / (1.01 * 2.0 ** -8 * (ref.abs() + a) + wide * b)).max())
    assert worst <= 1.0, f"{worst:.2f} of the bound"


@pytest.mark.parametrize("d,page,parts", [(64, 64, 1), (64, 64, 4), (128, 64, 1), (48, 32, 1)])
def test_values_next_to_the_largest_number(d, page, parts):
    """A float32 number beyond bfloat16's largest one, whose code stands for more than that: a portion of a prompt has no number
    for it where it is seen, and what it was where it is not."""
    g = torch.Generator().manual_seed(d)
    held, new, kv = 150, 60, 2
    k, v = (torch.randn(held + new, kv, d, generator=g) for _ in range(2))
    q = torch.zeros(new, kv * d, dtype=torch.bfloat16)                    # (weights of one before they are divided by their sum)
    want = _attend(k, v, q, held, page, 0.2, parts)
    at = held + new // 2
    v[at, 0, :32] = torch.tensor([3.4028e38, 1e38] * 16)
    got = _attend(k, v, q, held, page, 0.2, parts)
    seen = torch.zeros(new, kv, d, dtype=torch.bool)
    seen[at - held:, 0, :32] = True
    assert torch.equal(got[~seen], want[~seen])
    assert not bool(torch.isfinite(got[seen]).any())


# ------------------------------------------------------------------------------------ tables
@pytest.mark.parametrize("captured", [False, True])
def test_pages_taken_for_refused_tokens_are_used_by_the_next_step(captured):
    """Steps that bring drafted tokens and keep some, with pages from a list: a page a request took stays its own, the list
    gives no more than the requests ever held, no page is given twice, and nothing comes to the host."""
    ops = _ops()
    g = torch.Generator().manual_seed(1)
    n, page, wide, lanes, rounds, drafts = 70, 16, 12, 75, 40, 7
    lane = torch.randperm(lanes, generator=g)[:n].tolist()
    free = torch.randperm(n * wide + 9, generator=g).tolist()
    kept = torch.randint(0, drafts + 2, (rounds, n), generator=g)          # of the drafted tokens and the one before them
    kept[:, 0] = 0                                                        # (a request that refuses everything)
    cap = n * (drafts + 1)
    tables, held, brought = _ints([[-1] * wide] * lanes), _ints([0] * n), _ints([drafts + 1] * n)
    have, have_next, start, nxt = _ints([0] * n), _ints([-1] * n), _ints([4]), _ints([-1])
    out = dict(q_start=_ints([0] * (n + 1)), kv_len=_ints([0] * n), positions=_ints([0] * cap), seq_of_token=_ints([0] * cap),
               slots=_ints([0] * cap), block_table=_ints([[0] * wide] * n))
    status, step_kept, lane_d, free_d = _status(), _ints([0] * n), _ints(lane), _ints(free)

    def one_round():
        ops.step_tables(lane_d, held, brought, tables, page, *out.values(), status, free_pages=free_d, free_start=start,
                        free_next=nxt, have_pages=have, have_next=have_next)
        start.copy_(nxt)
        have.copy_(have_next)
        held.add_(step_kept)
    go = one_round
    if captured:
        first = [t.clone() for t in (tables, held, have, start)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one_round()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one_round()
        for t, was in zip((tables, held, have, start), first):
            t.copy_(was)
        go = graph.replay
    length, pages, at = [0] * n, [[] for _ in range(n)], 4
    for r in range(rounds):
        fits = [min(drafts + 1, wide * page - x) for x in length]
        brought.copy_(torch.tensor(fits, dtype=torch.int32))
        step_kept.copy_(torch.minimum(kept[r].to(torch.int32), torch.tensor(fits, dtype=torch.int32)))
        go()
        want_slots = []
        for b in range(n):
            need = -(-(length[b] + fits[b]) // page)
            while len(pages[b]) < need:
                pages[b].append(free[at])
                at += 1
            want_slots += [pages[b][x // page] * page + x % page for x in range(length[b], length[b] + fits[b])]
        assert status.tolist() == [0] * 4
        assert out["slots"].tolist() == want_slots + [-1] * (cap - len(want_slots))
        needs = [-(-(x + f) // page) for x, f in zip(length, fits)]
        assert out["block_table"].tolist() == [(p[:m] + [-1] * wide)[:wide] for p, m in zip(pages, needs)]
        assert have.tolist() == [len(p) for p in pages] and start.tolist() == [at]
        length = [x + min(int(k), f) for x, k, f in zip(length, kept[r], fits)]
        assert held.tolist() == length
    flat = [p for own in pages for p in own]
    assert len(flat) == len(set(flat)) == at - 4
    table = tables.tolist()
    assert all(table[row][:len(p)] == p for row, p in zip(lane, pages))


def test_pages_a_row_cannot_hold_are_reported():
    ops = _ops()

    def go(held, have, start=0):
        n = len(held)
        table, status, nxt, have_next = _ints([[5, 6, -1]] * n), _status(), _ints([-1]), _ints([-9] * n)
        o = [_ints([9] * k) for k in (n + 1, n, 8, 8, 8)]
        ops.step_tables(_ints(list(range(n))), _ints(held), _ints([2] * n), table, 16, *o, _ints([[9] * 3] * n), status,
                        free_pages=_ints([20, 21, 22]), free_start=_ints([start]), free_next=nxt, have_pages=_ints(have),
                        have_next=have_next)
        return [x.tolist() for x in o], table.tolist(), nxt.tolist(), have_next.tolist(), status.tolist()
    o, table, nxt, have_next, status = go([30, 3], [4, 1])                # more pages than a row has places
    assert status[:3] == [2, 0, 30] and o[0] == [0, 0, 2] and o[1] == [0, 5] and have_next == [4, 1] and nxt == [0]
    o, table, nxt, have_next, status = go([30, 3], [-1, 1])
    assert status[0] == 2 and o[1] == [0, 5] and have_next == [-1, 1]
    # fewer than its tokens lie in: those it has are looked up as without the count
    o, table, nxt, have_next, status = go([31, 3], [0, 1])
    assert status == [0] * 4 and table == [[5, 6, 20], [5, 6, -1]] and have_next == [3, 1] and nxt == [1]
    assert o[4][:2] == [6 * 16 + 15, 20 * 16]
    # a list that has run out: what is missing is not counted
    o, table, nxt, have_next, status = go([31, 3], [2, 1], start=3)
    assert status[0] == 4 and have_next == [2, 1] and o[4][:2] == [6 * 16 + 15, -1]
