"""The engine with its cache held in 4 bits, against the plain implementation whose keys and values go through 4 bits, and
the operators of a step with drafted tokens run together."""
import math

import pytest
import torch

import plain_cache4 as plain
import plain_gpt2
from helpers import ATOL, TINY, Replayer, make_folder, oracle_logits, random_tokens

pytestmark = pytest.mark.gpu
CUDA = "cuda"


def _oracle4(folder, prompts, monkeypatch):
    """The plain implementation with every key and value as a 4-bit cache gives it back."""
    def attention(x_ln, c_attn_w, c_attn_b, c_proj_w, c_proj_b, n_head, scale, window=None):
        t, d = x_ln.shape
        qkv = plain_gpt2.linear_conv1d(x_ln, c_attn_w, c_attn_b)
        q = qkv[:, :d].view(t, n_head, -1)
        k, v = (sum(plain.values(*plain.quantize(x.reshape(t, n_head, -1)))).float()
                for x in (qkv[:, d:2 * d], qkv[:, 2 * d:]))
        s = torch.einsum("ihd,jhd->hij", q, k) * scale
        s = s.masked_fill(torch.ones(t, t).triu(1).bool(), -math.inf)
        out = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(t, d)
        return plain_gpt2.linear_conv1d(out, c_proj_w, c_proj_b)
    with monkeypatch.context() as m:
        m.setattr(plain_gpt2, "causal_attention", attention)
        return oracle_logits(folder, prompts)


def _tolerance(rounded, exact):
    """A 32-bit product that is off by 1e-7 of itself may take a number next to the border of two codes to the other one:
    one code of some tens of thousands, worth one step.  What rounding ALL keys and values by up to half a step does to the
    logits is known (the two plain runs); one that is a whole step off is worth far less than a quarter of it."""
    moved = max(float((rounded[r] - exact[r]).abs().max()) for r in exact)
    assert moved > 20 * ATOL["float32"]                    # (so that the test tells the two apart)
    return 0.25 * moved + ATOL["float32"]


def _check(rows, oracle, atol):
    for (rid, pos), row in rows.items():
        err = float((row - oracle[rid][pos]).abs().max())
        assert err <= atol, (rid, pos, err, atol)


@pytest.mark.parametrize("name", ["A", "B", "C"])
@pytest.mark.parametrize("page", [16, 64])
def test_logits_in_every_way_of_cutting_the_work(name, page, tmp_path, monkeypatch):
    raw, seed = TINY[name]
    # (matrices ten times as large as usual: keys and values whose rounding shows in the logits)
    folder = make_folder(str(tmp_path / "m"), raw, seed, "float32")
    _scale(folder, 6.0)
    n = {"A": 100, "B": 200, "C": 300}[name]
    prompts = {"x": random_tokens(n, raw["vocab_size"], 1), "y": random_tokens(n // 3, raw["vocab_size"], 2),
               "z": random_tokens(1, raw["vocab_size"], 3)}
    exact = oracle_logits(folder, prompts)
    want = _oracle4(folder, prompts, monkeypatch)
    atol = _tolerance(want, exact)
    whole = Replayer(folder, "float32", 4 * (n + page), page_size=page, cache_bits=4, max_batched_tokens=512)
    whole.step([(r, ids, range(len(ids))) for r, ids in prompts.items()], end=list(prompts))
    _check(whole.rows, want, atol)
    mixed = Replayer(folder, "float32", 4 * (n + page), page_size=page, cache_bits=4, max_batched_tokens=512)
    at = {r: 0 for r in prompts}
    for k in range(400):
        entries = []
        for i, (r, ids) in enumerate(prompts.items()):
            take = [1, 7, 33, 2][(k + i) % 4]
            part = ids[at[r]:at[r] + take]
            if part:
                entries.append((r, part, range(len(part))))
                at[r] += len(part)
        if not entries:
            break
        mixed.step(entries)
    _check(mixed.rows, want, atol)


def _scale(folder, by):
    """The attention's and feed-forward's matrices of a folder times ``by``."""
    import os
    from safetensors_lite import load, save
    path = os.path.join(folder, "model.safetensors")
    tensors = load(path)
    save(path, {k: v * by if "attn.c_" in k and k.endswith("weight") else v for k, v in tensors.items()})


@pytest.mark.parametrize("graphs", [True, False])
def test_generation_in_bfloat16(graphs, tmp_path, monkeypatch):
    """Greedy tokens from a 4-bit cache: with and without graphs, alone and in a batch the same requests."""
    from pretrained_rstr_b200 import generate_batch, generate_ids, load_lm
    from pretrained_rstr_b200.settings import SETTINGS
    monkeypatch.setattr(SETTINGS, "graphs", graphs)
    folder = make_folder(str(tmp_path / "m"), TINY["C"][0], 2, "bfloat16")
    m = load_lm(folder, max_lanes=4, cache_bits=4)
    assert all(t.dtype == torch.uint8 for t in m.loaded.storage.kv)
    prompts = [random_tokens(n, 700, n) for n in (3, 70, 129, 1, 40)]
    out = generate_batch(m, prompts, 20)
    assert [len(o) for o in out] == [20] * 5 and all(0 <= t < 700 for o in out for t in o)
    assert generate_ids(m, prompts[0], 20) == generate_ids(m, prompts[0], 20)


def test_a_fork_copies_the_page_it_writes_into(tmp_path):
    folder = make_folder(str(tmp_path / "m"), TINY["C"][0], 2, "float32")
    ids = random_tokens(90, 700, 5)
    r = Replayer(folder, "float32", 1024, cache_bits=4)
    r.step([("a", ids[:80], [79])])
    r.lm.cache.fork("a", "b")
    r.pos["b"] = 80
    r.step([("b", [1, 2, 3], [2]), ("a", ids[80:], [9])])
    alone = Replayer(folder, "float32", 1024, cache_bits=4)
    alone.step([("a", ids[:80], [79])])
    alone.step([("a", ids[80:], [9])])
    assert r.lm.runner.counters["cow_copies"] >= 1           # (each that writes into the shared page may copy it)
    assert float((r.rows[("a", 89)] - alone.rows[("a", 89)]).abs().max()) <= ATOL["float32"]


def test_what_does_not_go_in_4_bits_is_refused(tmp_path):
    from pretrained_rstr_b200 import load_lm
    from pretrained_rstr_b200.engine.loading import random_model_folder
    folder = make_folder(str(tmp_path / "m"), TINY["A"][0], 0, "float32")
    with pytest.raises(ValueError, match="cache_bits"):
        load_lm(folder, cache_bits=8)
    with pytest.raises(ValueError, match="pages"):
        load_lm(folder, cache_bits=4, page_size=8)
    with random_model_folder("redisun-tiny", 0) as other:
        with pytest.raises(ValueError, match="cache_bits=4"):
            load_lm(other, cache_bits=4)


# ------------------------------------------------------------------------------- all of them together
@pytest.mark.parametrize("captured", [False, True])
def test_steps_with_drafted_tokens(captured):
    """Rounds of: tables from the lengths, keys and values into the cache, attention, logits, verification; the lengths of
    the next round come from the verification and never leave the device.  Captured: a round is a CUDA graph, replayed."""
    from pretrained_rstr_b200.csrc import ops
    g = torch.Generator().manual_seed(11)
    vocab, d, heads, kv, page, wide, lanes = 40, 32, 4, 2, 16, 6, 5
    b, drafts = 3, [2, 0, 3]
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    emb, wq, wk, wv, wo = rnd(vocab, 24), rnd(24, heads * d), rnd(24, kv * d), rnd(24, kv * d), 0.3 * rnd(heads * d, vocab)
    lane = [3, 0, 4]
    table = torch.full((lanes, wide), -1, dtype=torch.int32)
    table[lane] = torch.randperm(b * wide, generator=g).to(torch.int32).view(b, wide)
    temps = [1.0, 0.0, 0.7]
    brought = [n + 1 for n in drafts]
    starts = [0, 3, 4, 8]
    rows, cap = starts[-1], starts[-1] + 2
    rounds = 6
    given = torch.randint(vocab, (rounds, rows), generator=g)               # drafted tokens; a request's first is its last known
    uniforms = torch.rand(rounds, rows, 2, generator=g)
    first = [7, 11, 2]

    # ---- plain
    history = [[] for _ in range(b)]
    last = list(first)
    want = []
    for r in range(rounds):
        logits, drafted = torch.zeros(rows, vocab, dtype=torch.float64), [0] * rows
        for i in range(b):
            seq = history[i] + [last[i]] + given[r, starts[i] + 1:starts[i + 1]].tolist()
            x = emb[seq].double()
            k, v = (sum(plain.values(*plain.quantize((x.float() @ w).view(len(seq), kv, d)))) for w in (wk, wv))
            for j in range(brought[i]):
                at = len(history[i]) + j
                q = (emb[seq[at]] @ wq).double().view(heads, d)
                o = torch.cat([torch.softmax(0.2 * (k[:at + 1, h // 2] @ q[h]), 0) @ v[:at + 1, h // 2] for h in range(heads)])
                logits[starts[i] + j] = o @ wo.double()
                drafted[starts[i] + j] = int(given[r, starts[i] + j + 1]) if j + 1 < brought[i] else 0
        tokens, accepted = plain.verify(logits.float(), starts, drafted, uniforms[r].tolist(), temps)
        want.append((tokens, accepted))
        for i in range(b):
            history[i] += [last[i]] + tokens[starts[i]:starts[i] + accepted[i]]
            last[i] = tokens[starts[i] + accepted[i]]

    # ---- on the device
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=CUDA)  # noqa: E731
    dev = {n: t.to(CUDA) for n, t in dict(emb=emb, wq=wq, wk=wk, wv=wv, wo=wo).items()}
    tables, held, new, last_d = table.to(CUDA), ints([0] * b), ints(brought), ints(first)
    arr = dict(q_start=ints([0] * (b + 1)), kv_len=ints([0] * b), positions=ints([0] * cap), seq=ints([0] * cap),
               slots=ints([0] * cap), block=ints([[0] * wide] * b))
    tile = plain.tile_bytes(page, d)
    kt, vt = (torch.zeros(b * wide, kv, tile, dtype=torch.uint8, device=CUDA) for _ in range(2))
    status, tokens, accepted = ints([0] * 4), ints([0] * rows), ints([0] * b)
    out, row_start, temp = torch.zeros(cap, heads * d, device=CUDA), ints(starts), torch.tensor(temps, device=CUDA)
    step_tokens, step_uniforms = ints([0] * rows), torch.zeros(rows, 2, device=CUDA)
    firsts, tile_rows = ints(starts[:-1]), ints(brought)
    lane_d, reqs = ints(lane), ints(list(range(b)))
    nxt = torch.tensor([j + 1 if j + 1 not in starts else j for j in range(rows)], device=CUDA)

    def one_round():
        step_tokens[firsts.long()] = last_d
        ops.step_tables(lane_d, held, new, tables, page, arr["q_start"], arr["kv_len"], arr["positions"], arr["seq"],
                        arr["slots"], arr["block"], status)
        x = torch.zeros(cap, 24, device=CUDA)
        x[:rows] = dev["emb"][step_tokens.long()]
        ops.kv_append_4bit(kt, vt, x @ dev["wk"], x @ dev["wv"], arr["slots"], cap, d, page, status)
        ops.attention_4bit(out, x @ dev["wq"], kt, vt, arr["block"], arr["positions"], reqs, firsts, tile_rows, max(brought),
                           heads, d, page, 0.2, None, wide * page, status)
        logits = out[:rows] @ dev["wo"]
        ops.verify_drafts(tokens, accepted, logits, row_start, step_tokens[nxt].contiguous(), step_uniforms, temp, status)
        held.add_(accepted + 1)
        last_d.copy_(tokens[(row_start[:-1] + accepted).long()])

    replay = one_round
    if captured:
        keep = [t.clone() for t in (held, last_d)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one_round()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one_round()
        for t, was in zip((held, last_d), keep):
            t.copy_(was)
        replay = graph.replay
    for r in range(rounds):
        step_tokens.copy_(given[r])
        step_uniforms.copy_(uniforms[r])
        replay()
        assert status.tolist() == [0] * 4
        assert (tokens.tolist(), accepted.tolist()) == want[r], r
    assert held.tolist() == [len(h) for h in history]
