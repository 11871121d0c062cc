"""The engine in its default type over a cache held in 4 bits, against the plain implementation whose keys and values go
through 4 bits: prompts whole, in portions that go to the tensor-memory kernel, a few tokens at a time and one by one,
launched kernel by kernel and replayed as CUDA graphs; the tiny configurations and GPT-2's own widths."""
import math

import pytest
import torch

import plain_cache4 as plain
import plain_gpt2
from helpers import ATOL, TINY, Replayer, bf16_atol, make_folder, oracle_rows, random_tokens, real_width

pytestmark = pytest.mark.gpu
WIDTHS = {"A": TINY["A"], "B": TINY["B"], "C": TINY["C"], "small": (real_width("small"), 2), "xl": (real_width("xl"), 4)}
LENGTHS = {"A": [100, 40, 9], "B": [200, 70, 9], "C": [300, 131, 9], "small": [300, 131, 40], "xl": [260, 70, 9]}


def _attention(rounded, weight=1.0):
    """The plain attention with every key and value as a 4-bit cache gives it back (or as it is)."""
    def attention(x_ln, c_attn_w, c_attn_b, c_proj_w, c_proj_b, n_head, scale, window=None):
        t, d = x_ln.shape
        qkv = plain_gpt2.linear_conv1d(x_ln, c_attn_w, c_attn_b)
        q, k, v = (x.reshape(t, n_head, -1) for x in qkv.split(d, 1))
        if rounded:
            k, v = (sum(plain.values(*plain.quantize(x))).float() for x in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * scale
        s = s.masked_fill(torch.ones(t, t).triu(1).bool(), -math.inf)
        out = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(t, d)
        return plain_gpt2.linear_conv1d(weight * out, c_proj_w, c_proj_b)
    return attention


def _picked(n):
    return sorted({0, 1, 2, 8, 9, 62, 63, 64, 65, 127, 128, 129} & set(range(n)) | set(range(max(0, n - 20), n)))


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    """Folder, prompts, plain logits and the tolerance per model, made when first asked for."""
    made = {}

    def get(name):
        if name not in made:
            raw, seed = WIDTHS[name]
            folder = make_folder(str(tmp_path_factory.mktemp(name)), raw, seed, "bfloat16")
            prompts = {f"r{i}": random_tokens(n, raw["vocab_size"], 7 * i + n) for i, n in enumerate(LENGTHS[name])}
            wanted = {r: _picked(len(ids)) for r, ids in prompts.items()}
            runs = []
            for rounded, weight in ((True, 1.0), (False, 1.0), (True, 0.0)):
                with pytest.MonkeyPatch.context() as m:
                    m.setattr(plain_gpt2, "causal_attention", _attention(rounded, weight))
                    runs.append(oracle_rows(folder, prompts, wanted))
            want, exact, none = runs
            apart = lambda a, b: torch.stack([a[r][p] - b[r][p] for r in a for p in a[r]])  # noqa: E731
            # bfloat16 activations move a key or value by up to 2^-8 of itself, which takes one code in some fifty to its
            # neighbour, a whole step: together less than what rounding ALL of them by up to half a step does to the logits,
            # which the two plain runs say.  Half of that again, since the largest of some ten thousands is compared, and
            # what roundings of activations do beside the cache.
            moved = apart(want, exact)
            atol = 1.5 * float(moved.abs().max()) + (ATOL["bfloat16"] if name in TINY else bf16_atol(raw["n_embd"]))
            # (so that the test tells the attention from one that adds nothing)
            assert float(apart(want, none).abs().amax(-1)[1:].min()) > 1.5 * atol
            made[name] = folder, prompts, wanted, want, atol, float(moved.square().mean().sqrt())
        return made[name]
    return get


def _compare(rows, want, wanted, atol, rms):
    errors = []
    for r, picked in wanted.items():
        for p in picked:
            err = rows[(r, p)] - want[r][p]
            assert float(err.abs().max()) <= atol, (r, p, float(err.abs().max()), atol)
            errors.append(err)
    together = float(torch.stack(errors).square().mean().sqrt())
    assert together <= rms + 3e-3, (together, rms)


def _replay(rp, prompts, wanted, sizes):
    """Every request in portions of ``sizes`` tokens, in turn; the wanted logits rows."""
    at, k = {r: 0 for r in prompts}, 0
    while any(at[r] < len(ids) for r, ids in prompts.items()):
        entries = []
        for i, (r, ids) in enumerate(prompts.items()):
            part = ids[at[r]:at[r] + sizes[(k + i) % len(sizes)]]
            if part:
                entries.append((r, part, [p - at[r] for p in wanted[r] if at[r] <= p < at[r] + len(part)]))
                at[r] += len(part)
        rp.step(entries)
        k += 1


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("sizes", [[512], [129, 40], [33, 9, 64], [1, 8, 2], [1]], ids=str)
@pytest.mark.parametrize("name", list(WIDTHS))
def test_logits_in_bfloat16(models, name, sizes, graphs):
    folder, prompts, wanted, want, atol, rms = models(name)
    if sizes == [1]:
        prompts, wanted = ({r: ids[:70] for r, ids in prompts.items()}, {r: [p for p in w if p < min(70, len(prompts[r]))] for r, w in wanted.items()})
    rp = Replayer(folder, "bfloat16", 1024, cache_bits=4, max_batched_tokens=1024)
    rp.lm.runner.use_graphs = graphs
    _replay(rp, prompts, wanted, sizes)
    if max(sizes) <= 8:
        assert bool(rp.lm.runner._graphs) == graphs
    _compare(rp.rows, want, wanted, atol, rms)
