"""What the entry points of the 4-bit cache, the step tables and the drafted tokens refuse before anything is launched,
and the plain statement that their kernels are tested against."""
import math

import pytest
import torch

import plain_cache4 as plain


def test_packing_and_unpacking():
    g = torch.Generator().manual_seed(0)
    for d in (16, 48, 64, 80, 112, 128):
        x = torch.randn(3, 2, 16, d, generator=g)
        q = plain.quantize(x)
        tiles = plain.pack(*q)
        assert tiles.shape == (3, 2, plain.tile_bytes(16, d))
        for a, b in zip(plain.unpack(tiles, 16, d), q):
            assert torch.equal(a.double(), b.double())


def test_a_number_comes_back_within_its_roundings():
    """Half a step, and where step and middle were rounded (2^-8 of each) at the ends of the range."""
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(1)).double()
    codes, step, middle = plain.quantize(x)
    a, b = plain.values(codes, step, middle)
    wide = step.repeat_interleave(32, -1)
    err = (a + b - x).abs()
    assert bool((err <= wide * (0.5 + 8 * 2.0 ** -8) + middle.abs().repeat_interleave(32, -1) * 2.0 ** -8).all())


def test_values_on_the_border_of_two_codes_go_to_the_even_one():
    x = torch.zeros(1, 32)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3], x[0, 4] = -8.0, 7.0, 0.5, 1.5, -2.5
    codes, step, middle = plain.quantize(x)
    assert step.item() == 1.0 and middle.item() == 0.0
    assert codes[0, :5].tolist() == [0.0, 15.0, 8.0, 10.0, 6.0]


def test_the_plain_attention_is_a_softmax_over_what_the_cache_stands_for():
    g = torch.Generator().manual_seed(2)
    kt, vt = (plain.pack(*plain.quantize(torch.randn(3, 1, 16, 32, generator=g))) for _ in range(2))
    q = torch.randn(1, 64, generator=g)
    out, _terms = plain.attention(q, kt, vt, [[2, 0]], [20], [0], 2, 32, 16, 0.3, 5)
    read = lambda t: sum(plain.values(*plain.unpack(t[[2, 0]], 16, 32))).transpose(0, 1).flatten(1, 2)[0, 16:21]  # noqa: E731
    k, v = read(kt), read(vt)
    for h in range(2):
        w = torch.exp(0.3 * (k @ q[0, 32 * h:32 * h + 32].double()))
        assert torch.allclose(out[0, 32 * h:32 * h + 32], (w @ v) / w.sum(), atol=1e-12)


def test_the_plain_verification_follows_the_rule():
    logits = torch.log(torch.tensor([[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]]))
    q = torch.tensor([[0.2, 0.7, 0.1], [0.3, 0.3, 0.4]])
    # stays: 0.4 * 0.7 < 0.3; behind it the last row's own draw
    assert plain.verify(logits, [0, 2], [1, 0], [[0.4, 0.9], [0.0, 0.15]], [1.0], q) == ([1, 1], [1])
    # refused: 0.5 * 0.7 > 0.3; the rest of p - q is (0.3, 0, 0.1)
    assert plain.verify(logits, [0, 2], [1, 0], [[0.5, 0.7], [0.0, 0.0]], [1.0], q) == ([0, -1], [0])
    assert plain.verify(logits, [0, 2], [1, 0], [[0.5, 0.8], [0.0, 0.0]], [1.0], q) == ([2, -1], [0])
    assert plain.verify(logits, [0, 2], [0, 0], [[0.5, 0.8], [0.0, 0.0]], [0.0]) == ([0, 2], [1])


@pytest.mark.parametrize("group", [1, 2, 4, 8, 40])
def test_tiles_of_a_step(group):
    """Every token of a step lies in one tile of its request, in order; short ones in the list of few rows."""
    import numpy as np
    from pretrained_rstr_b200.parts.attention import Attention4Work
    work = Attention4Work(group)
    lengths = [1, 130, 8, 9, 1, 300, 2, 128]
    room = {n: np.full(words, fill, np.int32) for n, (words, fill) in work.arrays(sum(lengths), len(lengths)).items()}
    counts = work.fill(room, lengths)
    seen = []
    for name, counter, most in (("few", "few", work.few_most), ("tile", "tiles", work.tile_most)):
        for i in range(counts[counter]):
            req, row, n = (int(room[f"{name}_{part}"][i]) for part in ("req", "row0", "rows"))
            assert 1 <= n <= most and n * group <= (max(8, group) if name == "few" else max(128, group))
            seen += [(t, req) for t in range(row, row + n)]
        assert set(room[f"{name}_req"][counts[counter]:]) <= {-1}
    assert sorted(seen) == list(enumerate(b for b, n in enumerate(lengths) for _ in range(n)))
    assert counts["few"] == sum(1 for n in lengths if n <= work.few_most)
    one = work.fill({n: np.full(words, fill, np.int32) for n, (words, fill) in work.arrays(8, 8).items()}, [1] * 8)
    assert one["tiles"] == 0 and one["few"] == 8 and one["_used"] == ["few_req", "few_row0", "few_rows"]


# ------------------------------------------------------------------------------------ refusals
# (shapes and types are looked at before the library is asked for anything: no device is needed to be refused)
class _FakeCuda(torch.Tensor):
    """A tensor that says it lies on the GPU; nothing may get as far as its memory."""
    def get_device(self):
        return 0


def fake(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_FakeCuda)


@pytest.fixture
def ops(monkeypatch):
    from pretrained_rstr_b200.csrc import ops as module

    def launched(*_a, **_k):
        raise AssertionError("a refused call reached the library")
    monkeypatch.setattr(module, "lib", launched)
    monkeypatch.setattr(module, "_LIB", None)
    return module


def _append_args(**kw):
    a = dict(k_tiles=fake(4, 2, plain.tile_bytes(16, 32), dtype=torch.uint8),
             v_tiles=fake(4, 2, plain.tile_bytes(16, 32), dtype=torch.uint8), k=fake(5, 64, dtype=torch.bfloat16),
             v=fake(5, 64, dtype=torch.bfloat16), slots=fake(5), n_tokens=5, head_dim=32, page_size=16, status=fake(4))
    a.update(kw)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(head_dim=24), "multiples of 16"), (dict(head_dim=144), "up to 128"), (dict(page_size=8), "pages"),
    (dict(k=fake(5, 60, dtype=torch.bfloat16)), "k must be"), (dict(v=fake(4, 64, dtype=torch.bfloat16)), "v must be"),
    (dict(k=fake(5, 64, dtype=torch.float32)), "differ in type"), (dict(k=fake(5, 64, dtype=torch.float16)), "not supported"),
    (dict(slots=fake(4)), "slots"), (dict(slots=fake(5, dtype=torch.int64)), "slots"),
    (dict(k_tiles=fake(4, 2, 100, dtype=torch.uint8)), "k_tiles"), (dict(status=fake(2)), "status"),
    (dict(v_tiles=fake(3, 2, plain.tile_bytes(16, 32), dtype=torch.uint8)), "differ in shape"),
    (dict(k=torch.zeros(5, 64, dtype=torch.bfloat16)), "not on a CUDA device"),
    (dict(n_tokens=-1), "n_tokens"), (dict(k=fake(1, 64, dtype=torch.bfloat16).expand(5, 64), n_tokens=6), "k must be")])
def test_rows_refused(ops, change, word):
    with pytest.raises(ops.KernelArgumentError, match=word):
        ops.kv_append_4bit(**_append_args(**change))
    back = _append_args(**change)
    back["k_out"], back["v_out"] = back.pop("k"), back.pop("v")
    with pytest.raises(ops.KernelArgumentError, match=word.replace("k must", "k_out must").replace("v must", "v_out must")):
        ops.kv_read_4bit(**back)


def _attention_args(**kw):
    a = dict(out=fake(6, 128, dtype=torch.bfloat16), q=fake(6, 128, dtype=torch.bfloat16),
             k_tiles=fake(4, 2, plain.tile_bytes(16, 32), dtype=torch.uint8),
             v_tiles=fake(4, 2, plain.tile_bytes(16, 32), dtype=torch.uint8), block_table=fake(3, 7), positions=fake(6),
             tile_req=fake(2), tile_row0=fake(2), tile_rows=fake(2), tile_most=4, n_heads=4, head_dim=32, page_size=16,
             scale=0.1, window=None, max_context=50, status=fake(4))
    a.update(kw)
    return a


_Q = fake(6, 128, dtype=torch.bfloat16)


@pytest.mark.parametrize("change,word", [
    (dict(n_heads=3), "multiple"), (dict(n_heads=0), "multiple"), (dict(q=fake(6, 120, dtype=torch.bfloat16)), "q must be"),
    (dict(out=fake(5, 128, dtype=torch.bfloat16)), "out must be"), (dict(out=fake(6, 128, dtype=torch.float32)), "differ in type"),
    (dict(positions=fake(5)), "positions"), (dict(tile_rows=fake(1)), "tile_rows"), (dict(window=0), "window"),
    (dict(window=-3), "window"), (dict(tile_count=fake(0)), "tile_count"), (dict(block_table=fake(7)), "block_table"),
    (dict(block_table=fake(3, 7, dtype=torch.int64)), "block_table"), (dict(q=_Q, out=_Q), "out must not be q"),
    (dict(tile_most=0), "tile_most"), (dict(max_context=0), "max_context"), (dict(parts=9), "parts"),
    (dict(out=fake(1, 128, dtype=torch.bfloat16).expand(6, 128)), "out must be"), (dict(scale=math.nan), "scale"), (dict(head_dim=40), "multiples of 16")])
def test_attention_refused(ops, change, word):
    with pytest.raises(ops.KernelArgumentError, match=word):
        ops.attention_4bit(**_attention_args(**change))


def _table_args(**kw):
    a = dict(rows=fake(3), held=fake(3), brought=fake(3), tables=fake(5, 4), page_size=16, q_start=fake(4), kv_len=fake(3),
             positions=fake(9), seq_of_token=fake(9), slots=fake(9), block_table=fake(3, 4), status=fake(4),
             free_pages=fake(2), free_start=fake(1), free_next=fake(1))
    a.update(kw)
    return a


_ONE = fake(1)
_T = fake(5, 4)


@pytest.mark.parametrize("change,word", [
    (dict(rows=fake(2)), "rows"), (dict(q_start=fake(3)), "q_start"), (dict(slots=fake(8)), "slots"),
    (dict(block_table=fake(2, 4)), "block_table"), (dict(block_table=fake(3, 5)), "block_table"),
    (dict(tables=fake(4)), "tables"), (dict(page_size=0), "page_size"), (dict(held=fake(0)), "requests"),
    (dict(held=fake(4097)), "requests"), (dict(free_start=None), "free_start"), (dict(free_next=None), "free_next"),
    (dict(free_start=_ONE, free_next=_ONE), "free_next must not"), (dict(brought=fake(3, dtype=torch.int64)), "brought"),
    (dict(tables=_T, block_table=_T), "two tensors")])
def test_tables_refused(ops, change, word):
    with pytest.raises(ops.KernelArgumentError, match=word):
        ops.step_tables(**_table_args(**change))


def _verify_args(**kw):
    f = torch.float32
    a = dict(tokens=fake(6), accepted=fake(2), logits=fake(6, 10, dtype=f), row_start=fake(3), drafted=fake(6),
             uniforms=fake(6, 2, dtype=f), temperature=fake(2, dtype=f), status=fake(4), draft_probs=fake(6, 10, dtype=f))
    a.update(kw)
    return a


_W = fake(6)


@pytest.mark.parametrize("change,word", [
    (dict(logits=fake(6, 10, dtype=torch.bfloat16)), "logits"), (dict(draft_probs=fake(6, 9, dtype=torch.float32)), "differ in shape"),
    (dict(uniforms=fake(5, 2, dtype=torch.float32)), "uniforms"), (dict(row_start=fake(2)), "row_start"),
    (dict(accepted=fake(1)), "accepted"), (dict(temperature=fake(2, dtype=torch.float64)), "temperature"),
    (dict(logits=fake(6, 0, dtype=torch.float32), draft_probs=None), "vocabulary"), (dict(drafted=fake(6, dtype=torch.int64)), "drafted"),
    (dict(tokens=_W, drafted=_W), "two tensors"), (dict(tokens=fake(5)), "tokens")])
def test_verification_refused(ops, change, word):
    with pytest.raises(ops.KernelArgumentError, match=word):
        ops.verify_drafts(**_verify_args(**change))


# Tensors that share memory: the library itself refuses them, before it asks for a device.
@pytest.fixture
def real_ops(monkeypatch):
    from pretrained_rstr_b200.csrc import ops as module
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda _d: 0, raising=False)
    return module


@pytest.mark.parametrize("ours,theirs", [
    ("kv_len", "held"), ("kv_len", "brought"), ("kv_len", "rows"), ("q_start", "held"), ("slots", "positions"),
    ("positions", "seq_of_token"), ("free_next", "held"), ("block_table", "free_pages"), ("kv_len", "q_start")])
@pytest.mark.parametrize("behind", [0, 2])
def test_tables_that_share_memory_are_refused(real_ops, ours, theirs, behind):
    a = _table_args()
    pool = fake(64)
    if behind and a[theirs].numel() <= behind:
        behind = 0
    for name, at in ((theirs, 8), (ours, 8 + behind)):
        a[name] = pool[at:at + a[name].numel()].view(a[name].shape)
    with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
        real_ops.step_tables(**a)


@pytest.mark.parametrize("ours,theirs", [("accepted", "row_start"), ("accepted", "drafted"), ("tokens", "row_start"),
                                         ("tokens", "accepted"), ("tokens", "uniforms"), ("accepted", "temperature"),
                                         ("tokens", "logits"), ("accepted", "draft_probs")])
def test_verification_of_shared_memory_is_refused(real_ops, ours, theirs):
    a = _verify_args()
    a[ours] = a[theirs].view(torch.int32).flatten()[-a[ours].numel():] if a[theirs].numel() >= a[ours].numel() else a[ours]
    if a[theirs].numel() < a[ours].numel():
        a[theirs] = a[ours][:a[theirs].numel()].view(a[theirs].dtype)
    with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
        real_ops.verify_drafts(**a)


@pytest.mark.parametrize("q_at,out_at,stride", [(0, 256, 256), (256, 0, 256), (0, 64, 256), (64, 0, 256), (0, 192, 256),
                                                (0, 512 + 100, 256)])
def test_attention_rows_that_share_memory_are_refused(real_ops, q_at, out_at, stride):
    pool = fake(4096, dtype=torch.bfloat16)

    def rows(at):
        return pool.as_strided((6, 128), (stride, 1), at)
    with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
        real_ops.attention_4bit(**_attention_args(q=rows(q_at), out=rows(out_at)))


def test_cache_rows_that_share_memory_are_refused(real_ops):
    a = _append_args()
    with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
        real_ops.kv_append_4bit(**dict(a, v_tiles=a["k_tiles"]))
    rows = fake(5, 100, dtype=torch.bfloat16)
    back = {k: v for k, v in a.items() if k not in "kv"}
    for v_out in (rows[:, :64], rows[:, 36:]):
        with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
            real_ops.kv_read_4bit(k_out=rows[:, :64], v_out=v_out, **back)


# ------------------------------------------------------------------------------------ layout of a model's caches
def _layout(bits, specs, readers=()):
    """A model of one layer a spec, and of layers that read the cache of layer 0: only its layout is derived."""
    from types import SimpleNamespace as Some
    from pretrained_rstr_b200.models.assembly import Model
    blocks = [Some(mixer=Some(kv_spec=lambda s=s: s, state_specs=lambda: ())) for s in (*specs, *readers)]
    order = [Some(layer=i, cache_layer=i if i < len(specs) else 0, writes_cache=i < len(specs)) for i in range(len(blocks))]
    m = Some(runtime=Some(cache_bits=bits), order=order, blocks=blocks, embedding=object(), state_specs={}, group_specs=[],
             layer_group={})
    Model._derive_cache_layout(m)
    return m


def test_layout_of_caches_in_4_bits():
    from pretrained_rstr_b200.parts.interfaces import KVSpec
    four, plain_kv = KVSpec(4, 64, bits=4), KVSpec(4, 64)
    assert [g.bits for g in _layout(4, [four, four], [four]).group_specs] == [4]
    assert [g.bits for g in _layout(None, [plain_kv], [plain_kv]).group_specs] == [None]
    with pytest.raises(ValueError, match="runtime's type only"):
        _layout(4, [four, plain_kv])
    with pytest.raises(ValueError, match="bits differ"):
        _layout(4, [four], [plain_kv])
    with pytest.raises(ValueError, match="no keys and values"):
        _layout(4, [None])
    assert _layout(None, [None]).group_specs == []


# ------------------------------------------------------------------------------------ the edges of what the calls take
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.125, -math.inf, math.inf])
def test_a_scale_that_is_not_above_zero_is_refused(ops, scale):
    """Scores are masked and compared before they are scaled: a scale below zero would make the masked ones the largest."""
    with pytest.raises(ops.KernelArgumentError, match="scale"):
        ops.attention_4bit(**_attention_args(scale=scale))


@pytest.mark.parametrize("scale", [1e-60, 1e300, 1e38])
def test_a_scale_that_32_bits_do_not_hold_is_refused(real_ops, scale):
    with pytest.raises(real_ops.KernelArgumentError, match="bad argument"):
        real_ops.attention_4bit(**_attention_args(scale=scale))


def _over(a, ours, theirs, end):
    """The arguments with tensor ``ours`` beginning in the last (``end``) or first bytes of ``theirs``."""
    t, o = a[theirs], a[ours]
    span = (t.shape[0] - 1) * t.stride(0) * t.element_size() + t[0].numel() * t.element_size()
    own = o.numel() * o.element_size()
    pool = fake(span + own + 64, dtype=torch.uint8)
    at = (span - 1) // 16 * 16 if end else 0
    if t.is_contiguous():
        theirs_now = pool[:span].view(t.dtype).view(t.shape)
    else:
        theirs_now = pool[:(t.shape[0] - 1) * t.stride(0) * t.element_size() + t.stride(0) * t.element_size()].view(t.dtype) \
            .view(t.shape[0], -1)[:, :t.shape[1]]
    return dict(a, **{theirs: theirs_now, ours: pool[at:at + own].view(o.dtype).view(o.shape)})


@pytest.mark.parametrize("end", [False, True])
@pytest.mark.parametrize("ours,theirs", [("k_tiles", "k"), ("k_tiles", "v"), ("v_tiles", "k"), ("v_tiles", "v"), ("k_tiles", "slots"),
                                         ("v_tiles", "slots"), ("k_tiles", "v_tiles"), ("k_tiles", "status"), ("status", "slots")])
def test_rows_into_what_the_call_reads_are_refused(real_ops, ours, theirs, end):
    with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
        real_ops.kv_append_4bit(**_over(_append_args(), ours, theirs, end))


@pytest.mark.parametrize("end", [False, True])
@pytest.mark.parametrize("ours,theirs", [("k_out", "k_tiles"), ("k_out", "v_tiles"), ("v_out", "k_tiles"), ("v_out", "v_tiles"),
                                         ("k_out", "slots"), ("v_out", "slots"), ("k_out", "status"), ("status", "v_tiles")])
def test_rows_back_over_what_the_call_reads_are_refused(real_ops, ours, theirs, end):
    a = _append_args()
    a["k_out"], a["v_out"] = a.pop("k"), a.pop("v")
    with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
        real_ops.kv_read_4bit(**_over(a, ours, theirs, end))


@pytest.mark.parametrize("end", [False, True])
@pytest.mark.parametrize("ours,theirs", [("out", n) for n in ("k_tiles", "v_tiles", "block_table", "positions", "tile_req",
                                                              "tile_row0", "tile_rows", "tile_count", "status")] +
                         [("status", "q"), ("status", "k_tiles"), ("status", "block_table")])
def test_attention_over_what_the_call_reads_is_refused(real_ops, ours, theirs, end):
    with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
        real_ops.attention_4bit(**_over(_attention_args(tile_count=fake(1)), ours, theirs, end))


@pytest.mark.parametrize("name", ["rows", "held", "brought", "tables", "slots", "block_table", "free_pages"])
def test_a_status_word_within_a_steps_tables_is_refused(real_ops, name):
    with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
        real_ops.step_tables(**_over(_table_args(), "status", name, False))


@pytest.mark.parametrize("name", ["tokens", "accepted", "logits", "drafted", "uniforms", "temperature", "row_start"])
def test_a_status_word_within_what_is_verified_is_refused(real_ops, name):
    with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
        real_ops.verify_drafts(**_over(_verify_args(), "status", name, False))


@pytest.mark.parametrize("change,word", [
    (dict(have_pages=fake(3)), "come together"), (dict(have_next=fake(3)), "come together"),
    (dict(have_pages=fake(3), have_next=fake(3), free_pages=None, free_start=None, free_next=None), "with free_pages"),
    (dict(have_pages=fake(2), have_next=fake(3)), "have_pages"), (dict(have_pages=fake(3), have_next=fake(2)), "have_next"),
    (dict(have_pages=fake(3, dtype=torch.int64), have_next=fake(3)), "have_pages"),
    (dict(have_pages=fake(3), have_next=torch.zeros(3, dtype=torch.int32)), "have_next is not on")])
def test_counts_of_pages_refused(ops, change, word):
    with pytest.raises(ops.KernelArgumentError, match=word):
        ops.step_tables(**_table_args(**change))


@pytest.mark.parametrize("theirs", ["have_pages", "held", "rows", "kv_len", "tables", "free_pages"])
def test_counts_of_pages_that_share_memory_are_refused(real_ops, theirs):
    a = _table_args(have_pages=fake(3), have_next=fake(3))
    with pytest.raises(real_ops.KernelArgumentError, match="overlaps"):
        real_ops.step_tables(**_over(a, "have_next", theirs, False))
