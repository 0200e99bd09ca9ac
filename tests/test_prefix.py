"""What the operators of shared beginnings and beams refuse, which way a call takes, and their books: without a GPU."""

import ctypes

import pytest
import torch

THREE = ctypes.c_int64 * 3
AT = ctypes.c_void_p(1 << 20)      # aligned, never followed: every call here is refused or has nothing to do
OFF = ctypes.c_void_p((1 << 20) + 2)


@pytest.fixture(scope="module")
def lib():
    from tessiq_b200 import _lib

    return _lib


@pytest.mark.parametrize("changed, code", [
    ({"dtype": 0}, "TQ_UNSUPPORTED"), ({"width": 72}, "TQ_UNSUPPORTED"), ({"width": 144}, "TQ_UNSUPPORTED"), ({"page": 8}, "TQ_UNSUPPORTED"), ({"page": 2048}, "TQ_UNSUPPORTED"),
    ({"pages": -1}, "TQ_INVALID_ARGUMENT"), ({"heads": 5}, "TQ_INVALID_ARGUMENT"), ({"kv_heads": 0}, "TQ_INVALID_ARGUMENT"), ({"runs": 0}, "TQ_INVALID_ARGUMENT"),
    ({"runs": 4}, "TQ_INVALID_ARGUMENT"), ({"runs": -1}, "TQ_INVALID_ARGUMENT"), ({"lengths": None}, "TQ_INVALID_ARGUMENT"), ({"shared": None}, "TQ_INVALID_ARGUMENT"),
    ({"table": None}, "TQ_INVALID_ARGUMENT"), ({"ks": None}, "TQ_INVALID_ARGUMENT"), ({"q": OFF}, "TQ_UNSUPPORTED"), ({"v": OFF}, "TQ_UNSUPPORTED"),
    ({"shared": OFF}, "TQ_UNSUPPORTED"), ({"blocks": 1 << 27}, "TQ_UNSUPPORTED"), ({"batch": 3 << 22, "heads": 16, "kv_heads": 1, "runs": 1}, "TQ_UNSUPPORTED"), ({"scale": 0.0}, "TQ_UNSUPPORTED"),
    ({"scale": float("inf")}, "TQ_UNSUPPORTED"), ({"q_strides": THREE(256, 60, 64)}, "TQ_UNSUPPORTED"), ({"batch": 0}, "TQ_OK"), ({"q_tokens": 0}, "TQ_OK"),
], ids=str)
def test_prefix_attention_refuses(lib, changed, code):
    a = dict(dtype=lib.F16, q=AT, k=AT, v=AT, ks=AT, vs=AT, table=AT, lengths=AT, shared=AT, out=AT, batch=6, heads=4, kv_heads=2, q_tokens=1, width=64, pages=9, page=16, blocks=4,
             table_stride=4, runs=2, q_strides=THREE(256, 64, 64), out_strides=THREE(256, 64, 64), scale=0.1)
    a.update(changed)
    got = lib.lib.tq_prefix_attention_launch(a["dtype"], a["q"], a["k"], a["v"], a["ks"], a["vs"], a["table"], a["lengths"], a["shared"], a["out"], a["batch"], a["heads"],
                                             a["kv_heads"], a["q_tokens"], a["width"], a["pages"], a["page"], a["blocks"], a["table_stride"], a["runs"], a["q_strides"],
                                             a["out_strides"], a["scale"], None, 0, 0, None)
    assert got == getattr(lib, code), lib.last_error()


@pytest.mark.parametrize("changed, code", [
    ({"dtype": 1}, "TQ_UNSUPPORTED"), ({"beams": 129}, "TQ_UNSUPPORTED"), ({"keep": 129}, "TQ_UNSUPPORTED"), ({"vocab": 1 << 24}, "TQ_UNSUPPORTED"), ({"requests": 40000}, "TQ_UNSUPPORTED"),
    ({"requests": -1}, "TQ_INVALID_ARGUMENT"), ({"keep": 9, "vocab": 2}, "TQ_INVALID_ARGUMENT"), ({"beams": 0}, "TQ_INVALID_ARGUMENT"), ({"logits": None}, "TQ_INVALID_ARGUMENT"),
    ({"scores": None}, "TQ_INVALID_ARGUMENT"), ({"out": None}, "TQ_INVALID_ARGUMENT"), ({"finished": AT, "end": 100}, "TQ_INVALID_ARGUMENT"), ({"finished": AT, "end": -1}, "TQ_INVALID_ARGUMENT"),
    ({"scores": OFF}, "TQ_UNSUPPORTED"), ({"stride": -1}, "TQ_UNSUPPORTED"), ({}, "TQ_INVALID_ARGUMENT"), ({"requests": 0}, "TQ_OK"), ({"keep": 0}, "TQ_OK"),
], ids=str)
def test_beam_select_refuses(lib, changed, code):
    a = dict(dtype=lib.F32, logits=AT, scores=AT, finished=None, out=AT, requests=2, beams=4, vocab=100, keep=4, end=0, stride=400)
    a.update(changed)      # (the one as it is: for want of a workspace)
    got = lib.lib.tq_beam_select_launch(a["dtype"], a["logits"], a["scores"], a["finished"], a["out"], AT, AT, a["requests"], a["beams"], a["vocab"], a["keep"], a["end"],
                                        a["stride"], 100, None, 0, 0, None)
    assert got == getattr(lib, code), lib.last_error()


@pytest.mark.parametrize("changed, code", [
    ({"page": 24}, "TQ_UNSUPPORTED"), ({"batch": -1}, "TQ_INVALID_ARGUMENT"), ({"pages": 1 << 30}, "TQ_UNSUPPORTED"), ({"batch": 1 << 20}, "TQ_UNSUPPORTED"),
    ({"blocks": 1 << 27, "stride": 1 << 27}, "TQ_UNSUPPORTED"), ({"table": None}, "TQ_INVALID_ARGUMENT"), ({"lengths": None}, "TQ_INVALID_ARGUMENT"), ({"counts": None}, "TQ_INVALID_ARGUMENT"),
    ({"starts": None}, "TQ_INVALID_ARGUMENT"), ({"stride": 3}, "TQ_INVALID_ARGUMENT"), ({"parents": OFF}, "TQ_UNSUPPORTED"), ({"count": 5}, "TQ_INVALID_ARGUMENT"),
    ({"new_table": AT, "new_stride": 5}, "TQ_INVALID_ARGUMENT"), ({}, "TQ_INVALID_ARGUMENT"), ({"batch": 0}, "TQ_UNSUPPORTED"), ({"batch": 0, "pages": 0}, "TQ_OK"),
], ids=str)
def test_cache_advance_refuses(lib, changed, code):
    elsewhere = ctypes.c_void_p(1 << 24)
    a = dict(count=0, table=AT, lengths=AT, references=AT, counts=AT, parents=AT, new_table=elsewhere, new_lengths=elsewhere, new_references=elsewhere, starts=elsewhere, batch=4, blocks=4,
             pages=30, page=16, stride=4, new_stride=4)
    a.update(changed)      # (the one as it is: for want of a workspace)
    got = lib.lib.tq_cache_advance_launch(None, a["count"], a["table"], a["lengths"], a["references"], a["counts"], a["parents"], a["new_table"], a["new_lengths"], a["new_references"],
                                          a["starts"], a["batch"], a["blocks"], a["pages"], a["page"], a["stride"], a["new_stride"], None, 0, 0, None)
    assert got == getattr(lib, code), lib.last_error()


def test_python_refuses_before_the_library():
    from tessiq_b200 import ops

    codes, scales = torch.zeros(9, 2, 16, 64, dtype=torch.float8_e4m3fn), torch.ones(9, 2)
    cache = (codes, codes, scales, scales)
    q, table, lengths, shared = torch.zeros(6, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(6, 3, dtype=torch.int32), torch.zeros(6, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for wrong in (torch.zeros(4, dtype=torch.int32), torch.zeros(2), torch.zeros(0, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="shared is"):
            ops.prefix_attention(q, *cache, table, lengths, wrong)
    with pytest.raises(ValueError, match="evenly"):
        ops.prefix_attention(q[:, :3], *cache, table, lengths, shared)
    with pytest.raises(ValueError, match="lengths are"):
        ops.prefix_attention(q, *cache, table, lengths.long(), shared)
    with pytest.raises(TypeError):
        ops.prefix_attention(q[0], *cache, table, lengths, shared)

    logits, scores = torch.zeros(2, 3, 10), torch.zeros(2, 3)
    for call, what in (((logits[0], scores, 2), "logits are"), ((logits, scores.half(), 2), "scores are"), ((logits, scores.t(), 2), "scores are"), ((logits, scores, 31), "cannot be kept"),
                       ((logits, scores, -1), "cannot be kept"), ((logits, scores, 2, scores > 0, 10), "no token"), ((logits, scores, 2, scores), "finished are")):
        with pytest.raises(ValueError, match=what):
            ops.beam_select(*call)
    with pytest.raises(TypeError):
        ops.beam_select(torch.zeros(2, 10, 3).transpose(1, 2), scores, 2)
    with pytest.raises(TypeError):
        ops.beam_select(logits, scores, 2.0)

    references, counts = torch.zeros(9, dtype=torch.int32), torch.ones(6, dtype=torch.int32)
    good = [*cache, table, lengths, references, counts]
    for at, wrong, what in ((0, codes[0], "cache's pages are"), (0, torch.zeros(9, 2, 16, 64), "pages are float8"), (2, scores, "scales are"), (4, table.long(), "table is"), (4, table[0], "table is"),
                            (5, lengths[:5], "lengths are"), (6, references[:8], "references are"), (6, references.long(), "references are"), (7, counts.long(), "counts are")):
        with pytest.raises(ValueError, match=what):
            ops.cache_advance(*[wrong if i == at else t for i, t in enumerate(good)])
    with pytest.raises(ValueError, match="parents are"):
        ops.cache_advance(*good, torch.zeros(6, dtype=torch.int64))


def form(lib, *extents):
    kind, parts, rows = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int32()
    lib.check(lib.lib.tq_prefix_attention_form(*extents, -1, ctypes.byref(kind), ctypes.byref(parts), ctypes.byref(rows)))
    return {0: "streamed", 1: "tiles", 3: "apart"}[kind.value]


def test_which_way_a_call_takes(lib):
    """batch, heads, kv_heads, q_tokens, width, page_tokens, blocks, runs."""
    assert form(lib, 4, 12, 12, 1, 64, 16, 20, 1) == "apart"                # little to read
    assert form(lib, 64, 32, 8, 1, 128, 64, 133, 64) == "apart"             # nobody to share with
    assert form(lib, 256, 64, 8, 1, 128, 64, 474, 1) == "tiles"
    assert form(lib, 64, 12, 12, 1, 64, 64, 64, 16) == "streamed"
    with pytest.raises(ValueError):
        form(lib, 5, 4, 4, 1, 64, 16, 20, 2)


def test_scratch_is_asked_for_what_a_launch_takes(lib):
    """No scratch where there is nothing to do or the call is refused; some otherwise."""
    size = ctypes.c_size_t()
    for extents in ((0, 4, 4, 1, 64, 16, 20, 1), (4, 4, 3, 1, 64, 16, 20, 1), (4, 4, 4, 1, 64, 16, 20, 3), (4, 4, 4, 1, 64, 24, 20, 1), (4, 4, 4, -1, 64, 16, 20, 1)):
        lib.check(lib.lib.tq_prefix_attention_workspace_bytes(*extents, -1, ctypes.byref(size)))
        assert size.value == 0
    lib.check(lib.lib.tq_prefix_attention_workspace_bytes(256, 64, 8, 1, 128, 64, 474, 1, -1, ctypes.byref(size)))
    assert size.value > 256 * 64 * 128 * 4
    for extents in ((0, 4, 100, 4), (2, 129, 100, 4), (2, 4, 0, 4), (1 << 40, 4, 100, 4)):
        lib.check(lib.lib.tq_beam_select_workspace_bytes(lib.BF16, *extents, ctypes.byref(size)))
        assert size.value == 0
    lib.check(lib.lib.tq_beam_select_workspace_bytes(lib.BF16, 2, 4, 100, 4, ctypes.byref(size)))
    assert size.value >= 8 * 4 * 8
    lib.check(lib.lib.tq_cache_advance_workspace_bytes(4, 1 << 27, 10, 16, ctypes.byref(size)))
    assert size.value == 0


def test_pages_set_aside_and_adopted():
    from tessiq_b200.cache import Pages

    books = Pages(12, 16)
    a = books.start()
    books.extend([a], [20])
    reserved = books.reserve(4)
    assert reserved == [2, 3, 4, 5] and books.free_pages == 6
    with pytest.raises(MemoryError):
        books.reserve(7)
    b = books.adopt([*books.pages_of(a)[:1], 3], 25)
    books.free(a)
    books.drop(reserved)
    assert books.pages_of(b) == [0, 3] and books.length(b) == 25 and books.references[:6] == [1, 0, 0, 1, 0, 0]
    c = books.fork(b)
    assert books.shared_tokens([b, c]) == 25
    books.extend([c], [40])
    assert books.shared_tokens([b, c]) == 16 and books.shared_tokens([c]) == 65
    books.free(b), books.free(c)
    assert books.free_pages == 12


def test_runs_of_an_extended_step():
    from tessiq_b200.cache import PagedCache

    cache = PagedCache(1, 1, 16, 64, 16, device="cpu")
    a, b = cache.start(), cache.start()
    cache.books.extend([a, b], [40, 7])
    rows = [a, cache.books.fork(a), b, cache.books.fork(b)]
    step = cache.extend(rows, 0, runs=2)
    assert step.shared.tolist() == [40, 7] and cache.extend(rows, 0).shared is None
    with pytest.raises(ValueError, match="equal runs"):
        cache.extend(rows, 0, runs=3)
    with pytest.raises(ValueError, match="equal runs"):
        cache.extend(rows, 0, runs=0)


def test_a_step_made_by_position():
    """Books' counts are its sixth and seventh, as before steps knew of shared tokens."""
    from tessiq_b200.cache import Step

    numbers = torch.zeros(1, dtype=torch.int32)
    step = Step(numbers[None], numbers, numbers, numbers, 3, 5, {1: (2, 0)})
    assert step.changes == 5 and step.sequences == {1: (2, 0)} and step.shared is None and step.search is None


@pytest.mark.parametrize("fails", ["tensor", "fork"])
def test_beams_that_cannot_be_made_leave_the_books_as_they_were(monkeypatch, fails):
    from tessiq_b200.cache import PagedCache

    cache = PagedCache(1, 1, 16, 64, 16, device="cpu")
    a, b = cache.start(), cache.start()
    cache.books.extend([a, b], [40, 7])
    before = (list(cache.books.references), sorted(cache.books._free), cache.books.sequences, cache._searches)
    real, calls = cache.books.fork, []

    def fork(sequence):
        calls.append(sequence)
        if len(calls) == 2:
            raise MemoryError("no room")
        return real(sequence)

    def tensor(*_, **__):
        raise torch.OutOfMemoryError("no room")

    with monkeypatch.context() as patch:
        patch.setattr(cache.books, "fork", fork) if fails == "fork" else patch.setattr(torch, "tensor", tensor)
        with pytest.raises((MemoryError, torch.OutOfMemoryError)):
            cache.beams([a, b], 4, 30)
    assert (list(cache.books.references), sorted(cache.books._free), cache.books.sequences, cache._searches) == before
    cache.beams([a, b], 4, 30).free()
    assert (list(cache.books.references), sorted(cache.books._free), cache.books.sequences, cache._searches) == before
    cache.compact()


def test_which_attention_a_step_takes(monkeypatch):
    """What runs share is read once where it is a whole tile and a third of the longest sequence; a window, or little in common, leaves each sequence its own."""
    from tessiq_b200 import cache as module
    from tessiq_b200.cache import PagedCache

    taken = []
    monkeypatch.setattr(module.ops, "prefix_attention", lambda *given: taken.append("together"))
    monkeypatch.setattr(module.ops, "cache_attention", lambda *given: taken.append("each"))
    monkeypatch.setattr(module.ops, "copy_pages", lambda *given, **how: None)
    cache = PagedCache(1, 1, 16, 2000, 16, device="cpu")

    def route(prompts, own, **how):
        sequences = []
        for prompt in prompts:
            first = cache.start()
            cache.books.extend([first], [prompt])
            sequences += [first, cache.books.fork(first)]
        step = cache.extend(sequences, own, runs=len(prompts))
        assert step.shared.tolist() == [prompt // 16 * 16 if own else prompt for prompt in prompts]
        cache.attention(step, 0, None, **how)
        for sequence in sequences:
            cache.books.free(sequence)
        return taken.pop()

    assert route([300], 1) == "together" and route([300], 1, window=64) == "each"
    assert route([30], 1) == "each" and route([127], 0) == "each" and route([128], 0) == "together"      # (no whole tile)
    assert route([320], 600) == "together" and route([320], 700) == "each"
    assert route([320, 20], 200) == "each" and route([320, 320], 200) == "together"
    for prompt, tokens, way in ((300, 64, "together"), (100, 64, "each"), (300, 2000, "each")):
        first = cache.start()
        cache.books.extend([first], [prompt])
        search = cache.beams([first], 2, tokens)
        step = module.Step(search.table, search.lengths, search.lengths, search.lengths, 1, cache.books.changes, {}, search.shared, search.together, search, search.steps)
        cache.attention(step, 0, None)
        assert taken.pop() == way
        search.free(), cache.books.free(first)


def test_scratch_is_enough_for_a_pool_of_no_pages(lib):
    """Such a call is cache_attention's, with what it takes: whichever way the extents choose otherwise."""
    size = [ctypes.c_size_t() for _ in range(2)]
    for batch, heads, kv_heads, q_tokens, width, page, blocks, runs in ((7, 8, 2, 4, 32, 128, 1961, 1), (2, 2, 2, 64, 96, 1024, 635, 1), (56, 16, 2, 2, 128, 16, 333, 8),
                                                                       (64, 12, 12, 1, 64, 64, 64, 16), (256, 64, 8, 1, 128, 64, 474, 1)):
        lib.check(lib.lib.tq_prefix_attention_workspace_bytes(batch, heads, kv_heads, q_tokens, width, page, blocks, runs, -1, ctypes.byref(size[0])))
        lib.check(lib.lib.tq_cache_attention_workspace_bytes(batch, heads, kv_heads, q_tokens, width, page, blocks, 0, 0, -1, ctypes.byref(size[1])))
        assert form(lib, batch, heads, kv_heads, q_tokens, width, page, blocks, runs) != "apart" and size[0].value >= size[1].value
