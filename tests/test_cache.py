"""Window attention and the paged cache without a GPU: what their entry points refuse."""

import ctypes

import pytest
import torch

THREE = ctypes.c_int64 * 3


@pytest.fixture(scope="module")
def lib():
    from tessiq_b200 import _lib

    return _lib


AT = ctypes.c_void_p(1 << 20)      # aligned, never followed: every call here is refused or has nothing to do
OFF = ctypes.c_void_p((1 << 20) + 2)


def window(lib, **changed):
    a = dict(dtype=lib.BF16, q=AT, k=AT, v=AT, out=AT, batch=2, heads=4, kv_heads=2, q_tokens=3, k_tokens=50, width=64, scale=0.125, window=8, sinks=2,
             q_strides=THREE(4 * 3 * 64, 3 * 64, 64), k_strides=THREE(2 * 50 * 64, 50 * 64, 64), out_strides=THREE(4 * 3 * 64, 3 * 64, 64))
    a.update(changed)
    return lib.lib.tq_window_attention_launch(a["dtype"], a["q"], a["k"], a["v"], a["out"], a["batch"], a["heads"], a["kv_heads"], a["q_tokens"], a["k_tokens"],
                                              a["width"], a["q_strides"], a["k_strides"], a["k_strides"], a["out_strides"], a["scale"], a["window"], a["sinks"],
                                              None, 0, 0, None)


@pytest.mark.parametrize("changed, code", [
    ({"dtype": 0}, "TQ_UNSUPPORTED"), ({"width": 63}, "TQ_UNSUPPORTED"), ({"width": 136}, "TQ_UNSUPPORTED"), ({"heads": 3}, "TQ_INVALID_ARGUMENT"),
    ({"kv_heads": 0}, "TQ_INVALID_ARGUMENT"), ({"batch": -1}, "TQ_INVALID_ARGUMENT"), ({"window": -1}, "TQ_INVALID_ARGUMENT"), ({"sinks": -2}, "TQ_INVALID_ARGUMENT"),
    ({"scale": 0.0}, "TQ_UNSUPPORTED"), ({"scale": float("nan")}, "TQ_UNSUPPORTED"), ({"scale": 3e38}, "TQ_UNSUPPORTED"), ({"q": None}, "TQ_INVALID_ARGUMENT"), ({"out": None}, "TQ_INVALID_ARGUMENT"),
    ({"v": None}, "TQ_INVALID_ARGUMENT"), ({"q": OFF}, "TQ_UNSUPPORTED"), ({"k": OFF}, "TQ_UNSUPPORTED"), ({"k_strides": THREE(6400, 3200, 60)}, "TQ_UNSUPPORTED"),
    ({"k_strides": THREE(6400, 0, 64)}, "TQ_UNSUPPORTED"), ({"q_strides": THREE(768, 196, 64)}, "TQ_UNSUPPORTED"), ({"out_strides": THREE(768, -192, 64)}, "TQ_INVALID_ARGUMENT"),
    ({"k_tokens": 1 << 31}, "TQ_UNSUPPORTED"), ({"q_tokens": 1 << 31}, "TQ_UNSUPPORTED"), ({"k_strides": None}, "TQ_INVALID_ARGUMENT"),
    ({"batch": 0}, "TQ_OK"), ({"heads": 0, "kv_heads": 0}, "TQ_OK"), ({"q_tokens": 0}, "TQ_OK"),
], ids=str)
def test_window_attention_refuses(lib, changed, code):
    assert window(lib, **changed) == getattr(lib, code), lib.last_error()


def attend(lib, **changed):
    a = dict(dtype=lib.F16, q=AT, k=AT, v=AT, ks=AT, vs=AT, table=AT, lengths=AT, out=AT, batch=2, heads=4, kv_heads=2, q_tokens=1, width=64, pages=9, page=16, blocks=4,
             table_stride=4, q_strides=THREE(256, 64, 64), out_strides=THREE(256, 64, 64), scale=0.1, window=0, sinks=0)
    a.update(changed)
    return lib.lib.tq_cache_attention_launch(a["dtype"], a["q"], a["k"], a["v"], a["ks"], a["vs"], a["table"], a["lengths"], a["out"], a["batch"], a["heads"], a["kv_heads"],
                                             a["q_tokens"], a["width"], a["pages"], a["page"], a["blocks"], a["table_stride"], a["q_strides"], a["out_strides"],
                                             a["scale"], a["window"], a["sinks"], None, 0, 0, None)


@pytest.mark.parametrize("changed, code", [
    ({"dtype": 1}, "TQ_UNSUPPORTED"), ({"width": 72}, "TQ_UNSUPPORTED"), ({"width": 144}, "TQ_UNSUPPORTED"), ({"page": 8}, "TQ_UNSUPPORTED"), ({"page": 48}, "TQ_UNSUPPORTED"),
    ({"page": 2048}, "TQ_UNSUPPORTED"), ({"pages": -1}, "TQ_INVALID_ARGUMENT"), ({"heads": 5}, "TQ_INVALID_ARGUMENT"), ({"kv_heads": 0}, "TQ_INVALID_ARGUMENT"),
    ({"window": -4}, "TQ_INVALID_ARGUMENT"), ({"lengths": None}, "TQ_INVALID_ARGUMENT"), ({"table": None}, "TQ_INVALID_ARGUMENT"), ({"ks": None}, "TQ_INVALID_ARGUMENT"),
    ({"q": OFF}, "TQ_UNSUPPORTED"), ({"v": OFF}, "TQ_UNSUPPORTED"), ({"table": OFF}, "TQ_UNSUPPORTED"), ({"blocks": 1 << 27}, "TQ_UNSUPPORTED"),
    ({"scale": -1.0}, "TQ_UNSUPPORTED"), ({"scale": float("inf")}, "TQ_UNSUPPORTED"), ({"scale": 1e39}, "TQ_UNSUPPORTED"), ({"batch": 0}, "TQ_OK"), ({"q_tokens": 0}, "TQ_OK"),
], ids=str)
def test_cache_attention_refuses(lib, changed, code):
    assert attend(lib, **changed) == getattr(lib, code), lib.last_error()


def store(lib, **changed):
    a = dict(dtype=lib.F16, k=AT, v=AT, kp=AT, vp=AT, ks=AT, vs=AT, table=AT, starts=AT, counts=None, batch=2, kv_heads=2, tokens=3, width=64, pages=9, page=16, blocks=4,
             table_stride=4, strides=THREE(384, 192, 64))
    a.update(changed)
    return lib.lib.tq_cache_store_launch(a["dtype"], a["k"], a["v"], a["kp"], a["vp"], a["ks"], a["vs"], a["table"], a["starts"], a["counts"], a["batch"], a["kv_heads"],
                                         a["tokens"], a["width"], a["pages"], a["page"], a["blocks"], a["table_stride"], a["strides"], a["strides"], 0, None)


@pytest.mark.parametrize("changed, code", [
    ({"dtype": 0}, "TQ_UNSUPPORTED"), ({"width": 8}, "TQ_UNSUPPORTED"), ({"page": 17}, "TQ_UNSUPPORTED"), ({"tokens": -1}, "TQ_INVALID_ARGUMENT"), ({"k": None}, "TQ_INVALID_ARGUMENT"),
    ({"starts": None}, "TQ_INVALID_ARGUMENT"), ({"vp": None}, "TQ_INVALID_ARGUMENT"), ({"strides": THREE(384, 190, 64)}, "TQ_UNSUPPORTED"), ({"v": OFF}, "TQ_UNSUPPORTED"),
    ({"counts": OFF}, "TQ_UNSUPPORTED"), ({"tokens": 0}, "TQ_OK"), ({"batch": 0}, "TQ_OK"),
], ids=str)
def test_cache_store_refuses(lib, changed, code):
    assert store(lib, **changed) == getattr(lib, code), lib.last_error()


def copy(lib, sources, targets, pages=10, **changed):
    one = dict(base=1 << 20, layers=1, layer_stride=0, page_stride=64, page_bytes=64)
    one.update(changed)
    tensors = (lib.tq_paged_tensor * 1)(lib.tq_paged_tensor(**one))
    return lib.lib.tq_copy_pages_launch(tensors, 1, pages, (ctypes.c_int64 * len(sources))(*sources), (ctypes.c_int64 * len(targets))(*targets), len(sources), 0, None)


@pytest.mark.parametrize("sources, targets, changed", [
    ([0], [10], {}), ([10], [0], {}), ([-1], [0], {}), ([0], [-1], {}), ([0, 1], [2, 2], {}), ([0, 1], [1, 2], {}), ([3], [3], {}), ([0, 1, 2], [5, 6, 0], {}),
    ([0], [1], {"page_stride": 60}), ([0], [1], {"layers": -1}), ([0], [1], {"base": None}),
], ids=str)
def test_copy_pages_refuses(lib, sources, targets, changed):
    assert copy(lib, sources, targets, **changed) == lib.TQ_INVALID_ARGUMENT, lib.last_error()


@pytest.mark.parametrize("changed", [{"layers": 65536}, {"page_bytes": 1 << 34}, {"layers": 65535, "page_bytes": 1 << 33}, {"layers": 4096, "page_bytes": 1 << 33}], ids=str)
def test_copy_pages_beyond_a_launch(lib, changed):
    """(A tensor's layers may lie anywhere, on one another too, so these are not beyond what memory can hold.)"""
    assert copy(lib, [0], [1], **{**changed, "page_stride": 1 << 35}) == lib.TQ_UNSUPPORTED, lib.last_error()


def test_copy_pages_with_nothing_to_do(lib):
    assert copy(lib, [], []) == lib.TQ_OK
    assert lib.lib.tq_copy_pages_launch(None, 0, 4, None, None, 3, 0, None) == lib.TQ_OK


def test_python_refuses_before_the_library():
    from tessiq_b200 import ops
    from tessiq_b200._lib import Declined

    q, k = torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 9, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.window_attention(q, k, k, 4)
    with pytest.raises(ValueError, match="at least one key"):
        ops.window_attention(q, k, k, 0)
    with pytest.raises(ValueError, match="first keys"):
        ops.window_attention(q, k, k, 4, -1)
    with pytest.raises(ValueError, match="do not agree"):
        ops.window_attention(q, k, k[:, :, :5])
    with pytest.raises(ValueError, match="do not agree"):
        ops.window_attention(q[:, :3], k, k)
    with pytest.raises(Declined, match="element type"):
        ops.window_attention(q, k.half(), k)
    with pytest.raises(Declined, match="batch, heads"):
        ops.window_attention(q[0], k, k)
    pages = torch.zeros(7, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales, table, lengths = torch.ones(7, 2), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    good = (pages, pages, scales, scales, table)
    with pytest.raises(ValueError, match="CUDA"):
        ops.cache_attention(q, *good, lengths)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        ops.cache_attention(q, pages.view(torch.uint8), pages, scales, scales, table, lengths)
    with pytest.raises(ValueError, match="scales"):
        ops.cache_attention(q, pages, pages, scales[:6], scales, table, lengths)
    with pytest.raises(ValueError, match="scales"):
        ops.cache_attention(q, pages, pages, scales, scales.double(), table, lengths)
    with pytest.raises(ValueError, match="table"):
        ops.cache_attention(q, pages, pages, scales, scales, table.long(), lengths)
    with pytest.raises(ValueError, match="table"):
        ops.cache_attention(q, pages, pages, scales, scales, table[:1], lengths)
    with pytest.raises(ValueError, match="lengths"):
        ops.cache_attention(q, *good, lengths.long())
    with pytest.raises(ValueError, match="holds"):
        ops.cache_attention(q[..., :32], *good, lengths)
    with pytest.raises(ValueError, match="packed"):
        ops.cache_attention(q, pages.transpose(0, 0)[::2], pages[::2], scales[:4], scales[:4], table, lengths)
    with pytest.raises(ValueError, match="evenly"):
        ops.cache_attention(q[:, :3], *good, lengths)
    with pytest.raises(ValueError, match="differ"):
        ops.cache_store(k, k[:, :, :4], *good, lengths)
    with pytest.raises(ValueError, match="counts"):
        ops.cache_store(k, k, *good, lengths, lengths[:1])
    with pytest.raises(ValueError, match="same number of pages"):
        ops.copy_pages([pages.view(torch.uint8), scales[:3]], [0], [1])
    with pytest.raises(ValueError, match="sources"):
        ops.copy_pages([scales], [0, 1], [2])
    with pytest.raises(Declined, match="contiguous"):
        ops.copy_pages([torch.zeros(7, 4, 4).transpose(1, 2)], [0], [1])
    with pytest.raises(Declined, match="axis"):
        ops.copy_pages([scales], [0], [1], page_axis=2)
    ops.copy_pages([], [0], [1])


@pytest.mark.parametrize("page", [7, -1, 1 << 64, (1 << 64) + 2, -(1 << 63) - 1])
def test_pages_are_numbers_of_pages(page):
    from tessiq_b200 import ops

    scales = torch.ones(7, 2)
    for pair in (([page], [1]), ([1], [page]), ([0, page], [2, 3])):
        with pytest.raises(ValueError, match=f"no page {page}"):
            ops.copy_pages([scales], *pair)
    with pytest.raises(TypeError):
        ops.copy_pages([scales], [0.5], [1])


def test_windows_and_sinks_of_any_length():
    from tessiq_b200 import ops

    for n in (1 << 31, (1 << 63) - 1, 1 << 63, (1 << 64) + 3, 10**30):
        window, sinks = ops._window(n, n)
        assert 1 << 30 <= window < 1 << 63 and 1 << 30 <= sinks < 1 << 63
    assert ops._window(None, 0) == (0, 0) and ops._window(7, 3) == (7, 3)


# ---- the books -----------------------------------------------------------------------------------


def test_pages_are_handed_out_lowest_first_and_taken_back():
    from tessiq_b200.cache import Pages

    books = Pages(6, 16)
    a, b = books.start(), books.start()
    assert books.extend([a, b], [17, 16]) == ([], [])
    assert books.pages_of(a) == [0, 1] and books.pages_of(b) == [2] and books.free_pages == 3
    books.extend([b], [0])
    assert books.pages_of(b) == [2]
    books.extend([b], [1])
    assert books.pages_of(b) == [2, 3] and books.length(b) == 17
    books.free(a)
    assert books.free_pages == 4 and books.sequences == [b]
    with pytest.raises(KeyError):
        books.length(a)
    c = books.start()
    books.extend([c], [3])
    assert books.pages_of(c) == [0]


def test_a_call_that_cannot_be_met_changes_nothing():
    from tessiq_b200.cache import Pages

    books = Pages(4, 16)
    a = books.start()
    books.extend([a], [20])
    b = books.fork(a)
    with pytest.raises(MemoryError):
        books.extend([a, b], [13, 17])      # a page of its own for a, one more for each
    assert books.free_pages == 2 and books.length(a) == books.length(b) == 20 and books.pages_of(a) == books.pages_of(b) == [0, 1]
    with pytest.raises(ValueError):
        books.extend([a, a], [1, 1])
    with pytest.raises(ValueError):
        books.extend([a], [-1])
    with pytest.raises(ValueError):
        books.truncate(a, 21)
    assert books.extend([a, b], [1, 1]) == ([1], [2])      # the second one has the shared page to itself by then
    assert books.pages_of(a) == [0, 2] and books.pages_of(b) == [0, 1] and books.references[:3] == [2, 1, 1]


def test_the_books_against_copies_of_every_sequence():
    """Random calls: each sequence's tokens, followed through writes, page copies and moves, stay its own."""
    import random

    from tessiq_b200.cache import Pages

    rng, page = random.Random(3), 4
    books, memory, tokens, serial = Pages(30, page), {}, {}, 0
    for _ in range(3000):
        kind = rng.choice(["start", "fork", "extend", "extend", "extend", "truncate", "free", "compact"])
        known = list(tokens)
        if kind == "start" and len(known) < 8:
            tokens[books.start()] = []
        elif kind == "fork" and known and len(known) < 8:
            old = rng.choice(known)
            tokens[books.fork(old)] = list(tokens[old])
        elif kind == "extend" and known:
            some = rng.sample(known, rng.randint(1, len(known)))
            counts = [rng.randint(0, 9) for _ in some]
            try:
                sources, targets = books.extend(some, counts)
            except MemoryError:
                continue
            assert not set(sources) & set(targets) and len(set(targets)) == len(targets)
            for s, t in zip(sources, targets):
                memory.update({(t, i): memory.get((s, i)) for i in range(page)})
            for sequence, count in zip(some, counts):
                for _ in range(count):
                    at, serial = len(tokens[sequence]), serial + 1
                    where = books.pages_of(sequence)[at // page]
                    assert books.references[where] == 1
                    memory[where, at % page] = serial
                    tokens[sequence].append(serial)
        elif kind == "truncate" and known:
            sequence = rng.choice(known)
            length = rng.randint(0, len(tokens[sequence]))
            books.truncate(sequence, length)
            del tokens[sequence][length:]
        elif kind == "free" and known:
            sequence = rng.choice(known)
            books.free(sequence)
            del tokens[sequence]
        elif kind == "compact":
            sources, targets = books.compact()
            assert not set(sources) & set(targets)
            for s, t in zip(sources, targets):
                memory.update({(t, i): memory.get((s, i)) for i in range(page)})
            used = len(books.references) - books.free_pages
            assert all(books.references[:used]) and not any(books.references[used:])
        for sequence, held in tokens.items():
            pages = books.pages_of(sequence)
            assert books.length(sequence) == len(held) and len(pages) == -(-len(held) // page)
            assert [memory[pages[i // page], i % page] for i in range(len(held))] == held
        counted = [0] * len(books.references)
        for sequence in tokens:
            for where in books.pages_of(sequence):
                counted[where] += 1
        assert counted == books.references and books.free_pages == counted.count(0)


def test_a_step_names_pages_starts_and_lengths():
    from tessiq_b200.cache import PagedCache

    cache = PagedCache(2, 3, 32, pages=9, page_tokens=16, device="cpu")
    a, b = cache.start(), cache.start()
    step = cache.extend([a, b], [17, 5])
    assert step.table.tolist() == [[0, 1], [2, 0]] and step.starts.tolist() == [0, 0] and step.counts.tolist() == [17, 5] and step.lengths.tolist() == [17, 5]
    step = cache.extend([b, a], 2)
    assert step.starts.tolist() == [5, 17] and step.lengths.tolist() == [7, 19] and step.tokens == 2
    assert step.table.dtype == torch.int32 and step.table.tolist() == [[2, 0], [0, 1]]
    assert cache.extend([], 1).table.shape == (0, 0)
    with pytest.raises(ValueError, match="nobody wrote"):
        cache.store(step, 0, torch.zeros(2, 3, 1, 32).half(), torch.zeros(2, 3, 1, 32).half())
    for bad in (dict(page_tokens=48), dict(width=24), dict(layers=0), dict(pages=0)):
        with pytest.raises(ValueError):
            PagedCache(**{**dict(layers=1, kv_heads=2, width=64, pages=4, device="cpu"), **bad})


def test_a_step_that_has_ended_is_refused(monkeypatch):
    """Each way in which pages or tokens that a step names stop being its sequences' own; steps of other sequences go on."""
    from tessiq_b200 import cache as module

    launched = []
    monkeypatch.setattr(module.ops, "copy_pages", lambda *a, **k: launched.append("copy"))
    monkeypatch.setattr(module.ops, "cache_store", lambda *a: launched.append("store"))
    monkeypatch.setattr(module.ops, "cache_attention", lambda *a: launched.append("attend"))
    k = torch.zeros(1, 1, 9, 16).half()

    def made():
        cache = module.PagedCache(1, 1, 16, pages=20, page_tokens=16, device="cpu")
        a, other = cache.start(), cache.start()
        return cache, a, cache.extend([a], 9), cache.extend([other], 2)

    def ended(cache, step, other, stores=True, reads=True):
        for refused, call in ((stores, lambda s: cache.store(s, 0, k, k)), (reads, lambda s: cache.attention(s, 0, k))):
            launched.clear()
            if refused:
                with pytest.raises(ValueError, match="sequence"):
                    call(step)
                assert not launched
            else:
                call(step)
            call(other)
            assert len(launched) == 2 - refused

    cache, a, step, other = made()
    ended(cache, step, other, False, False)
    b = cache.fork(a)                        # writing what both of them have is what both of them see
    ended(cache, step, other, False, False)
    cache.truncate(a, 9)                     # nothing forgotten
    ended(cache, step, other, False, False)
    cache.extend([b], 0)
    ended(cache, step, other, False, False)
    cache.extend([b], 1)                     # b has a copy from before what is stored now
    ended(cache, step, other, True, False)
    later = cache.extend([a], 1)             # (alone on its page again)
    ended(cache, step, other, True, False)
    ended(cache, later, other, False, False)
    for end in ("truncate", "free", "exchange", "compact"):
        cache, a, step, other = made()
        if end == "truncate":
            cache.truncate(a, 8)
        elif end == "free":
            cache.free(a)
        elif end == "exchange":              # a moves to a copy, the page it wrote is its fork's
            cache.fork(a)
            later = cache.extend([a], 1)
            ended(cache, later, other, False, False)
        else:
            low = cache.start()
            third = cache.extend([low], 20)
            cache.free(a)
            a, step, other = low, third, other
            assert cache.compact() == 1
        ended(cache, step, other)


# ---- window attention in ATen, for what the kernels decline ----------------------------------------


def by_rows(q, k, v, window, sinks, scale):
    """The definition, a query and head at a time, in 64 bits, over the keys that it sees and nothing else."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(q.shape[0]):
        for h in range(q.shape[1]):
            for i in range(q.shape[2]):
                at, head = k.shape[2] - q.shape[2] + i, h // (q.shape[1] // k.shape[1])
                seen = [j for j in range(at + 1) if window is None or j > at - window or j < sinks]
                if seen:
                    weights = torch.softmax(k[b, head, seen].double() @ q[b, h, i].double() * scale, 0)
                    out[b, h, i] = (weights[:, None] * v[b, head, seen].double()).sum(0)
    return out


def roundings(q, k, v, scale):
    """How many half steps of the type that is computed in a result may be off, times the largest value: a score's width + 4 roundings of its products' sizes
    count twice in a probability; the exponential, the sums over the keys and the quotient have the rest."""
    q, k, v = (t.double().nan_to_num(0.0, 0.0, 0.0).abs() for t in (q, k, v))
    if k.shape[2] == 0:
        return 0.0
    sizes = (q @ k.repeat_interleave(q.shape[1] // k.shape[1], 1).transpose(-1, -2)).max().item() * scale
    return (2 * (q.shape[3] + 4) * sizes + 2 * k.shape[2] + 20) * v.max().item()


@pytest.mark.parametrize("window, sinks", [(None, 0), (3, 0), (4, 2), (1, 1)], ids=str)
@pytest.mark.parametrize("queries, keys", [(6, 6), (3, 11), (9, 4), (2, 0)], ids=str)
def test_the_aten_form_in_64_bits(window, sinks, queries, keys):
    from tessiq_b200.ops import _window_attention_by_aten

    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, n, t, 7, generator=g, dtype=torch.float64) for n, t in ((4, queries), (2, keys), (2, keys)))
    got = _window_attention_by_aten(q, k, v, window, sinks, None)
    assert got.dtype == torch.float64 and got.is_contiguous()
    torch.testing.assert_close(got, by_rows(q, k, v, window, sinks, 7**-0.5), rtol=0, atol=2.0**-53 * roundings(q, k, v, 7**-0.5))


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16], ids=str)
def test_the_aten_form_lets_nobody_see_what_is_hidden(dtype):
    """Key 7 is the last query's alone, key 2 lies between the sinks and the first query's window: NaN and infinities there, and in a value that two queries see."""
    from tessiq_b200.ops import _window_attention_by_aten

    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 2, t, 4, generator=g).to(dtype) for t in (3, 8, 8))
    k[0, 0, 2], v[0, 0, 2] = float("nan"), float("nan")
    v[0, 0, 7, 1], v[0, 0, 7, 2], v[0, 0, 7, 3], v[0, 1, 6, 0] = float("nan"), float("inf"), float("-inf"), float("inf")
    k[0, 1, 7] = float("inf")                    # scores of infinity, or NaN: the last query's row of head 1
    got, exact = _window_attention_by_aten(q, k, v, 3, 2, 0.5).double(), by_rows(q, k, v, 3, 2, 0.5)
    assert got[:, 0, :2].isfinite().all() and got[0, 1, 0].isfinite().all()
    assert torch.equal(got.isnan(), exact.isnan()) and torch.equal(got.isinf(), exact.isinf())
    assert torch.equal(got[got.isinf()], exact[exact.isinf()])
    fine = exact.isfinite()
    inside = torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).eps / 2
    assert ((got - exact).abs()[fine] <= torch.finfo(dtype).eps / 2 * exact.abs()[fine] + inside * roundings(q, k, v, 0.5)).all()


def test_the_aten_form_keeps_scores_in_32_bits():
    """f16 operands whose scores pass 65504 before they are scaled, and lie a step of f16 apart after it."""
    from tessiq_b200.ops import _window_attention_by_aten

    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, 1, t, 256, generator=g).mul(size).half() for t, size in ((2, 60.0), (5, 60.0), (5, 1.0)))
    scale = 2.0**-12
    got, exact = _window_attention_by_aten(q, k, v, None, 0, scale).double(), by_rows(q, k, v, None, 0, scale)
    assert ((got - exact).abs() <= 2.0**-11 * exact.abs() + 2.0**-24 * roundings(q, k, v, scale)).all()
