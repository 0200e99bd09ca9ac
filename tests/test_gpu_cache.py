"""Attention with a window and sinks, the paged cache in 8 bits, its writer and the copies of its pages, against plain 64-bit forms.

How far a result may be off (`bound`): half a step of its type, relative (bf16 2^-8, f16 2^-11); half a step of the probabilities' rounding
relative to sum_j p_j |v_j| (f16 2^-11, below its normal range 2^-25 a key absolutely; bf16 2^-8 in the tensor-core tiles, the
coarser of the forms); an error d of a score is a relative error of 2 d in the probabilities, and f32 sums of `width` products give
d = (width + 4) 2^-24 sum |q| |k| scale, ex2.approx another 2^-21; f32 sums over n keys (n + 8) 2^-24. Codes, scales and copies are exact."""

import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def tq():
    if not torch.cuda.is_available():
        pytest.fail("the gpu tests need a CUDA device")
    from tessiq_b200 import ops

    return ops


def status(device=0):
    from tessiq_b200 import _lib

    code = ctypes.c_int32(-1)
    _lib.check(_lib.lib.tq_status_poll(device, None, ctypes.byref(code)))
    return code.value


def reference(q, k, v, lengths, window, sinks, scale):
    """(result, bound) in f64 on the CPU: q [batch, heads, queries, width], k and v [batch, kv_heads, keys, width]; only visible keys are touched."""
    q, k, v = (t.detach().cpu() for t in (q, k, v))
    dtype = q.dtype
    u_out = torch.finfo(dtype).eps / 2
    batch, heads, queries, width = q.shape
    group = heads // k.shape[1]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape, 1e-30, dtype=torch.float64)
    for b in range(batch):
        for i in range(queries):
            p = lengths[b] - queries + i
            if p < 0:
                continue
            j = torch.arange(p + 1)
            j = j[(j > p - window) | (j < sinks)] if window is not None else j
            for h in range(heads):
                qq, kk, vv = q[b, h, i].double(), k[b, h // group, j].double(), v[b, h // group, j].double()
                weight = torch.softmax(kk @ qq * scale, 0)
                out[b, h, i] = weight @ vv
                spread = weight @ vv.abs()
                d = (width + 4) * 2.0**-24 * (kk.abs() @ qq.abs()).max().item() * scale + 2.0**-21
                bound[b, h, i] += u_out * out[b, h, i].abs() + (u_out + 2 * d + (len(j) + 8) * 2.0**-24) * spread
                bound[b, h, i] += 2.0**-25 * vv.abs().sum(0)
    return out, bound


def held(got, expected):
    exact, bound = expected
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), exact.isnan())
    error = (got - exact).abs()
    over = (error / bound).nan_to_num(0.0).max().item()
    assert over <= 1.0, f"{over:.2f} times what roundings explain"


def drawn(shape, dtype, seed, spread=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype).cuda()


def by_token(shape, dtype, seed):
    """[batch, heads, tokens, width] as a projection's [batch, tokens, heads, width] is seen."""
    batch, heads, tokens, width = shape
    return drawn((batch, tokens, heads, width), dtype, seed).transpose(1, 2)


# ---- dense keys ----------------------------------------------------------------------------------

WINDOWS = [  # batch, heads, kv_heads, queries, keys, width, window, sinks
    (1, 1, 1, 1, 1, 64, None, 0), (1, 1, 1, 1, 1, 64, 1, 0), (2, 3, 3, 1, 77, 64, 10, 4), (1, 4, 2, 3, 130, 128, 40, 0), (1, 8, 1, 1, 300, 64, 64, 1),
    (2, 16, 2, 2, 333, 128, 100, 33), (1, 2, 2, 5, 3, 64, None, 0), (1, 2, 1, 9, 4, 64, 2, 1), (1, 2, 2, 100, 100, 64, 7, 3), (1, 6, 2, 130, 130, 96, 64, 64),
    (2, 2, 1, 129, 200, 128, 128, 5), (1, 1, 1, 257, 257, 64, 1, 0), (1, 2, 2, 300, 300, 64, 1000, 2), (1, 1, 1, 70, 600, 40, 200, 500), (1, 2, 1, 260, 90, 64, 30, 10),
    (1, 3, 3, 17, 1100, 8, 129, 4), (1, 12, 12, 4, 2049, 64, 2048, 4), (1, 2, 2, 384, 384, 128, 65, 1),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", WINDOWS, ids=lambda c: "-".join(map(str, c)))
def test_window_attention(tq, case, dtype):
    batch, heads, kv_heads, queries, keys, width, window, sinks = case
    q, k, v = by_token((batch, heads, queries, width), dtype, 1), by_token((batch, kv_heads, keys, width), dtype, 2), by_token((batch, kv_heads, keys, width), dtype, 3)
    got = tq.window_attention(q, k, v, window, sinks)
    assert got.shape == q.shape and got.dtype == dtype
    held(got, reference(q, k, v, [keys] * batch, window, sinks, 1 / math.sqrt(width)))
    assert status() == 0


def form(*extents):
    from tessiq_b200 import _lib

    kind, keys = ctypes.c_int32(), ctypes.c_int32()
    _lib.check(_lib.lib.tq_window_attention_form(*extents, 0, ctypes.byref(kind), ctypes.byref(keys)))
    return keys.value


FORMS = [  # batch, heads, kv_heads, queries, keys, width, window, sinks: every form, at its edges
    ((1, 2, 2, 20, 3000, 64, 2500, 4), 0), ((1, 4, 1, 40, 1500, 128, 0, 0), 0), ((2, 12, 12, 200, 260, 64, 0, 0), 128), ((1, 8, 8, 300, 2000, 128, 0, 8), 128),
    ((40, 12, 6, 130, 130, 64, 50, 2), 64), ((12, 16, 8, 150, 200, 96, 90, 70), 64),
]


@pytest.mark.parametrize("case, keys", FORMS, ids=str)
def test_every_form_of_window_attention(tq, case, keys):
    batch, heads, kv_heads, queries, k_tokens, width, window, sinks = case
    assert form(*case) == keys
    q, k, v = by_token((batch, heads, queries, width), torch.bfloat16, 1), by_token((batch, kv_heads, k_tokens, width), torch.bfloat16, 2), by_token((batch, kv_heads, k_tokens, width), torch.bfloat16, 3)
    got = tq.window_attention(q, k, v, window or None, sinks)
    some = [0, batch - 1] if batch > 1 else [0]
    held(got[some, :2], reference(q[some, :2], k[some, : max(1, 2 * kv_heads // heads)], v[some, : max(1, 2 * kv_heads // heads)], [k_tokens] * len(some), window or None, sinks, 1 / math.sqrt(width)))
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case, keys", FORMS[:1] + FORMS[2:], ids=str)
def test_a_result_at_any_alignment(tq, case, keys, dtype):
    """Through the C interface a result may begin at any element and have any strides; what lies between its rows stays."""
    from tessiq_b200 import _lib

    batch, heads, kv_heads, queries, k_tokens, width, window, sinks = case
    q, k, v = by_token((batch, heads, queries, width), dtype, 1), by_token((batch, kv_heads, k_tokens, width), dtype, 2), by_token((batch, kv_heads, k_tokens, width), dtype, 3)
    expected = tq.window_attention(q, k, v, window or None, sinks)
    buffer = torch.full((1 + batch * heads * queries * (width + 3),), 7.0, dtype=dtype, device="cuda")
    out = buffer[1:].view(batch, heads, queries, width + 3)
    three = [(ctypes.c_int64 * 3)(*t.stride()[:3]) for t in (q, k, v, out)]
    scratch = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    need = ctypes.c_size_t()
    _lib.check(_lib.lib.tq_window_attention_workspace_bytes(batch, heads, kv_heads, queries, k_tokens, width, window, sinks, 0, ctypes.byref(need)))
    assert need.value <= scratch.numel()
    _lib.check(_lib.lib.tq_window_attention_launch(_lib.BF16 if dtype == torch.bfloat16 else _lib.F16, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), batch, heads,
                                                   kv_heads, queries, k_tokens, width, *three, 1 / math.sqrt(width), window, sinks, scratch.data_ptr(), need.value, 0,
                                                   torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[..., :width], expected)
    assert (out[..., width:] == 7).all() and buffer[0] == 7
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", [(1, 2, 1, 1, 40000, 64, 0, 0), (1, 4, 2, 2, 9000, 128, 8000, 4), (2, 2, 1, 7, 20000, 80, 0, 0)], ids=lambda c: "-".join(map(str, c)))
def test_dense_keys_of_few_heads_are_joined_by_warps_and_then_by_ctas(tq, case, dtype):
    batch, heads, kv_heads, queries, keys, width, window, sinks = case
    assert form(*case) == 0
    q, k, v = by_token((batch, heads, queries, width), dtype, 1), by_token((batch, kv_heads, keys, width), dtype, 2), by_token((batch, kv_heads, keys, width), dtype, 3)
    got = tq.window_attention(q, k, v, window or None, sinks)
    held(got, reference(q, k, v, [keys] * batch, window or None, sinks, 1 / math.sqrt(width)))
    for _ in range(20):
        assert torch.equal(tq.window_attention(q, k, v, window or None, sinks), got)
    assert status() == 0


def test_without_a_window_it_is_causal_attention(tq):
    q, k, v = (drawn((2, 4, 200, 64), torch.bfloat16, s) for s in (1, 2, 3))
    expected = reference(q, k, v, [200, 200], None, 0, 0.2)
    held(tq.window_attention(q, k, v, scale=0.2), expected)
    held(tq.attention(q, k, v, 0.2, causal=True), expected)


@pytest.mark.parametrize("token_major", [True, False])
def test_window_attention_writes_either_order(tq, token_major):
    q, k, v = (drawn((2, 4, 5, 64), torch.float16, s) for s in (1, 2, 3))
    got = tq.window_attention(q, k, v, 3, 1, token_major=token_major)
    assert got.is_contiguous() != token_major
    held(got, reference(q, k, v, [5, 5], 3, 1, 0.125))


def test_window_attention_over_no_keys_and_no_queries(tq):
    q = drawn((2, 4, 3, 64), torch.bfloat16, 1)
    none = torch.empty(2, 2, 0, 64, dtype=torch.bfloat16, device="cuda")
    assert tq.window_attention(q, none, none, 4, 1).count_nonzero().item() == 0
    assert tq.window_attention(q[:, :, :0], none, none).shape == (2, 4, 0, 64)
    assert tq.window_attention(q[:0], none[:0], none[:0]).shape == (0, 4, 3, 64)


@pytest.mark.parametrize("batch, queries", [(1, 1), (1, 3), (1, 70), (40, 70), (40, 200)], ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_no_query_sees_does_not_reach_a_result(tq, batch, queries, bad):
    """Keys 20 to 39 lie between the sinks and the first query's window, and the last keys are the last queries' own. The large batches run on tiles."""
    keys, window = queries + 100, 50
    assert (form(batch, 4, 2, queries, keys, 64, window, 20) > 0) == (batch > 1)
    q, k, v = drawn((batch, 4, queries, 64), torch.bfloat16, 1), drawn((batch, 2, keys, 64), torch.bfloat16, 2), drawn((batch, 2, keys, 64), torch.bfloat16, 3)
    k[:, :, 20:40], v[:, :, 20:40] = bad, bad
    expected = reference(q[-1:], k[-1:], v[-1:], [keys], window, 20, 0.125)
    assert not expected[0].isnan().any()
    got = tq.window_attention(q, k, v, window, 20)
    held(got[-1:], expected)
    assert got.isfinite().all()


@pytest.mark.parametrize("batch, queries", [(1, 4), (1, 150), (40, 150)], ids=str)
def test_a_value_that_is_not_a_number_reaches_the_queries_that_see_it(tq, batch, queries):
    """Key `at` is seen from the query at `at` for a window's length, and by those alone; sinks by all of them. The large batch runs on tiles."""
    keys, window, at = queries + 30, 20, 29 + queries // 2
    assert (form(batch, 2, 2, queries, keys, 64, window, 3) > 0) == (batch > 1)
    q, k, v = (drawn((batch, 2, n, 64), torch.float16, s) for n, s in ((queries, 1), (keys, 2), (keys, 3)))
    v[0, 1, at, 5] = math.nan
    v[0, 0, keys - 1, 7] = math.inf
    expected = reference(q[:1], k[:1], v[:1], [keys], window, 3, 0.125)
    got = tq.window_attention(q, k, v, window, 3)
    assert got[1:].isfinite().all()
    got = got[:1].cpu().double()
    assert expected[0].isnan().any() and torch.equal(got.isnan(), expected[0].isnan()) and torch.equal(got.isinf(), expected[0].isinf())
    fine = expected[0].isfinite()
    assert ((got - expected[0]).abs()[fine] <= expected[1][fine]).all()


TILES = [(40, 12, 6, 150, 180, 64, 70, 3, 64), (1, 12, 12, 300, 1500, 64, 0, 0, 128), (12, 16, 8, 150, 200, 96, 90, 70, 64), (1, 8, 8, 300, 2000, 128, 0, 8, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", TILES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("bad", ["a sink", "a channel", "signs", "scattered", "keys", "queries", "everything"])
def test_what_is_no_number_on_the_tiles(tq, case, dtype, bad):
    """Seen by all rows, by some, or by none of a tile: each row has what its own keys make of it."""
    *extents, tiles = case
    batch, heads, kv_heads, queries, keys, width, window, sinks = extents
    assert form(*extents) == tiles
    q, k, v = (by_token((1, n, t, width), dtype, s) for n, t, s in ((heads, queries, 1), (kv_heads, keys, 2), (kv_heads, keys, 3)))
    at = torch.randint(0, keys, (9,), generator=torch.Generator().manual_seed(4)).tolist()
    if bad == "a sink":
        v[:, :, 0, 5], v[:, :, 1, 6] = math.nan, math.inf
    elif bad == "a channel":
        v[:, :, :, 7] = math.inf
    elif bad == "signs":
        v[:, :, keys // 2, 2], v[:, :, keys // 2 + 3, 2], v[:, :, keys // 2 + 9, 3] = math.inf, -math.inf, -math.inf
    elif bad == "scattered":
        for n, j in enumerate(at):
            v[:, :, j, (7 * n) % width] = (math.nan, math.inf, -math.inf)[n % 3]
    elif bad == "keys":
        k[:, :, at, 1] = math.nan
    elif bad == "queries":
        q[:, :, ::7] = math.nan
    else:
        q, k, v = (torch.full_like(t, math.nan) for t in (q, k, v))
    got = tq.window_attention(*(t.expand(batch, -1, -1, -1).clone(memory_format=torch.preserve_format) if batch > 1 else t for t in (q, k, v)), window or None, sinks)
    rows = sorted({0, 1, 30, 31, 32, 33, 62, 63, 127, 128, 129, queries - 1, *(j - keys + queries + d for j in at for d in (-1, 0, 1) if 0 <= j - keys + queries + d < queries)})
    some = max(1, 2 * kv_heads // heads)
    exact, bound = (torch.cat(parts, 2) for parts in zip(*(reference(q[:, :2, i : i + 1], k[:, :some], v[:, :some], [keys - queries + i + 1], window or None, sinks, width**-0.5)
                                                           for i in rows)))
    got = got[-1:, :2, rows].cpu().double()
    assert torch.equal(got.isnan(), exact.isnan()) and torch.equal(got[got.isinf()], exact[exact.isinf()]) and torch.equal(got.isinf(), exact.isinf())
    fine = exact.isfinite()
    assert ((got - exact).abs()[fine] <= bound[fine]).all()
    assert status() == 0


@pytest.mark.parametrize("bad", ["everything", "a key", "a value"])
def test_a_nan_that_everybody_sees_costs_no_second_reading(tq, bad):
    """(It was 800 times the launch; a reading of the values by each warp is a few times it.)"""
    q, k, v = (drawn((2, 12, 4096, 64), torch.bfloat16, s) for s in (1, 2, 3))

    def time_of(q, k, v):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        for n in range(4):
            if n == 1:
                start.record()
            got = tq.window_attention(q, k, v, 1024, 4)
        end.record()
        torch.cuda.synchronize()
        return start.elapsed_time(end), got

    fine, _ = time_of(q, k, v)
    if bad == "everything":
        q, k, v = (torch.full_like(t, math.nan) for t in (q, k, v))
    elif bad == "a key":
        k[:, :, 0] = math.nan
    else:
        v[:, :, 0] = math.nan
    slow, got = time_of(q, k, v)
    assert got.isnan().all() and slow < 50 * fine


def test_scores_that_are_all_minus_infinity_are_not_a_number(tq):
    """As softmax over them is; a query that sees nothing is zeros instead."""
    q, k, v = (drawn((1, 1, 2, 64), torch.bfloat16, s).abs() + 0.5 for s in (1, 2, 3))
    k[:, :, 0] = -math.inf
    got = tq.window_attention(q, k, v, 1, 0)
    assert got[0, 0, 0].isnan().all() and got[0, 0, 1].isfinite().all()
    got = tq.window_attention(q, k[:, :, :1], v[:, :, :1])
    assert got[0, 0, 0].count_nonzero().item() == 0 and got[0, 0, 1].isnan().all()


# ---- the cache -----------------------------------------------------------------------------------


class Cache:
    """A pool with a table of scattered pages; what no sequence owns is NaN."""

    def __init__(self, batch, kv_heads, width, page, blocks, seed=0):
        self.page, pages = page, batch * blocks + 2
        g = torch.Generator().manual_seed(seed)
        shape = (pages, kv_heads, page, width)
        self.codes = [torch.full(shape, 0x7F, dtype=torch.uint8).view(E4M3).cuda() for _ in range(2)]
        self.scales = [torch.full(shape[:2], math.nan).cuda() for _ in range(2)]
        order = torch.randperm(pages, generator=g)
        self.table = order[: batch * blocks].to(torch.int32).reshape(batch, blocks).cuda()
        self.generator = g

    @property
    def tensors(self):
        return (*self.codes, *self.scales)

    def fill(self, lengths):
        """Random tokens at each sequence's first positions; the rest stays NaN."""
        for codes, scales in zip(self.codes, self.scales):
            for b, length in enumerate(lengths):
                for n in range(-(-length // self.page)):
                    page, tokens = int(self.table[b, n]), min(self.page, length - n * self.page)
                    part = (torch.randn(codes.shape[1], tokens, codes.shape[3], generator=self.generator) * 60).clamp(-448, 448).to(E4M3)
                    codes.view(torch.uint8)[page, :, :tokens] = part.view(torch.uint8).cuda()
                    scales[page] = torch.exp2(torch.randn(codes.shape[1], generator=self.generator) * 2 - 6).cuda()
        return self

    def decoded(self, which):
        """[batch, kv_heads, tokens, width] in f32 on the CPU."""
        pages = self.table.long().cpu()
        codes, scales = self.codes[which].view(torch.uint8).cpu()[pages].view(E4M3).float(), self.scales[which].cpu()[pages]
        values = codes * scales[..., None, None]
        return values.permute(0, 2, 1, 3, 4).flatten(2, 3)


CACHES = [  # heads, kv_heads, queries, width, page, window, sinks, lengths
    (1, 1, 1, 64, 16, None, 0, [1]), (2, 2, 1, 64, 16, None, 0, [0, 1, 15, 16, 17]), (12, 12, 1, 64, 64, None, 0, [100, 3, 64, 65]), (8, 1, 1, 128, 32, None, 0, [31, 33, 257]),
    (16, 2, 1, 128, 64, 100, 4, [1, 99, 104, 105, 640]), (6, 3, 4, 64, 16, 20, 5, [0, 1, 3, 4, 5, 200]), (16, 2, 4, 128, 64, None, 0, [2, 300]), (4, 4, 3, 16, 128, 30, 0, [500, 7]),
    (64, 8, 1, 80, 64, 64, 64, [63, 700]), (3, 1, 11, 96, 32, 33, 1, [5, 90]), (2, 1, 40, 32, 16, 17, 2, [39, 41, 130]), (5, 1, 2, 112, 1024, None, 0, [1500]), (14, 2, 1, 64, 32, 1, 0, [1, 50]),
    (8, 8, 1, 128, 64, None, 0, [5000, 1]), (32, 8, 2, 128, 16, 3000, 16, [4097]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", CACHES, ids=lambda c: "-".join(map(str, c[:7])) + f"-{len(c[7])}")
def test_cache_attention(tq, case, dtype):
    heads, kv_heads, queries, width, page, window, sinks, lengths = case
    batch = len(lengths)
    cache = Cache(batch, kv_heads, width, page, max(1, -(-max(lengths) // page))).fill(lengths)
    q = by_token((batch, heads, queries, width), dtype, 1)
    got = tq.cache_attention(q, *cache.tensors, cache.table, torch.tensor(lengths, dtype=torch.int32).cuda(), window, sinks)
    # (codes times scales in f64: the keys as they stand)
    expected = reference(q, cache.decoded(0).double(), cache.decoded(1).double(), lengths, window, sinks, 1 / math.sqrt(width))
    held(got, expected)
    assert status() == 0


@pytest.mark.parametrize("case", [(24, 16, 4, 1, 64, 64, None, 0, 2500), (40, 16, 8, 2, 128, 32, 700, 4, 1500), (1, 8, 1, 1, 128, 64, None, 0, 20000),
                                  (2, 6, 2, 3, 80, 16, 9000, 40, 12000), (300, 2, 1, 1, 64, 16, None, 0, 1600)], ids=lambda c: "-".join(map(str, c)))
def test_chunks_dealt_out_over_the_gpu(tq, case):
    """Sequences of all lengths in one batch, some empty: every form of the split, checked at some of them."""
    batch, heads, kv_heads, queries, width, page, window, sinks, longest = case
    lengths = [longest * (b * 7 % batch + 1) // batch if b % 5 else b % 3 for b in range(batch)]
    lengths[-1] = longest
    blocks = -(-longest // page)
    g = torch.Generator(device="cuda").manual_seed(1)
    pages = batch * blocks
    codes = [(torch.randn(pages, kv_heads, page, width, device="cuda", generator=g) * 60).clamp_(-448, 448).to(E4M3) for _ in range(2)]
    scales = [torch.exp2(torch.randn(pages, kv_heads, device="cuda", generator=g) - 6) for _ in range(2)]
    table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).reshape(batch, blocks)
    q = by_token((batch, heads, queries, width), torch.bfloat16, 1)
    got = tq.cache_attention(q, *codes, *scales, table, torch.tensor(lengths, dtype=torch.int32).cuda(), window, sinks)
    assert got.isfinite().all()
    for b in sorted({0, min(1, batch - 1), batch // 2, batch - 1}):
        at = table[b].long()
        k, v = ((c.view(torch.uint8)[at].view(E4M3).float() * s[at][..., None, None]).permute(1, 0, 2, 3).flatten(1, 2)[None] for c, s in zip(codes, scales))
        held(got[b : b + 1], reference(q[b : b + 1], k.double(), v.double(), [lengths[b]], window, sinks, width**-0.5))
    assert status() == 0


@pytest.mark.parametrize("case", [(batch, heads, kv_heads, queries, width, 64, window, 3, 11 * 8192 // width // 2) for batch in (1, 20, 58)
                                  for heads, kv_heads, queries, width, window in [(12, 12, 1, 64, None), (24, 12, 6, 128, 300)]],
                         ids=lambda c: "-".join(map(str, c)))
def test_a_unit_of_two_four_and_eight_warps(tq, case):
    """Eleven steps a key head, of 12, 240 and 696 of them: few units take eight warps each, more of them four, many two."""
    test_chunks_dealt_out_over_the_gpu(tq, case)


@pytest.mark.parametrize("spread", [2.0**-60, 2.0**-20, 2.0**20, 2.0**60])
def test_queries_of_any_size(tq, spread):
    """bf16 queries far outside the range of f16, with scores that stay moderate."""
    cache = Cache(1, 2, 64, 16, 4).fill([50])
    q = drawn((1, 4, 2, 64), torch.bfloat16, 1, spread)
    q[0, 1, 0] = 0.0
    scale = 0.125 / spread
    got = tq.cache_attention(q, *cache.tensors, cache.table, torch.tensor([50], dtype=torch.int32).cuda(), scale=scale)
    held(got, reference(q, cache.decoded(0).double(), cache.decoded(1).double(), [50], None, 0, scale))


@pytest.mark.parametrize("spread", [2.0**-102, 2.0**-115, 2.0**-125, 2.0**90, 2.0**125])
def test_queries_at_the_ends_of_bf16(tq, spread):
    """The largest element under 2^-100, or near the largest number; 2^-133 is the smallest."""
    test_queries_of_any_size(tq, spread)


def behind_a_strong_key(q, k, v, keys, scale):
    """`reference` without what f16 loses below its normal range: weights are kept 2^7 times as large, so half a step there is 2^-32 of the largest."""
    exact, bound = reference(q, k, v, [keys], None, 0, scale)
    group = q.shape[1] // k.shape[1]
    return exact, bound - (2.0**-25 - 2.0**-32) * v.double().cpu().abs().sum(2).repeat_interleave(group, 1)[:, :, None]


WEAK = math.log(2.0**24 / 1.4)      # a weight of 1.4 times f16's smallest number


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("keys, width, queries", [(700, 64, 1), (40000, 64, 1), (9000, 128, 3)], ids=str)
def test_many_weak_keys_behind_a_strong_one_in_the_cache(tq, keys, width, queries, dtype):
    cache = Cache(1, 2, width, 64, -(-keys // 64)).fill([keys])
    for codes, scales in zip(cache.codes, cache.scales):
        scales.fill_(1.0)
    first = int(cache.table[0, 0])
    cache.codes[0].view(torch.uint8).zero_()
    cache.codes[0][first, :, 0] = torch.ones(width, device="cuda").to(E4M3)
    cache.codes[1].view(torch.uint8).copy_((torch.rand(cache.codes[1].shape, generator=cache.generator) + 0.5).to(E4M3).view(torch.uint8))
    cache.codes[1].view(torch.uint8)[first, :, 0] = 0
    q = torch.ones(1, 4, queries, width, dtype=dtype, device="cuda")
    got = tq.cache_attention(q, *cache.tensors, cache.table, torch.tensor([keys], dtype=torch.int32).cuda(), scale=WEAK / width)
    held(got, behind_a_strong_key(q, cache.decoded(0)[:, :, :keys], cache.decoded(1)[:, :, :keys], keys, WEAK / width))


@pytest.mark.parametrize("batch, heads, kv_heads, queries, keys, width, tiles", [(1, 2, 1, 1, 700, 64, 0), (1, 2, 1, 2, 20000, 128, 0), (40, 12, 6, 150, 1500, 64, 64),
                                                                                 (1, 8, 8, 300, 2000, 128, 128)], ids=str)
def test_many_weak_keys_behind_a_strong_one_in_f16(tq, batch, heads, kv_heads, queries, keys, width, tiles):
    assert form(batch, heads, kv_heads, queries, keys, width, 0, 0) == tiles
    k = torch.zeros(1, kv_heads, keys, width, dtype=torch.float16, device="cuda")
    k[:, :, 0] = 1.0
    v = drawn((1, kv_heads, keys, width), torch.float32, 1).abs().clamp(0.5, 1.5).half()
    v[:, :, 0] = 0.0
    q = torch.ones(1, heads, queries, width, dtype=torch.float16, device="cuda")
    got = tq.window_attention(*(t.repeat(batch, 1, 1, 1) for t in (q, k, v)), scale=WEAK / width)
    assert torch.equal(got[0], got[-1])
    held(got[:1, :, -2:], behind_a_strong_key(q[:, :, -2:], k, v, keys, WEAK / width))


def test_scales_far_apart_between_pages(tq):
    cache = Cache(1, 1, 64, 16, 6).fill([96])
    cache.scales[1][cache.table[0].long(), 0] = torch.tensor([1e-12, 1e12, 3.0, 1e-30, 1e20, 0.7]).cuda()
    cache.scales[0][cache.table[0].long(), 0] = torch.tensor([0.01, 0.03, 1e-8, 0.02, 0.004, 0.01]).cuda()
    q = drawn((1, 1, 1, 64), torch.bfloat16, 1)
    for window in (None, 16, 40):
        got = tq.cache_attention(q, *cache.tensors, cache.table, torch.tensor([96], dtype=torch.int32).cuda(), window)
        held(got, reference(q, cache.decoded(0).double(), cache.decoded(1).double(), [96], window, 0, 0.125))


@pytest.mark.parametrize("case", [  # batch, kv_heads, queries, width, page (a chunk of keys or more), tokens: a unit a CTA, then shares
    (2, 3, 1, 64, 64, 1500), (2, 3, 1, 128, 32, 900), (1, 2, 3, 128, 128, 1100), (1, 1, 1, 64, 64, 40000), (24, 8, 1, 128, 32, 6000), (6, 2, 4, 64, 256, 9000)],
    ids=lambda c: "-".join(map(str, c)))
def test_every_chunk_takes_the_scales_of_its_own_page(tq, case):
    """Neighbouring pages' scales are 2^3 (keys) and 2^9 (values) apart or more: another page's scale would show at once."""
    batch, kv_heads, queries, width, page, tokens = case
    blocks = -(-tokens // page)
    g = torch.Generator(device="cuda").manual_seed(7)
    pages = batch * blocks
    table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).reshape(batch, blocks)
    nth = torch.empty(pages, device="cuda")
    nth[table.flatten().long()] = (torch.arange(blocks, device="cuda") % 4).float().repeat(batch)
    # keys of one size whatever their page's scale, so that every page has weight; values of one code, so that a page's size is its scale
    signs = torch.randint(0, 2, (pages, kv_heads, page, width), dtype=torch.int8, device="cuda", generator=g).float() * 2 - 1
    codes = [(signs * torch.exp2(3 * nth - 3)[:, None, None, None]).to(E4M3), torch.full_like(signs, 7.0).to(E4M3)]
    scales = [torch.exp2(power * nth)[:, None].expand(pages, kv_heads).contiguous() for power in (-3, -9)]
    q = by_token((batch, 2 * kv_heads, queries, width), torch.bfloat16, 1)
    lengths = torch.full((batch,), tokens, dtype=torch.int32, device="cuda")
    first = tq.cache_attention(q, *codes, *scales, table, lengths)
    for _ in range(20):
        assert torch.equal(tq.cache_attention(q, *codes, *scales, table, lengths), first)
    for b in {0, batch - 1}:
        at = table[b].long()
        k, v = ((c.view(torch.uint8)[at].view(E4M3).float() * s[at][..., None, None]).permute(1, 0, 2, 3).flatten(1, 2)[None, :, :tokens] for c, s in zip(codes, scales))
        held(first[b : b + 1], reference(q[b : b + 1], k.double(), v.double(), [tokens], None, 0, width**-0.5))
    assert status() == 0


def test_pages_that_are_not_there_are_left_out_and_reported(tq):
    from tessiq_b200.kernel import DeviceWaitError, check_status

    assert status() == 0
    lengths = [64, 64]
    cache = Cache(2, 1, 64, 16, 4).fill(lengths)
    q, at = drawn((2, 1, 1, 64), torch.bfloat16, 1), torch.tensor(lengths, dtype=torch.int32).cuda()
    keys, values = cache.decoded(0).double(), cache.decoded(1).double()
    table = cache.table.clone()
    table[1, 3] = 1 << 30
    table[1, 2] = -1
    got = tq.cache_attention(q, *cache.tensors, table, at)
    with pytest.raises(DeviceWaitError, match="outside the pool"):
        check_status()
    held(got[:1], reference(q[:1], keys[:1], values[:1], [64], None, 0, 0.125))
    weights = torch.softmax(keys[1, 0, :32] @ q[1, 0, 0].cpu().double() * 0.125, 0)
    torch.testing.assert_close(got[1, 0, 0].cpu().double(), weights @ values[1, 0, :32], rtol=2e-2, atol=2e-2)
    tq.cache_attention(q, *cache.tensors, cache.table, at + 1)
    with pytest.raises(DeviceWaitError, match="longer than its table"):
        check_status()
    starts = torch.tensor([0, 64], dtype=torch.int32).cuda()
    before = [t.clone().view(torch.uint8) if t.dtype == E4M3 else t.clone() for t in cache.tensors]
    k = drawn((2, 1, 1, 64), torch.bfloat16, 4)
    table[0, 0] = 99
    tq.cache_store(k, k, *cache.tensors, table, starts)
    with pytest.raises(DeviceWaitError):
        check_status()
    for was, now in zip(before, cache.tensors):
        assert torch.equal(was.nan_to_num() if was.dtype == torch.float32 else was, now.view(torch.uint8) if now.dtype == E4M3 else now.nan_to_num())
    assert status() == 0


def kept_reference(q, k, v, kept, scale):
    """`reference` where query i of every sequence sees the keys kept[i] and no others."""
    parts = [reference(q[:, :, i : i + 1], k[:, :, kept[i]], v[:, :, kept[i]], [len(kept[i])] * q.shape[0], None, 0, scale) for i in range(q.shape[2])]
    return torch.cat([r for r, _ in parts], 2), torch.cat([b for _, b in parts], 2)


HOLES = [(page, width, queries, blocks, long) for page, width in ((16, 64), (32, 64), (16, 128), (64, 64)) for queries in (1, 3)
         for blocks, long in ((800 // page, 700), (20000 // page, 19900))]      # a CTA a unit, and shares


@pytest.mark.parametrize("case", HOLES, ids=lambda c: "-".join(map(str, c)))
def test_a_page_that_is_not_there_takes_none_of_its_neighbours_along(tq, case):
    from tessiq_b200.kernel import DeviceWaitError, check_status

    page, width, queries, blocks, long = case
    assert status() == 0
    cache = Cache(1, 2, width, page, blocks).fill([long])
    keys, values = cache.decoded(0).double(), cache.decoded(1).double()
    table, gone = cache.table.clone(), [0, 5, 6, (long - queries) // page - 1]
    table[0, gone] = torch.tensor([-1, 1 << 30, table.numel() + 2, -7], dtype=torch.int32, device="cuda")
    q = by_token((1, 4, queries, width), torch.bfloat16, 1)
    got = tq.cache_attention(q, *cache.tensors, table, torch.tensor([long], dtype=torch.int32).cuda())
    with pytest.raises(DeviceWaitError, match="outside the pool"):
        check_status()
    kept = [[j for j in range(long - queries + i + 1) if j // page not in gone] for i in range(queries)]
    held(got, kept_reference(q, keys, values, kept, width**-0.5))


@pytest.mark.parametrize("case", HOLES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("gone", ["no page", "a page whose scales are no numbers"])
def test_pages_that_no_query_sees_are_not_looked_at(tq, case, gone):
    """What a window has left behind, but for the sinks: the window begins inside a chunk of keys, and so do the pages behind the sinks end there."""
    page, width, queries, blocks, long = case
    sinks, window = 5, 300 if blocks * page < 1000 else 19000
    while (long - queries - window + 1) % 64 < 33:      # from a chunk's last pages on
        window -= 1
    cache = Cache(1, 2, width, page, blocks).fill([long])
    keys, values = cache.decoded(0).double(), cache.decoded(1).double()
    unseen = list(range(-(-sinks // page), (long - queries - window + 1) // page))
    assert len(unseen) >= 2
    cache.table[0, unseen] = -1 if gone == "no page" else next(n for n in range(blocks + 2) if n not in cache.table[0].tolist())
    q = by_token((1, 4, queries, width), torch.bfloat16, 1)
    got = tq.cache_attention(q, *cache.tensors, cache.table, torch.tensor([long], dtype=torch.int32).cuda(), window, sinks)
    held(got, reference(q, keys, values, [long], window, sinks, width**-0.5))
    assert status() == 0


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("case", [(16, 64), (32, 64), (16, 128), (32, 128), (64, 64), (64, 128)], ids=lambda c: "-".join(map(str, c)))
def test_a_scale_that_is_no_number_reaches_the_queries_that_see_its_page(tq, case, bad):
    """Four queries whose window passes the end of a page, and the page that the last of them alone sees."""
    page, width = case
    lengths = [6 * page + 66, 12 * page + 1]
    windows = [lengths[0] - 4 - (4 * page - 2) + 1, 7 * page]      # the first query sees the last two keys of page 3 of the first sequence, the third none
    for b, window, block in ((0, windows[0], 3), (1, windows[1], 12)):
        cache = Cache(2, 2, width, page, 13 + 66 // page).fill(lengths)
        keys, values = cache.decoded(0).double(), cache.decoded(1).double()
        where = int(cache.table[b, block])
        cache.scales[1][where, 1] = bad
        q = by_token((2, 4, 4, width), torch.float16, 1)
        got = tq.cache_attention(q, *cache.tensors, cache.table, torch.tensor(lengths, dtype=torch.int32).cuda(), window, 3)
        exact, bound = reference(q, keys, values, lengths, window, 3, width**-0.5)
        hit = torch.zeros(2, 4, 4, dtype=torch.bool)
        for i in range(4):
            at = lengths[b] - 4 + i
            hit[b, 2:, i] = any(j > at - window and j <= at for j in range(block * page, (block + 1) * page))
        assert hit.any() and not hit[b, 2:].all()
        assert not got.cpu()[hit].isfinite().any()
        held(torch.where(hit[..., None], 0, got.cpu()), (torch.where(hit[..., None], 0, exact), bound))
        assert status() == 0


# ---- writing -------------------------------------------------------------------------------------


def nearest_code(x):
    """e4m3 of f64 values of at most 448, to nearest even, as f64; NaN where x is not finite."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-40))).clamp(min=-6) - 3)
    return torch.where(x.isfinite(), torch.round(x / step) * step, math.nan)


def stored(cache_codes, cache_scales, table, x, starts, counts, page):
    """What the pool holds after a write, by the definition, in f64 on the CPU: (codes, scales)."""
    codes, scales = cache_codes.cpu().float().double(), cache_scales.cpu().double()
    x, table = x.cpu().double(), table.cpu()
    for b in range(x.shape[0]):
        n = 0
        while starts[b] >= 0 and n < counts[b]:
            block, offset = divmod(starts[b] + n, page)
            take = min(page - offset, counts[b] - n)
            where, part = int(table[b, block]), x[b, :, n : n + take]
            for h in range(x.shape[1]):
                largest = torch.where(part[h].isfinite(), part[h].abs(), 0.0).max().item()
                s = 2.0**-126
                old = scales[where, h].item() if offset else 0.0
                while largest > 448 * s or s < old:      # (a power of two, whatever the scale that was there)
                    s *= 2
                if offset:
                    codes[where, h, :offset] = nearest_code(codes[where, h, :offset] * (old / s))
                codes[where, h, offset : offset + take] = nearest_code(part[h] / s)
                scales[where, h] = s
            n += take
    return codes, scales


def same(got, expected):
    return torch.equal(got.isnan(), expected.isnan()) and torch.equal(got.nan_to_num(), expected.nan_to_num())


STORES = [  # kv_heads, tokens, width, page, starts, counts
    (1, 1, 64, 16, [0], None), (2, 1, 64, 16, [0, 1, 15, 16, 31, -1], None), (12, 1, 64, 64, [999, 0, 63], None), (3, 5, 16, 16, [14, 0, 16, 30], [5, 0, 3, 2]),
    (2, 100, 128, 64, [0, 1, 63, 64], [100, 99, 1, 64]), (1, 300, 128, 128, [0, 100], None), (2, 40, 80, 16, [7, -5, 0], [40, 40, 17]), (1, 1100, 96, 1024, [3], None),
    (8, 2, 128, 32, [31, 30], None), (1, 17, 128, 16, [15], None),
    (5, 33, 64, 16, [0, 3, 16], [33, 20, 0]), (7, 3, 128, 64, [62, 5, 64], None), (3, 130, 64, 64, [0, 63, 10], [130, 1, 70]), (1, 90, 96, 32, [31, 0], None),
    (2, 150, 112, 64, [1], None), (3, 1, 16, 16, [15, 16, 2, 0, 7], None), (1, 31, 112, 16, [9, 100], None), (3, 66, 48, 32, [5, 31], [66, 2]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", STORES, ids=lambda c: "-".join(map(str, c[:4])) + f"-{len(c[4])}")
def test_cache_store(tq, case, dtype):
    kv_heads, tokens, width, page, starts, counts = case
    batch = len(starts)
    cache = Cache(batch, kv_heads, width, page, -(-(max(starts) + tokens) // page)).fill([max(s, 0) for s in starts])
    # from far smaller to far larger than what is there
    size = torch.exp2(torch.randn(batch, kv_heads, 1, 1, generator=cache.generator) * 4).cuda()
    k, v = (by_token((batch, kv_heads, tokens, width), torch.float32, s).mul(size).to(dtype) for s in (5, 6))
    given = [tokens] * batch if counts is None else counts
    expected = [stored(cache.codes[i], cache.scales[i], cache.table, x, starts, given, page) for i, x in ((0, k), (1, v))]
    tq.cache_store(k, v, *cache.tensors, cache.table, torch.tensor(starts, dtype=torch.int32).cuda(),
                   None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda())
    for i in range(2):
        assert same(cache.scales[i].cpu().double(), expected[i][1])
        assert same(cache.codes[i].cpu().float().double(), expected[i][0])
    assert status() == 0


def test_a_scale_is_the_smallest_power_of_two(tq):
    """Around the border 448 * 2^n, at zeros, at the smallest and the largest numbers."""
    values = [0.0, 448.0, 450.0, 446.0, 1.75, 1.7578125, 2.0**-126, 2.0**-133, 3.0e38, 1.0]
    cache = Cache(len(values), 1, 16, 16, 1)
    k = torch.zeros(len(values), 1, 1, 16)
    k[:, 0, 0, 3] = torch.tensor(values)
    k = k.bfloat16().cuda()
    starts = torch.zeros(len(values), dtype=torch.int32).cuda()
    tq.cache_store(k, -k, *cache.tensors, cache.table, starts)
    for i, x in ((0, k), (1, -k)):
        codes, scales = stored(cache.codes[i], cache.scales[i], cache.table, x, [0] * len(values), [1] * len(values), 16)
        assert same(cache.scales[i].cpu().double(), scales) and same(cache.codes[i].cpu().float().double(), codes)
    pages = cache.table[:, 0].long()
    back = cache.codes[0][pages][:, 0, 0, 3].float() * cache.scales[0][pages, 0]
    assert ((back - k[:, 0, 0, 3].float()).abs() <= 2.0**-4 * k[:, 0, 0, 3].float().abs()).all()


def test_what_is_not_finite_is_stored_as_nan_and_has_no_say_in_the_scale(tq):
    cache = Cache(1, 1, 16, 16, 1)
    k = torch.ones(1, 1, 4, 16).half().cuda()
    k[0, 0, 1, 2], k[0, 0, 2, 5], k[0, 0, 3, 7] = math.inf, -math.inf, math.nan
    tq.cache_store(k, k, *cache.tensors, cache.table, torch.zeros(1, dtype=torch.int32).cuda())
    page = int(cache.table[0, 0])
    assert cache.scales[0][page, 0].item() == 2.0**-8
    codes = cache.codes[0][page, 0, :4].float()
    assert torch.equal(codes.isnan(), ~k[0, 0].isfinite()) and (codes[~codes.isnan()] == 256.0).all()


@pytest.mark.parametrize("old", [2.0**126, 1.5 * 2.0**126, 2.0**127, 1.5 * 2.0**127, 2.0**-140, 0.0, -0.25], ids=str)
def test_a_store_behind_tokens_of_any_finite_scale(tq, old):
    """A pool may come with scales that `cache_store` does not make: the page's earlier tokens keep what they stood for, as far as e4m3 at the new scale has it, and
    a value beyond 448 times the largest power of two, which is beyond f32, becomes that."""
    cache = Cache(2, 2, 64, 16, 1).fill([7, 0])
    page = int(cache.table[0, 0])
    for scales in cache.scales:
        scales[page, 0] = old
    was = [c[page, 0, :7].cpu().float().double() * old for c in cache.codes]
    k, v = (by_token((2, 2, 2, 64), torch.bfloat16, s) for s in (5, 6))
    tq.cache_store(k, v, *cache.tensors, cache.table, torch.tensor([7, 0], dtype=torch.int32).cuda())
    for i, x in enumerate((k, v)):
        scale = cache.scales[i][page, 0].item()
        largest = x[0, 0].abs().max().item()
        s = 2.0**-126
        while largest > 448 * s or (s < abs(old) and s < 2.0**127):
            s *= 2
        assert scale == s
        codes = cache.codes[i][page, 0, :9].cpu().float().double()
        assert torch.equal(codes[7:], nearest_code(x[0, 0].cpu().double() / s))
        assert torch.equal(codes[:7], nearest_code((was[i] / s).clamp(-448, 448)))
    assert status() == 0


@pytest.mark.parametrize("old", [math.nan, math.inf, -math.inf], ids=str)
def test_a_store_behind_tokens_whose_scale_is_no_number(tq, old):
    """They are no numbers either, and have no say in the new scale."""
    cache = Cache(1, 1, 64, 16, 1).fill([7])
    page = int(cache.table[0, 0])
    for scales in cache.scales:
        scales[page] = old
    k = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    tq.cache_store(k, k, *cache.tensors, cache.table, torch.tensor([7], dtype=torch.int32).cuda())
    for codes, scales in zip(cache.codes, cache.scales):
        assert scales[page, 0].item() == 2.0**-8 and (codes[page, 0, 7:9].float() == 256.0).all() and codes[page, 0, :7].float().isnan().all()


@pytest.mark.parametrize("page, tokens, width", [(16, 1, 64), (16, 16, 64), (32, 30, 64), (64, 64, 64), (64, 64, 128), (128, 120, 128)])
def test_what_is_not_finite_stays_with_its_head(tq, page, tokens, width):
    """Every other head has a NaN or an infinity, its neighbours come out as without them."""
    before, *caches = [Cache(2, 6, width, page, 3).fill([5, 0]) for _ in range(3)]
    k, v = (by_token((2, 6, tokens, width), torch.bfloat16, s) for s in (5, 6))
    starts = torch.tensor([5, 0], dtype=torch.int32).cuda()
    tq.cache_store(k, v, *caches[0].tensors, caches[0].table, starts)
    for n, x in enumerate((k, v)):
        x[:, n::2, -1, 3], x[:, n::2, 0, -1] = math.nan, -math.inf
    tq.cache_store(k, v, *caches[1].tensors, caches[1].table, starts)
    for n in range(2):
        clean, bad = (c.codes[n].view(torch.uint8) for c in caches)
        assert torch.equal(clean[:, 1 - n :: 2], bad[:, 1 - n :: 2]) and same(caches[0].scales[n][:, 1 - n :: 2], caches[1].scales[n][:, 1 - n :: 2])
        expected = stored(before.codes[n], before.scales[n], before.table, (k, v)[n], [5, 0], [tokens] * 2, page)
        assert same(caches[1].scales[n].cpu().double(), expected[1]) and same(caches[1].codes[n].cpu().float().double(), expected[0])


def test_token_by_token_is_the_prompt_at_once(tq):
    """A cache filled a token at a time holds what a prompt written in one call holds, where codes have not gone below their normal range."""
    kv_heads, width, tokens = 2, 64, 70
    one, other = Cache(2, kv_heads, width, 32, 3, seed=3), Cache(2, kv_heads, width, 32, 3, seed=3)
    k, v = ((drawn((2, kv_heads, tokens, width), torch.float32, s).sign() * (1 + drawn((2, kv_heads, tokens, width), torch.float32, s + 9).abs())).bfloat16() for s in (1, 2))
    zero = torch.zeros(2, dtype=torch.int32).cuda()
    tq.cache_store(k, v, *one.tensors, one.table, zero)
    for t in range(tokens):
        tq.cache_store(k[:, :, t : t + 1], v[:, :, t : t + 1], *other.tensors, other.table, zero + t)
    for a, b in zip(one.tensors, other.tensors):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) if a.dtype == E4M3 else same(a, b)


# ---- copying -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.uint8, torch.float16, torch.float32, torch.float64, E4M3], ids=str)
@pytest.mark.parametrize("inner", [(1,), (3,), (12,), (2, 16, 64), (5, 7)], ids=str)
def test_copy_pages(tq, dtype, inner):
    pages = 40
    t = torch.randint(0, 100, (pages, *inner), generator=torch.Generator().manual_seed(1)).to(torch.float32).to(dtype).cuda()
    before = t.float().cpu()
    tq.copy_pages([t], [3, 0, 39, 3], [5, 38, 1, 7])
    expected = before.clone()
    expected[[5, 38, 1, 7]] = before[[3, 0, 39, 3]]
    assert torch.equal(t.float().cpu(), expected)


def test_copy_pages_of_layers_views_and_many_pairs(tq):
    g = torch.Generator().manual_seed(1)
    pages = 1000
    tensors = [torch.randn(3, pages, 2, 8, generator=g).cuda(), torch.randn(3, pages, 5, generator=g).cuda()[:, :, :],
               torch.randn(4, 2 * pages, 3, generator=g).cuda()[1:3, ::2, :2], torch.randint(0, 255, (5, pages, 20000 // 8), dtype=torch.uint8, generator=g).cuda()]
    tensors += [torch.randn(1, pages, 4, generator=g).cuda() for _ in range(20)]
    order = torch.randperm(pages, generator=g).tolist()
    sources, targets = order[:450], order[500:950]
    expected = [t.clone() for t in tensors]
    for t in expected:
        t[:, targets] = t[:, sources]
    beside = [t._base.clone() if t._base is not None else None for t in tensors]
    tq.copy_pages(tensors, sources, targets, page_axis=1)
    for t, e in zip(tensors, expected):
        assert torch.equal(t, e)
    untouched = tensors[2]._base
    assert torch.equal(untouched[:, 1::2], beside[2][:, 1::2]) and torch.equal(untouched[0], beside[2][0]) and torch.equal(untouched[..., 2], beside[2][..., 2])


def test_copy_pages_of_a_page_longer_than_a_share(tq):
    t = torch.randint(0, 255, (4, 100003), dtype=torch.uint8, generator=torch.Generator().manual_seed(2)).cuda()
    before = t.clone()
    tq.copy_pages([t], [0], [3])
    assert torch.equal(t[3], before[0]) and torch.equal(t[:3], before[:3])


# ---- together ------------------------------------------------------------------------------------


def test_a_conversation_a_fork_and_its_two_ends(tq):
    """Prompts, a step, a fork that copies the last page, and a step of both: attention over the cache is attention over what was stored."""
    heads, kv_heads, width, page = 8, 2, 64, 16
    cache = Cache(3, kv_heads, width, page, 5)
    prompts = [37, 20]
    k, v = (by_token((3, kv_heads, 60, width), torch.bfloat16, s) for s in (1, 2))
    counts = torch.tensor([*prompts, 0], dtype=torch.int32).cuda()
    zero = torch.zeros(3, dtype=torch.int32).cuda()
    tq.cache_store(k[:, :, :37], v[:, :, :37], *cache.tensors, cache.table, zero, counts)
    # the third sequence is the first one's fork: its full pages are shared, its last one is a copy
    cache.table[2, :2] = cache.table[0, :2]
    tq.copy_pages(cache.tensors, [int(cache.table[0, 2])], [int(cache.table[2, 2])])
    lengths = [38, 21, 38]
    step = torch.tensor([n - 1 for n in lengths], dtype=torch.int32).cuda()
    tq.cache_store(k[:, :, 40:41], v[:, :, 40:41], *cache.tensors, cache.table, step)
    q = by_token((3, heads, 1, width), torch.bfloat16, 7)
    for window, sinks in ((None, 0), (16, 4)):
        got = tq.cache_attention(q, *cache.tensors, cache.table, torch.tensor(lengths, dtype=torch.int32).cuda(), window, sinks)
        held(got, reference(q, cache.decoded(0).double(), cache.decoded(1).double(), lengths, window, sinks, 0.125))
    # what the cache holds is what went in, to half a step of e4m3 (2^-4) of it or, below the normal range, 2^-10 of the scale
    for which, x in ((0, k), (1, v)):
        values = cache.decoded(which)
        for b, n in ((0, 37), (1, 20)):
            error = (values[b, :, :n] - x[b, :, :n].float().cpu()).abs()
            pages = cache.table[b].long().cpu()
            step_of = cache.scales[which].cpu()[pages].T.repeat_interleave(page, 1)[:, :n, None] * 2.0**-10
            assert (error <= torch.maximum(2.0**-4 * x[b, :, :n].float().cpu().abs(), step_of)).all()
        assert torch.equal(values[0, :, :37].view(torch.uint8), values[2, :, :37].view(torch.uint8))
    assert status() == 0


@pytest.mark.parametrize("blocks, long", [(40, 600), (300, 4500)], ids=["whole units", "shares"])
def test_a_step_replayed_from_a_graph(tq, blocks, long):
    """Lengths, starts and tables are read on the device: a captured step goes on as they change. Two graphs share nothing, on two streams at once."""
    heads, kv_heads, width, page = 4, 2, 64, 16
    streams = [torch.cuda.Stream() for _ in range(2)]
    caches = [Cache(2, kv_heads, width, page, blocks, seed=i).fill([long, 5]) for i in range(2)]
    k, q = by_token((2, kv_heads, 1, width), torch.bfloat16, 1), by_token((2, heads, 1, width), torch.bfloat16, 2)
    starts = [torch.tensor([long, 5], dtype=torch.int32).cuda() for _ in range(2)]
    lengths = [s + 1 for s in starts]
    graphs, results = [], []
    for cache, start, length in zip(caches, starts, lengths):
        tq.cache_store(k, k, *cache.tensors, cache.table, start)
        tq.cache_attention(q, *cache.tensors, cache.table, length)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            tq.cache_store(k, k, *cache.tensors, cache.table, start)
            start.add_(1)
            results.append(tq.cache_attention(q, *cache.tensors, cache.table, length))
            length.add_(1)
        graphs.append(graph)
    for start, length in zip(starts, lengths):
        start.copy_(torch.tensor([long, 5]))
        length.copy_(torch.tensor([long + 1, 6]))
    torch.cuda.synchronize()
    for step in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for cache, got in zip(caches, results):
        held(got, reference(q, cache.decoded(0).double(), cache.decoded(1).double(), [long + 20, 25], None, 0, 0.125))
    assert status() == 0


@pytest.mark.parametrize("captured", [False, True], ids=["eager", "captured"])
@pytest.mark.parametrize("blocks, long", [(40, 600), (300, 4500)], ids=["whole units", "shares"])
def test_kernels_that_start_early_wait_for_what_they_read(tq, blocks, long, captured):
    """Copies, fills, another stream's work, stores, page copies and attention in turn, each reading what the one before wrote: as with a wait after each."""
    cache = Cache(2, 2, 64, 16, blocks, seed=3).fill([long, 5])
    before = [t.view(torch.uint8).clone() for t in cache.tensors]
    spare = [min(set(range(2 * blocks + 2)) - set(cache.table.flatten().tolist()))]
    last = [int(cache.table[0, (long + 1) // 16])]
    host = torch.randn(2, 1, 2, 64, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).pin_memory()
    starts, lengths = (torch.tensor([long + more, 5 + more], dtype=torch.int32).cuda() for more in (0, 1))
    k, q = torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()

    def chain(wait):
        main, results = torch.cuda.current_stream(), []
        for step in range(6):
            k.copy_(host, non_blocking=True)
            wait()
            tq.cache_store(k.transpose(1, 2), k.transpose(1, 2), *cache.tensors, cache.table, starts)
            wait()
            side.wait_stream(main)
            with torch.cuda.stream(side):
                q.fill_(step / 4 - 1)
                q[:, 1].zero_()
            main.wait_stream(side)
            wait()
            results.append(tq.cache_attention(q, *cache.tensors, cache.table, lengths))
            wait()
            tq.copy_pages(cache.tensors, last, spare)
            wait()
            cache.codes[1].view(torch.uint8)[last[0]].zero_()
            wait()
            results.append(tq.cache_attention(q, *cache.tensors, cache.table, lengths))
            wait()
            tq.copy_pages(cache.tensors, spare, last)
            wait()
            results.append(tq.cache_attention(q, *cache.tensors, cache.table, lengths))
            results.append(tq.window_attention(q, q, results[-1]))
            k.zero_()
            wait()
        return results

    expected = [t.clone() for t in chain(torch.cuda.synchronize)]
    for tensor, was in zip(cache.tensors, before):
        tensor.view(torch.uint8).copy_(was)
    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            results = chain(lambda: None)
        for _ in range(3):
            graph.replay()
    else:
        results = chain(lambda: None)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(results, expected)) and not torch.equal(expected[0], expected[1])
    assert status() == 0


@pytest.mark.parametrize("seen_before", [False, True])
def test_a_recorded_step_keeps_its_scratch(tq, seen_before):
    """A recipe replays launches with the addresses they were recorded with: scratch that went back to torch's allocator would be someone else's by then."""
    from tessiq_b200 import _lib

    cache = Cache(2, 2, 64, 16, 300).fill([4500, 5])
    lengths = torch.tensor([4500, 5], dtype=torch.int32).cuda()
    q, other = (by_token((2, 4, 1, 64), torch.bfloat16, s) for s in (1, 2))
    dense_q, dense_k = by_token((1, 4, 2, 64), torch.bfloat16, 3), by_token((1, 2, 5000, 64), torch.bfloat16, 4)
    expected, dense = tq.cache_attention(other, *cache.tensors, cache.table, lengths), tq.window_attention(dense_q, dense_k, dense_k)
    if not seen_before:
        q, dense_q = (t.clone() for t in (q.contiguous(), dense_q.contiguous()))      # (a signature of its own)
    handle = ctypes.c_void_p()
    _lib.check(_lib.lib.tq_recipe_create(ctypes.byref(handle)))
    assert _lib.lib.tq_is_recording() == 0
    _lib.check(_lib.lib.tq_recipe_begin_recording(handle))
    assert _lib.lib.tq_is_recording() == 1
    got, dense_got = tq.cache_attention(q, *cache.tensors, cache.table, lengths), tq.window_attention(dense_q, dense_k, dense_k)
    _lib.check(_lib.lib.tq_recipe_end_recording(handle))
    guards = [torch.full((1 << n,), 0x55, dtype=torch.uint8, device="cuda") for n in range(9, 23) for _ in range(4)]      # whatever was given back
    q.copy_(other)
    torch.cuda.synchronize()
    for _ in range(2):
        _lib.check(_lib.lib.tq_recipe_run(handle, 0, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(got, expected) and torch.equal(dense_got, dense)
    assert all((g == 0x55).all() for g in guards)
    assert _lib.lib.tq_recipe_steps(handle) == 2
    _lib.check(_lib.lib.tq_recipe_destroy(handle))


def test_recorded_steps_of_threads_on_one_stream(tq):
    """Recordings of one stream share its scratch: what one thread's attention leaves there for its join must not be another's by then."""
    import threading

    from test_threads import run_threads

    from tessiq_b200 import _lib

    count, recipes = 4, []
    caches = [Cache(1 + i, 2, 64, 16, 300, seed=i).fill([4500 - 700 * i, 60, 1, 900][: 1 + i]) for i in range(count)]
    lengths = [torch.tensor([4500 - 700 * i, 60, 1, 900][: 1 + i], dtype=torch.int32).cuda() for i in range(count)]
    queries = [by_token((1 + i, 4, 1 + i, 64), torch.bfloat16, i) for i in range(count)]
    expected = [tq.cache_attention(q, *c.tensors, c.table, n) for q, c, n in zip(queries, caches, lengths)]
    for q, c, n in zip(queries, caches, lengths):
        handle = ctypes.c_void_p()
        _lib.check(_lib.lib.tq_recipe_create(ctypes.byref(handle)))
        _lib.check(_lib.lib.tq_recipe_begin_recording(handle))
        recipes.append((handle, tq.cache_attention(q, *c.tensors, c.table, n)))
        _lib.check(_lib.lib.tq_recipe_end_recording(handle))
    stream = torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    turn = threading.Barrier(count)

    def work(i):
        for _ in range(20):
            turn.wait()
            for _ in range(20):
                _lib.check(_lib.lib.tq_recipe_run(recipes[i][0], 0, stream))
            turn.wait()
            if i == 0:
                torch.cuda.synchronize()
                for (_, got), right in zip(recipes, expected):
                    assert torch.equal(got, right)
                    got.zero_()
                torch.cuda.synchronize()

    run_threads(work, count)
    for handle, _ in recipes:
        _lib.check(_lib.lib.tq_recipe_destroy(handle))
    assert status() == 0


def test_repeated_calls_give_the_same_bits_on_any_stream_and_from_threads(tq):
    import threading

    cache = Cache(3, 2, 64, 16, 200).fill([3100, 40, 1])
    q, lengths = by_token((3, 8, 2, 64), torch.bfloat16, 1), torch.tensor([3100, 40, 1], dtype=torch.int32).cuda()
    first = tq.cache_attention(q, *cache.tensors, cache.table, lengths, 2500, 4)
    torch.cuda.synchronize()
    wrong = []

    def many():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                again = tq.cache_attention(q, *cache.tensors, cache.table, lengths, 2500, 4)
                if not torch.equal(again, first):
                    wrong.append(1)

    threads = [threading.Thread(target=many) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and status() == 0


def test_a_pool_beyond_four_gigabytes(tq):
    kv_heads, width, page, pages = 8, 128, 64, 72000      # 4.7 GB of codes each
    shape = (pages, kv_heads, page, width)
    codes = [torch.empty(shape, dtype=E4M3, device="cuda") for _ in range(2)]
    scales = [torch.empty(shape[:2], device="cuda") for _ in range(2)]
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32).cuda()
    k, v = (by_token((1, kv_heads, 150, width), torch.bfloat16, s) for s in (1, 2))
    tq.cache_store(k, v, *codes, *scales, table, torch.zeros(1, dtype=torch.int32).cuda())
    tq.copy_pages([*codes, *scales], [pages - 1], [40000])
    for t in (*codes, *scales):
        raw = t.view(torch.uint8) if t.dtype == E4M3 else t
        assert torch.equal(raw[40000], raw[pages - 1])
    table[0, 0] = 40000
    q = by_token((1, 16, 1, width), torch.bfloat16, 3)
    got = tq.cache_attention(q, *codes, *scales, table, torch.tensor([150], dtype=torch.int32).cuda())
    at = table[0].long()
    values = [(c.view(torch.uint8)[at].view(E4M3).float() * s[at][..., None, None]).permute(1, 0, 2, 3).flatten(1, 2)[None] for c, s in zip(codes, scales)]
    held(got, reference(q, values[0].double(), values[1].double(), [150], None, 0, width**-0.5))
    assert status() == 0


def test_on_another_device_than_the_current_one(tq):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    q, k = drawn((2, 4, 3, 64), torch.float16, 1).to("cuda:1"), drawn((2, 2, 2000, 64), torch.float16, 2).to("cuda:1")
    got = tq.window_attention(q, k, k, 1500, 4)
    assert got.device.index == 1 and torch.cuda.current_device() == 0
    held(got, reference(q, k, k, [2000, 2000], 1500, 4, 0.125))


def test_a_paged_cache_through_forks_drafts_and_moves(tq):
    """Two layers, three conversations: what each one's attention gives is attention over the tokens it was given, as the cache holds them."""
    from tessiq_b200.cache import PagedCache

    layers, heads, kv_heads, width = 2, 4, 2, 32
    cache = PagedCache(layers, kv_heads, width, pages=24, page_tokens=16)
    for t in cache.tensors:      # whatever memory held before
        (t.view(torch.uint8) if t.dtype == E4M3 else t).fill_(0x7F if t.dtype == E4M3 else math.nan)
    given = {}                   # sequence -> what was stored, [layers, 2, kv_heads, tokens, width]
    seeds = iter(range(1000))

    def write(sequences, tokens):
        counts = [tokens] * len(sequences) if isinstance(tokens, int) else tokens
        step = cache.extend(sequences, tokens)
        new = [[drawn((len(sequences), kv_heads, max(counts), width), torch.bfloat16, next(seeds)) for _ in range(2)] for _ in range(layers)]
        for layer, (k, v) in enumerate(new):
            cache.store(step, layer, k, v)
        for i, sequence in enumerate(sequences):
            more = torch.stack([torch.stack([x[i, :, : counts[i]] for x in pair]) for pair in new])
            given[sequence] = torch.cat([given[sequence], more], 3) if sequence in given else more
        return step

    def agrees(sequences, step, window=None, sinks=0):
        q = by_token((len(sequences), heads, 1, width), torch.bfloat16, next(seeds))
        for layer in range(layers):
            got = cache.attention(step, layer, q, window, sinks)
            for i, sequence in enumerate(sequences):
                pages = cache.books.pages_of(sequence)
                length = cache.length(sequence)
                k, v = ((codes[layer].view(torch.uint8)[pages].view(E4M3).float() * scales[layer][pages][..., None, None]).permute(1, 0, 2, 3).flatten(1, 2)[None, :, :length]
                        for codes, scales in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)))
                for held_values, was in ((k, given[sequence][layer, 0]), (v, given[sequence][layer, 1])):
                    # (half a step of e4m3, or of its smallest numbers at a scale of at most max / 224)
                    assert was.shape[1] == length
                    assert ((held_values[0] - was.float()).abs() <= 2.0**-4 * was.float().abs() + 2.0**-10 * was.float().abs().max() / 224).all()
                held(got[i : i + 1], reference(q[i : i + 1], k.double(), v.double(), [length], window, sinks, width**-0.5))

    a, b = cache.start(), cache.start()
    agrees([a, b], write([a, b], [37, 5]))
    c = cache.fork(a)
    given[c] = given[a]
    agrees([c, a, b], write([c, a, b], 1))
    d = cache.fork(b)
    given[d] = given[b]
    agrees([d, b], write([d, b], [4, 20]), 7, 2)
    cache.truncate(d, 8)
    given[d] = given[d][:, :, :, :8]
    cache.free(a)
    del given[a]
    assert cache.compact() > 0
    live = [b, c, d]
    agrees(live, write(live, [1, 16, 3]))
    agrees(live, write(live, 1), 20, 3)
    used = {page for sequence in live for page in cache.books.pages_of(sequence)}
    assert len(used) + cache.books.free_pages == 24 and status() == 0


@pytest.mark.parametrize("way", ["captured", "recorded"])
def test_the_books_are_not_kept_in_a_graph(tq, way):
    """A step's table is made on the host, as pages are handed out: in a graph it would be sent again from memory that is somebody else's by then, and the
    copies that the books count on would not have been made. Storing and attention go into a graph, extend and compact are refused and change nothing."""
    from tessiq_b200 import _lib
    from tessiq_b200.cache import PagedCache

    cache = PagedCache(1, 2, 32, pages=8, page_tokens=16)
    gone, a = cache.start(), cache.start()
    k, q = by_token((1, 2, 20, 32), torch.bfloat16, 1), by_token((1, 4, 1, 32), torch.bfloat16, 2)
    cache.extend([gone], 3)
    step = cache.extend([a], 20)
    cache.free(gone)
    cache.store(step, 0, k, k)
    expected = cache.attention(step, 0, q)
    torch.cuda.synchronize()
    before = (cache.books.pages_of(a), cache.length(a), cache.books.free_pages)

    def inside():
        for call in (lambda: cache.extend([a], 1), cache.compact):
            with pytest.raises(RuntimeError, match="graph"):
                call()
        cache.store(step, 0, k, k)
        return cache.attention(step, 0, q)

    if way == "captured":
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = inside()
        graph.replay()
    else:
        handle = ctypes.c_void_p()
        _lib.check(_lib.lib.tq_recipe_create(ctypes.byref(handle)))
        _lib.check(_lib.lib.tq_recipe_begin_recording(handle))
        got = inside()
        _lib.check(_lib.lib.tq_recipe_end_recording(handle))
        _lib.check(_lib.lib.tq_recipe_run(handle, 0, torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        _lib.check(_lib.lib.tq_recipe_destroy(handle))
    torch.cuda.synchronize()
    assert torch.equal(got, expected) and before == (cache.books.pages_of(a), cache.length(a), cache.books.free_pages)
    assert cache.compact() == 1 and cache.extend([a], 1).lengths.tolist() == [21] and status() == 0


def test_steps_of_nothing(tq):
    """No sequence, sequences without tokens, and no new tokens for those that have some."""
    from tessiq_b200.cache import PagedCache

    cache = PagedCache(1, 2, 32, pages=8, page_tokens=16)
    a, b = cache.start(), cache.start()
    k, q = by_token((2, 2, 5, 32), torch.bfloat16, 1), by_token((2, 4, 3, 32), torch.bfloat16, 2)
    nobody = cache.extend([], 1)
    cache.store(nobody, 0, k[:0], k[:0])
    assert cache.attention(nobody, 0, q[:0]).shape == (0, 4, 3, 32)
    empty = cache.extend([a, b], 0)
    cache.store(empty, 0, k[:, :, :0], k[:, :, :0])
    assert cache.attention(empty, 0, q).count_nonzero().item() == 0
    first = cache.extend([a, b], [5, 0])
    cache.store(first, 0, k, k)
    got = cache.attention(first, 0, q)
    assert got[1].count_nonzero().item() == 0 and got[0].count_nonzero().item() > 0
    again = cache.extend([a, b], 0)
    before = [t.view(torch.uint8).clone() for t in cache.tensors]
    cache.store(again, 0, k, k)
    assert torch.equal(cache.attention(again, 0, q), got) and all(torch.equal(t.view(torch.uint8), was) for t, was in zip(cache.tensors, before))
    assert status() == 0
