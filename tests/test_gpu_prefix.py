"""Attention of sequences that share their first keys, against a plain form in 64 bits.

How far a result may be off (`bound`): half a step of its type, relative (bf16 2^-8, f16 2^-11); half a step of the probabilities' rounding to f16, 2^-11,
relative to sum_j p_j |v_j|; below f16's normal range, 2^-14 of 2^7 times a probability times its page's scale over the largest scale, 2^-25 / 2^7 = 2^-32 a
key of the largest |v| that scale allows; an error d of a score is a relative error of 2 d in the probabilities, and f32 sums of `width` products give
d = (width + 4) 2^-24 sum |q| |k| scale, ex2.approx another 2^-21; f32 sums over n keys (n + 8) 2^-24."""

import ctypes
import math
import threading

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


def form(case):
    from tessiq_b200 import _lib

    kind, parts, rows = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int32()
    _lib.check(_lib.lib.tq_prefix_attention_form(case.batch, case.heads, case.kv_heads, case.q_tokens, case.width, case.page, case.table.shape[1], case.runs, 0,
                                                 ctypes.byref(kind), ctypes.byref(parts), ctypes.byref(rows)))
    return {0: "streamed", 1: f"tiles {rows.value}", 3: "apart"}[kind.value]


class Case:
    """`runs` runs of `each` sequences that have `prompt` tokens in common, on whole pages together, and tails of their own."""

    def __init__(self, runs, each, heads, kv_heads, q_tokens, prompt, tail, width, page, dtype=torch.bfloat16, seed=1, wide=None):
        self.runs, self.each, self.heads, self.kv_heads, self.q_tokens, self.width, self.page = runs, each, heads, kv_heads, q_tokens, width, page
        self.batch = batch = runs * each
        g, there = torch.Generator().manual_seed(seed), torch.Generator(device="cuda").manual_seed(seed)
        whole = prompt // page
        blocks = wide or max(1, -(-(prompt + tail) // page))
        pages = runs * whole + batch * (blocks - whole) + 3
        order = torch.randperm(pages, generator=g).int()
        table = torch.empty(runs, each, blocks, dtype=torch.int32)
        table[:, :, :whole] = order[: runs * whole].reshape(runs, 1, whole)
        table[:, :, whole:] = order[runs * whole : runs * whole + batch * (blocks - whole)].reshape(runs, each, blocks - whole)
        self.table = table.reshape(batch, blocks).cuda()
        shape = (pages, kv_heads, page, width)
        self.codes = [(torch.randn(shape, generator=there, device="cuda") * 64).clamp(-448, 448).to(E4M3) for _ in range(2)]
        self.scales = [torch.exp2(torch.randint(-8, -4, shape[:2], generator=there, device="cuda").float()) for _ in range(2)]
        tails = torch.randint(q_tokens, max(q_tokens, tail) + 1, (batch,), generator=g)
        self.lengths = (prompt + tails).int().clamp(max=blocks * page).cuda()
        self.shared = torch.full((runs,), whole * page, dtype=torch.int32, device="cuda")
        self.q = torch.randn(batch, q_tokens, heads, width, generator=g).to(dtype).cuda().transpose(1, 2)

    @property
    def tensors(self):
        return (*self.codes, *self.scales)

    def run(self, tq, **more):
        return tq.prefix_attention(self.q, *self.tensors, self.table, self.lengths, self.shared, **more)

    def reference(self, scale=None, absent=()):
        scale = 1 / math.sqrt(self.width) if scale is None else scale
        group = self.heads // self.kv_heads
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        bound = torch.full(self.q.shape, 1e-30, dtype=torch.float64, device="cuda")
        u_out = torch.finfo(self.q.dtype).eps / 2
        for b, length in enumerate(self.lengths.tolist()):
            length = min(max(length, 0), self.table.shape[1] * self.page)
            pages = self.table[b, : -(-length // self.page)].long()
            here = torch.tensor([p not in absent for p in pages.tolist()], device="cuda").repeat_interleave(self.page)[:length]
            pages = torch.where((pages >= 0) & (pages < self.codes[0].shape[0]), pages, 0)
            k, v = ((c.view(torch.uint8)[pages].view(E4M3).double() * s[pages].double()[..., None, None]).transpose(0, 1).reshape(self.kv_heads, -1, self.width)[:, :length]
                    for c, s in zip(self.codes, self.scales))
            largest = (self.scales[1][pages].double().abs().nan_to_num(0.0, 0.0).amax(0) if len(pages) else torch.zeros(self.kv_heads, device="cuda", dtype=torch.float64)) * 448
            for i in range(self.q_tokens):
                p = length - self.q_tokens + i
                if p < 0:
                    continue
                sees = here[: p + 1]
                kk, vv = k[:, : p + 1][:, sees], v[:, : p + 1][:, sees]
                q = self.q[b, :, i].double().reshape(self.kv_heads, group, self.width)
                if kk.shape[1] == 0:
                    out[b, :, i] = math.nan
                    continue
                weight = torch.softmax(q @ kk.transpose(1, 2) * scale, -1)
                out[b, :, i] = (weight @ vv).reshape(self.heads, self.width)
                spread = (weight @ vv.abs()).reshape(self.heads, self.width)
                d = (self.width + 4) * 2.0**-24 * (q.abs() @ kk.abs().transpose(1, 2)).amax(-1).reshape(self.heads, 1) * scale + 2.0**-21
                bound[b, :, i] += u_out * out[b, :, i].abs() + (2.0**-11 + 2 * d + (kk.shape[1] + 8) * 2.0**-24) * spread
                bound[b, :, i] += 2.0**-32 * kk.shape[1] * largest.repeat_interleave(group)[:, None]
        return out, bound

    def held(self, got, scale=None, absent=()):
        exact, bound = self.reference(scale, absent)
        got = got.detach().double()
        assert torch.equal(got.isnan(), exact.isnan())
        over = ((got - exact).abs() / bound).nan_to_num(0.0).max().item() if got.numel() else 0.0
        assert over <= 1.0, f"{over:.2f} times what roundings explain"


SHAPES = [  # runs, each, heads, kv_heads, q_tokens, prompt, tail, width, page, the way it takes
    (1, 1, 4, 2, 1, 300, 9, 64, 16, "apart"), (1, 2, 1, 1, 1, 127, 1, 64, 16, None), (1, 3, 2, 1, 1, 128, 1, 16, 16, None), (2, 5, 3, 3, 1, 129, 30, 32, 32, None),
    (12, 4, 12, 12, 1, 2048, 40, 64, 64, "streamed"), (16, 3, 16, 8, 2, 3000, 70, 128, 16, "streamed"), (20, 16, 8, 8, 1, 1500, 5, 80, 128, "streamed"),
    (16, 2, 40, 8, 1, 4096, 100, 128, 1024, "streamed"), (12, 8, 16, 16, 1, 2048, 100, 32, 256, "streamed"),
    (1, 128, 2, 1, 1, 9000, 33, 64, 16, "tiles 128"), (1, 80, 32, 8, 1, 4000, 33, 64, 32, "tiles 128"), (1, 24, 20, 4, 1, 9000, 33, 128, 64, "tiles 128"),
    (1, 200, 8, 2, 1, 4000, 40, 128, 64, "tiles 128"), (2, 100, 9, 3, 1, 3333, 50, 96, 128, "tiles 128"), (1, 300, 8, 8, 1, 2600, 8, 48, 256, "tiles 128"),
    (1, 256, 8, 4, 1, 6000, 33, 64, 16, "tiles 128"), (1, 100, 64, 8, 1, 3000, 40, 128, 64, "tiles 128"), (1, 150, 16, 4, 2, 1800, 40, 128, 32, "tiles 128"),
    (3, 70, 14, 2, 4, 1300, 11, 112, 16, "tiles 128"), (1, 200, 32, 4, 1, 5000, 30, 64, 1024, "tiles 256"),
    (1, 200, 32, 4, 1, 4000, 33, 64, 16, "tiles 256"), (1, 128, 64, 8, 1, 6000, 40, 128, 64, "tiles 256"), (1, 160, 16, 4, 4, 2500, 40, 128, 32, "tiles 256"),
    (3, 110, 14, 2, 4, 1300, 11, 112, 16, "tiles 256"), (2, 400, 16, 8, 1, 1500, 33, 48, 32, "tiles 256"), (1, 256, 64, 8, 1, 2000, 10, 80, 16, "tiles 128"),
    (1, 3, 4, 2, 130, 700, 150, 64, 16, None), (2, 2, 6, 1, 77, 1000, 90, 128, 32, None), (1, 5, 16, 4, 300, 2100, 310, 128, 64, None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_prefix_attention(tq, shape, dtype):
    case = Case(*shape[:9], dtype=dtype)
    if shape[9] is not None:
        assert form(case) == shape[9]
    got = case.run(tq)
    assert got.shape == case.q.shape and got.dtype == dtype
    case.held(got)
    assert status() == 0


KINDS = [  # a case of each way
    (12, 4, 12, 12, 1, 2048, 40, 64, 64), (1, 128, 2, 1, 1, 9000, 33, 64, 16, torch.float16), (1, 24, 20, 4, 1, 9000, 60, 128, 64), (1, 160, 16, 4, 4, 2500, 40, 128, 32),
    (1, 200, 32, 4, 1, 4000, 33, 64, 16),
]


def test_the_ways(tq):
    assert [form(Case(*kind)) for kind in KINDS] == ["streamed", "tiles 128", "tiles 128", "tiles 256", "tiles 256"]


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_what_is_said_to_be_shared(tq, which):
    """Any number of the tokens that are common may be said to be: none, less than a tile, no whole tiles, all; and runs may differ."""
    case = Case(*KINDS[which])
    whole = int(case.shared[0])
    for shared in (-5, 0, 1, 127, 128, 255, 1000, whole - 1, whole):
        case.shared.fill_(shared)
        case.held(case.run(tq))
    case.shared.copy_(torch.arange(case.runs) * 200 % (whole + 1))
    case.held(case.run(tq))
    assert status() == 0


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_sequences_that_are_shorter(tq, which):
    """Padding, sequences shorter than what the others share, one that ends just there, tables that name nothing behind a sequence's end: they take no part
    and read their own keys; a NaN in what they do not see does not reach them."""
    case = Case(*KINDS[which])
    whole = int(case.shared[0])
    lengths = [0, 1, case.page + 3, whole - 1, whole, whole + 1, -7, 130]
    for b in range(0, case.batch - 1, 2):
        case.lengths[b] = lengths[b // 2 % len(lengths)]
    for b, length in enumerate(case.lengths.tolist()):
        case.table[b, max(0, -(-length // case.page)) :] = -12345
    case.held(case.run(tq))
    assert status() == 0
    case.codes[0].view(torch.uint8)[case.table[-1, whole // case.page - 1].long()] = 0x7F      # the last sequence sees it
    case.codes[1].view(torch.uint8)[case.table[-1, whole // case.page - 2].long()] = 0xFF
    got = case.run(tq)
    assert got[-1].isnan().all() and not got[2].isnan().any()
    exact, _ = case.reference()
    assert torch.equal(got.isnan(), exact.isnan())
    assert status() == 0


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_nobody_takes_part(tq, which):
    case = Case(*KINDS[which])
    case.lengths.clamp_(max=100)
    case.held(case.run(tq))
    case.lengths.zero_()
    assert not case.run(tq).any()
    assert status() == 0


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_scores_that_rise(tq, which):
    """Every tile rises far above those before it, so that every step moves the rows' reference points, the last of a part too."""
    case = Case(*KINDS[which])
    unit = torch.zeros(case.width)
    unit[0] = 16.0
    case.q.copy_(unit.to(case.q.dtype).expand_as(case.q))
    codes = torch.zeros(case.codes[0].shape)
    for b in range(case.batch):
        for block, page in enumerate(case.table[b].tolist()):
            at = block * case.page + torch.arange(case.page)
            codes[page, :, :, 0] = (at / 16.0).floor().clamp(max=440)
    case.codes[0].copy_(codes.to(E4M3))
    case.scales[0].fill_(1.0)
    for scale in (0.25, 4.0):
        case.held(case.run(tq, scale=scale), scale=scale)
    case.codes[0].copy_((-codes).to(E4M3))
    case.held(case.run(tq, scale=0.25), scale=0.25)
    assert status() == 0


@pytest.mark.parametrize("which", range(len(KINDS)))
@pytest.mark.parametrize("spread", ["far", "wide", "odd", "negative"])
def test_scales_of_any_size(tq, which, spread):
    """Scales of the values that lie far apart are taken in walks of their own: the pages of large ones may hold zeros alone."""
    case = Case(*KINDS[which])
    g = torch.Generator().manual_seed(3)
    shape = case.scales[1].shape
    if spread == "far":
        case.scales[1].copy_(torch.exp2(torch.randint(-40, 41, shape, generator=g).float()))
        case.codes[1].view(torch.uint8)[case.scales[1] > 2.0**-10] = 0
    elif spread == "wide":
        case.scales[1].copy_(torch.exp2(torch.randint(-9, 4, shape, generator=g).float()))
    elif spread == "odd":
        case.scales[1].copy_(torch.rand(shape, generator=g) * 3 + 1e-4)
        case.scales[0].copy_(torch.rand(shape, generator=g) * 0.01 + 1e-4)
    else:
        for s in case.scales:
            s.mul_(torch.where(torch.rand(shape, generator=g) < 0.5, -1.0, 1.0).cuda())
    case.held(case.run(tq))
    assert status() == 0


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_scales_that_are_no_numbers_or_zero(tq, which):
    case = Case(*KINDS[which])
    first = case.table[0, 0].long()
    case.scales[1][first] = 0.0
    case.held(case.run(tq))
    case.scales[1].zero_()
    case.held(case.run(tq))
    case.scales[1].fill_(2.0**-126)
    case.scales[1][first] = 2.0**120
    case.codes[1][first] = 0.0
    case.held(case.run(tq))
    for which_scales in (0, 1):
        kept = case.scales[which_scales].clone()
        case.scales[which_scales][first, 0] = math.nan
        got, group = case.run(tq), case.heads // case.kv_heads
        assert got[: case.each, :group].isnan().all() and not got[:, group:].isnan().any()
        case.scales[which_scales].copy_(kept)
    assert status() == 0


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_pages_that_are_not_there(tq, which):
    """Left out for everybody who would see them, and reported."""
    case = Case(*KINDS[which])
    case.table[:, 3] = 1 << 30
    case.table[:, 5] = -1
    got = case.run(tq)
    assert status() == 0x50414745
    case.held(got, absent={1 << 30, -1})


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_sequences_longer_than_the_table(tq, which):
    case = Case(*KINDS[which])
    capacity = case.table.shape[1] * case.page
    case.lengths[-1] = capacity + 100
    case.shared.fill_(capacity * 2)      # (more than there is: what fits the table)
    case.table[: case.each] = case.table[0]
    if case.runs > 1:
        for r in range(case.runs):
            case.table[r * case.each : (r + 1) * case.each] = case.table[r * case.each]
    case.lengths[:-1] = capacity
    got = case.run(tq)
    assert status() == 0x4C454E47
    case.held(got)


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_queries_of_any_size(tq, which):
    case = Case(*KINDS[which])
    small = torch.finfo(case.q.dtype).tiny
    case.q[0].mul_(1e3)
    case.q[1] = 0.0
    case.q[2].mul_(small if case.q.dtype == torch.bfloat16 else 2.0**-10)
    case.held(case.run(tq))
    case.held(case.run(tq, scale=30.0), scale=30.0)
    case.q[1, 0, 0, 3] = math.nan
    got = case.run(tq)
    assert got[1, 0, 0].isnan().all() and got.isnan().sum() == case.width
    case.q[1, 0, 0, 3] = math.inf
    got = case.run(tq)
    assert got.isnan().sum() == case.width
    assert status() == 0


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_strides_and_layouts(tq, which):
    case = Case(*KINDS[which])
    expected = case.run(tq)
    assert expected.transpose(1, 2).is_contiguous()
    assert torch.equal(case.run(tq, token_major=False), expected) and case.run(tq, token_major=False).is_contiguous()
    q = torch.randn(case.batch, case.heads, case.q_tokens, 3 * case.width, device="cuda").to(case.q.dtype)
    q[..., case.width : 2 * case.width] = case.q
    table = torch.full((case.batch, case.table.shape[1] + 7), 77, dtype=torch.int32, device="cuda")
    table[:, : case.table.shape[1]] = case.table
    got = tq.prefix_attention(q[..., case.width : 2 * case.width], *case.tensors, table[:, : case.table.shape[1]], case.lengths, case.shared)
    assert torch.equal(got, expected)
    for _ in range(5):      # (the same again and again: no sum depends on who is first)
        assert torch.equal(case.run(tq), expected)
    assert status() == 0


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_graphs_streams_and_threads(tq, which):
    """Two graphs on two streams replayed at once, with lengths and prefixes that change between replays, and host threads."""
    case = Case(*KINDS[which])
    case.run(tq)
    streams, graphs, outs, lengths, shared = [torch.cuda.Stream() for _ in range(2)], [], [], [], []
    for stream in streams:
        lengths.append(case.lengths.clone())
        shared.append(case.shared.clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(tq.prefix_attention(case.q, *case.tensors, case.table, lengths[-1], shared[-1]))
        graphs.append(graph)
    whole = int(case.shared[0])
    for turn in range(3):
        expected = []
        torch.cuda.synchronize()
        for i in range(2):
            lengths[i].copy_(case.lengths - 7 * turn - 3 * i)
            shared[i].fill_(whole - 130 * (turn + i))
            expected.append(tq.prefix_attention(case.q, *case.tensors, case.table, lengths[i], shared[i]))
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, expected))
    expected, wrong = case.run(tq), []

    def many():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = case.run(tq)
            torch.cuda.current_stream().synchronize()
            if not torch.equal(got, expected):
                wrong.append(got)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=many) for _ in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong and status() == 0


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_a_recorded_call(tq, which):
    from tessiq_b200 import _lib

    case = Case(*KINDS[which])
    handle = ctypes.c_void_p()
    _lib.check(_lib.lib.tq_recipe_create(ctypes.byref(handle)))
    _lib.check(_lib.lib.tq_recipe_begin_recording(handle))
    out = case.run(tq)
    _lib.check(_lib.lib.tq_recipe_end_recording(handle))
    for _ in range(3):
        _lib.check(_lib.lib.tq_recipe_run(handle, 0, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(out, case.run(tq))
    _lib.check(_lib.lib.tq_recipe_destroy(handle))
    assert status() == 0


def test_a_pool_beyond_4_gb(tq):
    """Pages at the end of a pool of 5 GB."""
    case = Case(1, 100, 8, 2, 1, 4000, 40, 128, 64)
    pages, used = 5 * (1 << 30) // (2 * 64 * 128), case.codes[0].shape[0]
    expected = case.run(tq)
    for c in range(2):
        large = torch.empty(pages, 2, 64, 128, dtype=E4M3, device="cuda")
        large[pages - used :] = case.codes[c]
        scales = torch.ones(pages, 2, device="cuda")
        scales[pages - used :] = case.scales[c]
        case.codes[c], case.scales[c] = large, scales
    case.table += pages - used
    assert form(case) == "tiles 128" and torch.equal(case.run(tq), expected)
    assert status() == 0


def test_with_nothing_to_do(tq):
    case = Case(1, 4, 4, 2, 1, 300, 9, 64, 16)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    got = tq.prefix_attention(case.q[:0], *case.tensors, case.table[:0], case.lengths[:0], none)
    assert got.shape == (0, 4, 1, 64)
    assert tq.prefix_attention(case.q[:, :, :0], *case.tensors, case.table, case.lengths, case.shared).numel() == 0
    got = tq.prefix_attention(case.q, *case.tensors, case.table[:, :0], torch.zeros_like(case.lengths), case.shared)
    assert not got.any()
    assert status() == 0


def test_the_custom_operation(tq):
    tq.register_custom_ops()
    case = Case(*KINDS[2])
    got = torch.ops.tessiq.prefix_attention(case.q, *case.tensors, case.table, case.lengths, case.shared, None)
    assert torch.equal(got, case.run(tq)) and status() == 0


def test_a_plan_without_a_gpu_is_that_of_one(tq):
    """Device -1 stands for a B200: the way a call takes and the scratch it asks for, of paged and of dense keys, by extents drawn at random."""
    import random

    from tessiq_b200 import _lib

    rng = random.Random(3)

    def plan(device, extents, group, window):
        batch, heads, kv_heads, q_tokens, width, page, blocks, runs = extents
        way, size, sizes = [ctypes.c_int32() for _ in range(3)], ctypes.c_size_t(), []
        _lib.check(_lib.lib.tq_prefix_attention_form(*extents, device, *[ctypes.byref(n) for n in way]))
        for function, given in ((_lib.lib.tq_prefix_attention_workspace_bytes, extents), (_lib.lib.tq_cache_attention_workspace_bytes, (*extents[:7], window, 0)),
                                (_lib.lib.tq_window_attention_workspace_bytes, (batch, heads, kv_heads, q_tokens, page * blocks, width, window, 0))):
            _lib.check(function(*given, device, ctypes.byref(size)))
            sizes.append(size.value)
        return [n.value for n in way], sizes

    for _ in range(4000):
        runs, each, kv_heads, group = rng.choice([1, 1, 2, 3, 8, 16]), rng.choice([1, 2, 4, 7, 16, 64]), rng.choice([1, 2, 8, 12]), rng.choice([1, 2, 4, 8])
        extents = (runs * each, kv_heads * group, kv_heads, rng.choice([1, 1, 1, 2, 4]), rng.choice([64, 128, 32, 96]), rng.choice([16, 64, 128]), rng.randint(1, 400), runs)
        window = rng.choice([0, 0, 1000])
        assert plan(-1, extents, group, window) == plan(0, extents, group, window), extents


@pytest.mark.parametrize("extents", [(7, 8, 2, 4, 32, 128, 1961, 1), (56, 16, 2, 2, 128, 16, 333, 8), (64, 12, 12, 1, 64, 64, 64, 16)], ids=str)
def test_a_pool_of_no_pages(tq, extents):
    """Sequences of no tokens: zeros, as from cache_attention."""
    batch, heads, kv_heads, q_tokens, width, page, blocks, runs = extents
    codes, scales = torch.empty(0, kv_heads, page, width, dtype=E4M3, device="cuda"), torch.empty(0, kv_heads, device="cuda")
    table, lengths = torch.zeros(batch, blocks, dtype=torch.int32, device="cuda"), torch.zeros(batch, dtype=torch.int32, device="cuda")
    q = torch.randn(batch, heads, q_tokens, width, device="cuda").bfloat16()
    for shared in (0, 4096):
        out = tq.prefix_attention(q, codes, codes, scales, scales, table, lengths, torch.full((runs,), shared, dtype=torch.int32, device="cuda"))
        assert out.shape == q.shape and not out.any() and status() == 0


@pytest.mark.parametrize("which", range(len(KINDS)))
def test_a_scale_that_is_no_number_behind_pages_that_are_not_there(tq, which):
    """Of the shared keys one page is left, whose keys' scale is NaN in one head: that head's queries see it, whatever is missing before and behind it."""
    case = Case(*KINDS[which])
    shared = int(case.shared[0]) // case.page
    at = max(1, 64 // case.page)
    left = case.table[:, at].clone()
    case.table[:, :shared] = -1
    case.table[:, at] = left
    case.scales[0][left.long(), 0] = math.nan
    got, group = case.run(tq), case.heads // case.kv_heads
    assert status() == 0x50414745
    assert got[:, :group].isnan().all() and not got[:, group:].isnan().any()
