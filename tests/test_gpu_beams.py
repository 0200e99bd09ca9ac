"""Beam search's selection, the books of the cache on the device, and a search that uses both with the cache, against plain forms: values in 64 bits
(a selected value is rounded to f32 once, 2^-24 of it, after sums that are off by 1e-6 at most), numbers exact."""

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


# ---- selection -----------------------------------------------------------------------------------


def selected(logits, scores, keep, finished=None, end=0):
    """(values in f64, parents, tokens) of the definition."""
    requests, beams, vocab = logits.shape
    x = logits.double()
    total = x - torch.logsumexp(x, -1, keepdim=True) + scores.double()[..., None]
    broken = x.isnan().any(-1) | (x == math.inf).any(-1) | scores.isnan() | (scores == math.inf)
    nothing = ((x == -math.inf).all(-1) | (scores == -math.inf)) & ~broken
    total = torch.where(nothing[..., None], -math.inf, total)
    if finished is not None:
        stays = torch.where(torch.arange(vocab, device=x.device) == end, scores.double()[..., None], -math.inf).expand(total.shape)
        total = torch.where(finished[..., None], stays, total)
        broken = torch.where(finished, scores.isnan() | (scores == math.inf), broken)
    total = torch.where(broken[..., None], math.nan, total)
    values, index = torch.sort(total.flatten(1), dim=1, descending=True, stable=True)
    values, index = values[:, :keep], index[:, :keep]
    return values, index // vocab + torch.arange(requests, device=x.device)[:, None] * beams, index % vocab


def check(tq, logits, scores, keep, finished=None, end=0):
    got = tq.beam_select(logits, scores, keep, finished, end)
    values, parents, tokens = selected(logits, scores, keep, finished, end)
    assert [t.dtype for t in got] == [torch.float32, torch.int32, torch.int32]
    assert torch.equal(got[1].long(), parents) and torch.equal(got[2].long(), tokens)
    finite = values.isfinite()
    assert torch.equal(got[0].isnan(), values.isnan()) and torch.equal(got[0][~finite & ~values.isnan()].double(), values[~finite & ~values.isnan()])
    assert ((got[0].double() - values)[finite].abs() <= values[finite].abs() * 2.0**-24 + 1e-6).all()
    return got


def drawn(shape, dtype, seed=0, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * spread).to(dtype), -torch.rand(shape[:2], generator=g, device="cuda") * 5


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (1, 2, 2, 3), (3, 1, 7, 7), (1, 3, 33, 40), (2, 4, 255, 8), (1, 128, 300, 128), (5, 7, 4095, 14), (3, 4, 4088, 64), (2, 4, 4097, 5),
                                   (1, 4, 8184, 4), (1, 4, 8185, 128), (2, 3, 8192, 31), (3, 5, 16369, 33), (1, 4, 50257, 4), (64, 4, 50257, 8), (700, 1, 1000, 2), (2, 16, 128000, 32),
                                   (3, 128, 9000, 100), (1, 1, 1000003, 128), (600, 2, 33333, 4)], ids=str)
def test_beam_select(tq, shape, dtype):
    requests, beams, vocab, keep = shape
    logits, scores = drawn((requests, beams, vocab), dtype)
    check(tq, logits, scores, keep)
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
def test_rows_at_any_place(tq, dtype):
    """Logits out of a larger tensor: rows that begin at any element, strides of requests and beams, a beam that is all beams."""
    base, scores = drawn((3, 4, 9111), dtype)
    for offset in range(9):
        check(tq, base[:, :, offset : offset + 9001], scores, 8)
    check(tq, base.transpose(0, 1), scores.t().contiguous(), 8)
    check(tq, base[:, 1:2].expand(3, 4, 9111), scores, 8)
    check(tq, base[::2, ::3], scores[::2, ::3].contiguous(), 8)


@pytest.mark.parametrize("vocab", [5, 1000, 8192, 30000, 200000])
def test_equal_and_hidden_logits(tq, vocab):
    """Ties go to the lower beam and token: equal logits, masks that leave few tokens, one, or none, beams that are not there."""
    scores = torch.tensor([[-1.0, -1.0, -1.0], [-2.0, -1.0, -3.0]], device="cuda")
    logits = torch.zeros(2, 3, vocab, device="cuda")
    check(tq, logits, scores, 5)
    check(tq, logits, scores, min(128, 3 * vocab))
    for few in (1, 3):
        hidden = torch.full((2, 3, vocab), -math.inf, device="cuda")
        hidden[:, :, vocab - few :] = torch.randn(2, 3, few, device="cuda")
        check(tq, hidden, scores, 4)
        check(tq, hidden.bfloat16(), scores, min(20, 3 * vocab))
        hidden[0, 1] = -math.inf
        hidden[1] = -math.inf
        check(tq, hidden, scores, min(20, 3 * vocab))
    logits, _ = drawn((2, 3, vocab), torch.float32)
    scores = torch.tensor([[-1.0, -math.inf, -math.inf], [-math.inf, -math.inf, -math.inf]], device="cuda")
    check(tq, logits, scores, min(20, 3 * vocab))
    assert status() == 0


@pytest.mark.parametrize("vocab", [700, 8192, 50257, 200001])
def test_logits_in_rising_and_falling_order(tq, vocab):
    """Every chunk of a rising row is above all before it; sums that a later chunk carries beyond f32, or that a first chunk of large numbers would hide."""
    rising = torch.linspace(-30, 30, vocab, device="cuda")
    logits = torch.stack([rising, rising.flip(0), rising * 20, rising * -20])[None].contiguous()
    check(tq, logits, torch.tensor([[-1.0, -2.0, -1.5, -0.5]], device="cuda"), 16)
    steps = torch.full((1, 2, vocab), -300.0, device="cuda")
    steps[0, 0, vocab // 2 :] = 300.0 + torch.randn(vocab - vocab // 2, device="cuda")
    steps[0, 1, : vocab // 2] = -math.inf
    check(tq, steps, torch.tensor([[-1.0, -1.0]], device="cuda"), 8)
    huge = torch.randn(1, 3, vocab, device="cuda") * 1e30
    check(tq, huge, torch.zeros(1, 3, device="cuda"), 3)


def test_numbers_that_are_none(tq):
    logits, scores = drawn((6, 3, 20000), torch.float32)
    logits[0, 1, 15000] = math.nan
    logits[1, 2, 3] = math.inf
    scores[2, 0] = math.nan
    scores[3, 1] = math.inf
    logits[4, :, 7] = -math.inf
    scores[5, 0] = -math.inf
    logits[5, 0, 3] = math.nan
    check(tq, logits, scores, 10)
    check(tq, logits.bfloat16(), scores, 1)


# Parts of several chunks: 160 rows of 60000 are three parts each, of three chunks of two-byte logits or five of f32; 600 rows are one part each.


def in_other_orders(row, beams, g, place=None):
    """[beams, vocab]: `row` in as many orders, its largest where place() says."""
    rows = torch.stack([row[torch.randperm(len(row), generator=g)] for _ in range(beams)])
    for beam in range(beams if place else 0):
        at, to = int(rows[beam].argmax()), place()
        rows[beam, at], rows[beam, to] = rows[beam, to].clone(), rows[beam, at].clone()
    return rows


def behind_a_first_chunk(g):
    return lambda: int(torch.randint(0, 3, (1,), generator=g)) * 20000 + int(torch.randint(10000, 20000, (1,), generator=g))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("above", [3, 10, 20, 25, 40, 65])
def test_a_token_far_above_its_parts_first_chunk(tq, above, dtype):
    """Two beams of the same logits in two orders, scores 1e-8 to 3e-6 apart, either way: which is better is their scores' alone."""
    g = torch.Generator().manual_seed(above)
    rows = torch.randn(80, 60000, generator=g)
    rows[:, 0] = 4 + above + 4 * torch.rand(80, generator=g)
    logits = torch.stack([in_other_orders(row, 2, g, behind_a_first_chunk(g)) for row in rows]).to(dtype).cuda()
    apart = 10.0 ** (torch.rand(80, generator=g) * 2.5 - 8) * torch.where(torch.rand(80, generator=g) < 0.5, -1, 1)
    check(tq, logits, torch.stack([torch.zeros(80), apart], 1).cuda(), 4)
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("allowed", [1, 2, 5, 40])
def test_few_tokens_allowed_behind_a_first_chunk(tq, allowed, dtype):
    """Masks that leave few tokens, none of a part's first chunk among them. A lone token's value is its beam's score as it is, so that ties go to the lower beam."""
    g = torch.Generator().manual_seed(allowed)
    for level in (-70.0, -1.0, 45.0):
        logits = torch.full((40, 4, 60000), -math.inf)
        for r in range(40):
            place, kept = behind_a_first_chunk(g), level + 15 * torch.rand(allowed, generator=g)
            for beam in range(4):
                places = {place() for _ in range(3 * allowed + 9)}
                logits[r, beam, torch.tensor(sorted(places))[torch.randperm(len(places), generator=g)[:allowed]]] = kept
        logits = logits.to(dtype).cuda()
        if allowed == 1:
            got = check(tq, logits, torch.full((40, 4), -1.25, device="cuda"), 4)
            assert (got[0] == -1.25).all()
        scores = -torch.rand(40, 4, generator=g).cuda()
        check(tq, logits, scores, 3)
        check(tq, logits, scores, 30)      # (more than are allowed, or some that are not)
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_parts_of_several_chunks(tq, dtype):
    """Rising and falling rows, steps, equal logits and masks, where chunks come one after another."""
    vocab = 33333
    rising = torch.linspace(-30, 30, vocab, device="cuda")
    step = torch.full((vocab,), -300.0, device="cuda")
    step[vocab // 2 :] = 300.0 + torch.randn(vocab - vocab // 2, generator=torch.Generator().manual_seed(1)).cuda()
    hidden = torch.randn(vocab, generator=torch.Generator().manual_seed(2)).cuda()
    hidden[: vocab // 2] = -math.inf
    huge = torch.randn(vocab, generator=torch.Generator().manual_seed(3)).cuda() * 1e30
    for row in (rising, rising.flip(0), rising * 20, rising * -20, step, step.flip(0), hidden, hidden.flip(0), huge, torch.full_like(rising, 0.25)):
        logits = torch.stack([row, torch.randn(vocab, generator=torch.Generator().manual_seed(4)).cuda()]).to(dtype)[None].expand(300, 2, vocab).contiguous()
        scores = -torch.arange(600, device="cuda").reshape(300, 2) / 64.0
        got = [t.cpu() for t in tq.beam_select(logits, scores, 9)]
        values, parents, tokens = [t.cpu() for t in selected(logits[:1], scores[:1], 9)]
        for r in range(300):      # (a request's scores are the first one's, less 2 r / 64)
            assert torch.equal(got[1][r] - 2 * r, parents[0].int()) and torch.equal(got[2][r], tokens[0].int())
            expected = values[0] - 2 * r / 64.0
            assert ((got[0][r].double() - expected).abs() <= expected.abs() * 2.0**-24 + 1e-6).all()
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_numbers_that_are_none_in_a_later_chunk(tq, dtype):
    logits, scores = drawn((80, 2, 60000), dtype, 11)
    place = behind_a_first_chunk(torch.Generator().manual_seed(12))
    for r in range(0, 80, 2):
        logits[r, r // 2 % 2, place()] = (math.nan, math.inf)[r // 4 % 2]
        if r % 3 == 0:
            logits[r, r // 2 % 2, :9000] = -math.inf
            logits[r, r // 2 % 2, 20000:29000] = -math.inf
            logits[r, r // 2 % 2, 40000:49000] = -math.inf
    check(tq, logits, scores, 7)
    assert status() == 0


def test_finished_beams(tq):
    logits, scores = drawn((4, 4, 5000), torch.bfloat16)
    finished = torch.tensor([[True, False, False, True], [True, True, True, True], [False, False, False, False], [False, True, True, True]], device="cuda")
    for end in (0, 3, 4999):
        for keep in (4, 8, 40):
            check(tq, logits, scores, keep, finished, end)
    logits[0, 0] = math.nan      # (a finished beam's logits are not looked at)
    scores[1, 2] = -math.inf
    check(tq, logits, scores, 8, finished, 17)
    assert status() == 0


def test_values_that_are_close(tq):
    """Beams whose values differ by less than f32 sums of exponentials can tell: the same logits in another order, scores a few 1e-8 apart, either way."""
    logits, _ = drawn((40, 2, 60000), torch.float32)
    for r in range(40):
        logits[r, 1] = logits[r, 0][torch.randperm(60000, generator=torch.Generator().manual_seed(r)).cuda()]
    apart = (torch.arange(40, device="cuda") - 20).float() * 3e-9
    scores = torch.stack([torch.zeros(40, device="cuda"), apart], 1)
    check(tq, logits, scores, 6)
    same = logits.clone()
    same[:, 1] = same[:, 0]
    check(tq, same, torch.zeros_like(scores), 6)      # (beams of one sum: ties, to the lower beam)


def test_roundings_that_add_up(tq):
    """One token over a background of equal logits, whose exponents are all rounded the same way: two beams of other distances whose values are within 1e-7 or
    less of each other, either way."""
    g = torch.Generator().manual_seed(6)
    top = (8 + 1.5 * torch.rand(300, 2, generator=g)).cuda()
    low = torch.exp2(-1 - 12 * torch.rand(300, 2, generator=g)).cuda()
    logits = low[:, :, None].expand(300, 2, 50257).contiguous()
    logits[:, :, 30000] = top
    value = -torch.log1p(50256 * torch.exp(low.double() - top.double()))
    scores = torch.zeros(300, 2, device="cuda")
    scores[:, 1] = value[:, 0] - value[:, 1] + (torch.rand(300, generator=g).cuda() - 0.5) * 2e-7
    values = scores.double() + value
    got = tq.beam_select(logits, scores, 2)
    best = (values[:, 1] > values[:, 0]).int()
    rows = torch.arange(300, device="cuda", dtype=torch.int32) * 2
    assert torch.equal(got[1], torch.stack([rows + best, rows + 1 - best], 1)) and (got[2] == 30000).all()
    assert ((got[0].double() - values.sort(dim=1, descending=True).values).abs() <= 2.0**-24 + 2e-12 + 1e-6).all() and status() == 0


def test_beams_whose_sums_round_to_the_same(tq):
    """Backgrounds that are neighbours in f32, and whose exponents, times log2 e, are the same number: the sums are equal to the last bit and the values are not."""
    log2_e, low = torch.tensor(math.log2(math.e)), torch.tensor(-1.5)
    pairs = []
    while len(pairs) < 40:
        lower = torch.nextafter(low, torch.tensor(-2.0))
        if torch.equal(low * log2_e, lower * log2_e):
            pairs.append((low.item(), lower.item()))
        low = lower
    for vocab in (100, 3000, 20000):
        logits = torch.tensor(pairs, device="cuda")[:, :, None].repeat(1, 1, vocab)
        logits[:, :, vocab // 3] = 0.0
        for first, second in ((logits[:, 0], logits[:, 1]), (logits[:, 1], logits[:, 0])):
            check(tq, torch.stack([first, second], 1), torch.full((40, 2), -2.0, device="cuda"), 3)
    # more such values than a list has: 1500 zeros of each of 64 beams over one background, and over its neighbour in the last beam, the best
    high = torch.rand(3001, generator=torch.Generator().manual_seed(3)) < 0.5
    logits = torch.where(high, 0.0, pairs[0][0]).expand(2, 64, 3001).clone()
    logits[:, 63] = torch.where(high, 0.0, pairs[0][1])
    got = tq.beam_select(logits.cuda(), torch.full((2, 64), -1.25, device="cuda"), 64)
    assert got[1].tolist() == [[63] * 64, [127] * 64] and got[2].tolist() == [high.nonzero()[:64, 0].tolist()] * 2
    # ... and of a beam beside a finished one, whose score is that beam's value or a little off
    logits = torch.where(torch.rand(60000, generator=torch.Generator().manual_seed(4)) < 0.5, 0.0, pairs[0][0]).expand(40, 2, 60000).contiguous()
    total = torch.logsumexp(logits[0, 0].double(), 0)
    value = total.float().double() - total
    scores = torch.stack([total.float().expand(40), (value + torch.linspace(-4e-7, 4e-7, 40, dtype=torch.float64)).float()], 1)
    got = tq.beam_select(logits.cuda(), scores.cuda(), 128, torch.tensor([[False, True]] * 40, device="cuda"), 5)
    for r in range(40):
        first = scores[r, 1].double() > value
        assert got[1][r].tolist() == [2 * r + 1] * first + [2 * r] * (128 - int(first))
    assert status() == 0


@pytest.mark.parametrize("shape", [(1, 1, 2**24 - 1, 128), (65535, 1, 3, 2), (511, 128, 2, 128), (2, 128, 1, 128)], ids=str)
def test_selection_at_its_limits(tq, shape):
    requests, beams, vocab, keep = shape
    check(tq, *drawn((requests, beams, vocab), torch.float16, spread=4.0), keep)
    assert status() == 0


def test_beams_that_are_alike(tq):
    """All values of a request's beams are equal in pairs or more, so that every sum is taken again."""
    logits, _ = drawn((3, 1, 5000), torch.bfloat16)
    for scores in (torch.zeros(3, 48, device="cuda"), torch.arange(48, device="cuda").div(7, rounding_mode="floor").float().expand(3, 48).contiguous()):
        check(tq, logits.expand(3, 48, 5000), scores, 96)
        check(tq, logits.expand(3, 48, 5000).contiguous(), scores, 96)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
def test_more_equal_values_than_a_list_has(tq, dtype):
    """Beams that are alike at addresses that are not: thousands of equal values, of which the lowest beam's first tokens are the best."""
    g = torch.Generator().manual_seed(3)
    for vocab, beams, keep in ((3001, 64, 64), (50257, 128, 30), (777, 128, 128)):
        high = torch.rand(vocab, generator=g) < 0.5
        logits = torch.where(high, 1.1, 0.3).to(dtype).cuda().expand(2, beams, vocab).contiguous()
        scores = torch.full((2, beams), -1.25, device="cuda")
        scores[1, 0] = -1.3125                                # (its first beam is worse, the second the best)
        got = tq.beam_select(logits, scores, keep)
        assert got[1].tolist() == [[0] * keep, [beams + 1] * keep]
        assert got[2].tolist() == [high.nonzero()[:keep, 0].tolist()] * 2 and status() == 0


def test_selection_in_graphs_and_on_streams(tq):
    logits, scores = drawn((8, 4, 30000), torch.bfloat16)
    expected = check(tq, logits, scores, 8)
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for stream in streams:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(tq.beam_select(logits, scores, 8))
        graphs.append(graph)
    for turn in range(3):
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, expected))
        logits.copy_(drawn((8, 4, 30000), torch.bfloat16, 100 + turn)[0])
        expected = check(tq, logits, scores, 8)
    tq.register_custom_ops()
    assert all(torch.equal(a, b) for a, b in zip(torch.ops.tessiq.beam_select(logits, scores, 8, None, 0), expected))


def test_selection_recorded(tq):
    from tessiq_b200 import _lib

    logits, scores = drawn((3, 4, 30000), torch.float16)
    handle = ctypes.c_void_p()
    _lib.check(_lib.lib.tq_recipe_create(ctypes.byref(handle)))
    _lib.check(_lib.lib.tq_recipe_begin_recording(handle))
    out = tq.beam_select(logits, scores, 5)
    _lib.check(_lib.lib.tq_recipe_end_recording(handle))
    _lib.check(_lib.lib.tq_recipe_run(handle, 0, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, tq.beam_select(logits, scores, 5)))
    _lib.check(_lib.lib.tq_recipe_destroy(handle))


def test_selection_with_nothing_to_do(tq):
    logits, scores = drawn((2, 3, 10), torch.float32)
    assert [t.shape for t in tq.beam_select(logits[:0], scores[:0], 4)] == [(0, 4)] * 3
    assert [t.shape for t in tq.beam_select(logits, scores, 0)] == [(2, 0)] * 3


# ---- books on the device -------------------------------------------------------------------------


class Books:
    """A pool, a table and counts, and the same books on the host, a page at a time."""

    def __init__(self, rows, blocks, pages, page, layers=2, kv_heads=2, width=16, seed=0, stride=0):
        g = torch.Generator().manual_seed(seed)
        self.page, self.rows, self.blocks, self.pages = page, rows, blocks, pages
        shape = (layers, pages, kv_heads, page, width)
        self.codes = [torch.randint(0, 120, shape, generator=g, dtype=torch.uint8).cuda().view(E4M3) for _ in range(2)]
        self.scales = [torch.rand(shape[:3], generator=g).cuda() for _ in range(2)]
        self.wide = torch.full((rows, blocks + stride), -7, dtype=torch.int32, device="cuda")
        self.table = self.wide[:, :blocks]
        self.lengths = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.references = torch.zeros(pages, dtype=torch.int32, device="cuda")

    @property
    def pools(self):
        return (*self.codes, *self.scales)

    def host(self, counts, parents):
        """What a step makes of the books: (table, lengths, references, starts, copies), or the code that is reported where it cannot be made."""
        page, table, lengths, references = self.page, self.table.tolist(), self.lengths.tolist(), self.references.tolist()
        old = [row[: -(-n // page)] for row, n in zip(table, lengths)]
        rows = [list(old[p]) if p >= 0 else [] for p in parents]
        starts = [lengths[p] if p >= 0 else 0 for p in parents]
        for row in rows:
            for p in row:
                references[p] += 1
        for row in old:
            for p in row:
                references[p] -= 1
        free, pairs = iter([p for p, n in enumerate(references) if n == 0]), []
        if any(start + max(count, 0) > self.blocks * page for start, count in zip(starts, counts)):
            return 0x4C454E47
        try:
            for row, start, count in zip(rows, starts, counts):
                if count > 0 and start % page and references[row[-1]] > 1:
                    references[row[-1]] -= 1
                    pairs.append((row[-1], next(free)))
                    row[-1] = pairs[-1][1]
                    references[row[-1]] = 1
                while len(row) * page < start + max(count, 0):
                    row.append(next(free))
                    references[row[-1]] = 1
        except StopIteration:
            return 0x46554C4C
        now = [row + before[len(row) :] for row, before in zip(rows, table)]
        return now, [a + max(c, 0) for a, c in zip(starts, counts)], references, starts, pairs

    def step(self, tq, counts, parents=None, in_place=False, fault=None):
        expected = self.host(counts, list(range(self.rows)) if parents is None else parents) if fault is None else fault
        fault = expected if isinstance(expected, int) else 0
        before = [t.clone() for t in (self.table, self.lengths, self.references, *self.pools)]
        there = [None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (counts, parents)]
        got = tq.cache_advance(*self.pools, self.table, self.lengths, self.references, *there, in_place)
        assert status() == fault
        if in_place:
            assert got[0] is self.table and got[1] is self.lengths and got[2] is self.references
        else:
            assert all(torch.equal(a, b) for a, b in zip((self.table, self.lengths, self.references), before))
        if fault:
            assert all(torch.equal(a, b) for a, b in zip(got[:3], before)) and (got[3] == -1).all()
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(self.pools, before[3:]))
            return
        assert [t.tolist() for t in got] == list(expected[:4])
        for pool, was in zip(self.pools, before[3:]):
            for a, b in expected[4]:
                was.view(torch.uint8)[:, b] = was.view(torch.uint8)[:, a]
            assert torch.equal(pool.view(torch.uint8), was.view(torch.uint8))
        if not in_place:
            self.table.copy_(got[0]), self.lengths.copy_(got[1]), self.references.copy_(got[2])
        assert (self.wide[:, self.blocks :] == -7).all()
        return expected


BOOKS = [  # rows, blocks, pages, page, steps
    (1, 1, 1, 16, 3), (3, 4, 20, 16, 25), (8, 5, 60, 32, 30), (64, 33, 2500, 16, 12), (200, 7, 1600, 64, 10), (40, 100, 20000, 16, 8), (1500, 12, 18100, 16, 5), (33, 1000, 33500, 16, 4),
    (5000, 4, 20100, 128, 3),
]


@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in place"])
@pytest.mark.parametrize("case", BOOKS, ids=str)
def test_books_against_the_host(tq, case, in_place):
    """Steps in which rows go on from any rows, or from none, by counts of 0 to a few pages, in one CTA and in a cluster."""
    rows, blocks, pages, page, steps = case
    books = Books(rows, blocks, pages, page, stride=3, layers=1 if pages > 10000 else 2)
    g = torch.Generator().manual_seed(5)
    books.references[pages // 2] = 7                       # (others')
    for turn in range(steps):
        parents = torch.randint(-1 if turn else 0, rows, (rows,), generator=g).tolist() if turn % 3 else None
        longest = max(0, int(books.lengths.max()))
        most = max(0, min(2 * page + 3, (blocks * page - longest) if turn else blocks * page // 2))
        counts = torch.randint(0, most + 1, (rows,), generator=g)
        counts[torch.rand(rows, generator=g) < 0.3] = 0
        counts[torch.rand(rows, generator=g) < 0.3] = min(1, most)
        counts = counts.tolist()
        books.step(tq, counts, parents, in_place)


def filled(tq, rows=6, blocks=6, pages=30, page=16, **more):
    books = Books(rows, blocks, pages, page, **more)
    books.step(tq, [5 + 7 * i for i in range(rows)], None, True)
    return books


@pytest.mark.parametrize("large", [False, True], ids=["one CTA", "cluster"])
@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in place"])
def test_steps_that_cannot_be_made(tq, in_place, large):
    """Nothing changes, not the pools either, where pages, the table or a parent are missing; then steps go on."""
    books = filled(tq, pages=20000 if large else 30, layers=1)
    books.references[24:] = 3
    free = int((books.references == 0).sum())
    assert books.host([40] * 6, list(range(6))) == 0x46554C4C and books.host([0, 0, 0, 0, 0, 6 * 16], list(range(6))) == 0x4C454E47 and free < 18
    books.step(tq, [40] * 6, None, in_place)
    books.step(tq, [0, 0, 0, 0, 0, 6 * 16], None, in_place)
    books.step(tq, [1] * 6, [0, 1, 2, 3, 4, 6], in_place, 0x50415245)
    kept = books.table[2, 0].clone()
    for wrong in (-1, books.pages, 1 << 30):
        books.table[2, 0] = wrong
        before = [t.clone() for t in (books.table, books.lengths, books.references)]
        counts, flipped = torch.ones(6, dtype=torch.int32, device="cuda"), torch.arange(5, -1, -1, dtype=torch.int32, device="cuda")
        for parents in (None, flipped):
            got = tq.cache_advance(*books.pools, books.table, books.lengths, books.references, counts, parents, in_place)
            assert status() == 0x50414745 and (got[3] == -1).all()
            assert all(torch.equal(a, b) for a, b in zip(got, before)) and all(torch.equal(a, b) for a, b in zip((books.table, books.lengths, books.references), before))
    books.table[2, 0] = kept
    books.step(tq, [1, 0, 2, 0, 0, 1], [5, 5, 5, -1, 2, 2], in_place)
    books.step(tq, [-3, 0, 2, -1, 0, 1], None, in_place)


def test_one_layer_and_small_pools(tq):
    """A layer's own tensors, pages of one head, books out of larger tensors."""
    books = filled(tq)
    one = [t[1] for t in books.pools]
    counts, parents = torch.ones(6, dtype=torch.int32, device="cuda"), torch.tensor([5, 5, 5, 1, 2, 2], dtype=torch.int32, device="cuda")
    expected = tq.cache_advance(*books.pools, books.table, books.lengths, books.references, counts, parents)
    got = tq.cache_advance(*one, books.table, books.lengths, books.references, counts, parents)
    assert all(torch.equal(a, b) for a, b in zip(got, expected)) and status() == 0
    odd = torch.zeros(31, dtype=torch.int32, device="cuda")[1:]
    odd.copy_(books.references)
    got = tq.cache_advance(*books.pools, books.table, books.lengths, odd, counts, parents)
    assert all(torch.equal(a, b) for a, b in zip(got, expected))
    got = tq.cache_advance(*books.pools, books.table.clone(), books.lengths.clone(), odd, counts, parents, True)
    assert torch.equal(got[2], expected[2]) and got[2] is odd and status() == 0


def test_a_cluster_s_advance_in_a_graph(tq):
    a, b = (Books(3001, 6, 27009, 16, seed=4) for _ in range(2))
    for books in (a, b):
        books.step(tq, [5 + i % 60 for i in range(books.rows)], None, True)
    counts, parents = torch.ones(3001, dtype=torch.int32, device="cuda"), torch.arange(3001, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        starts = tq.cache_advance(*a.pools, a.table, a.lengths, a.references, counts, parents, True)[3]
    for turn in range(3):
        parents.copy_(torch.randint(0, 3001, (3001,), generator=torch.Generator().manual_seed(turn)))
        graph.replay()
        expected = tq.cache_advance(*b.pools, b.table, b.lengths, b.references, counts, parents, True)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((a.table, a.lengths, a.references, starts), expected))
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a.pools, b.pools))
    assert status() == 0


def test_advances_on_two_streams(tq):
    """Steps of two caches at once, of a CTA and of a cluster each, give what they give one after another."""
    sides = []
    for _ in range(2):
        sides.append([Books(rows, 6, 9 * rows, 16, seed=rows) for rows in (40, 3001, 41, 3002)])
        for books in sides[-1]:
            books.step(tq, [5 + i % 60 for i in range(books.rows)], None, True)
    streams = [torch.cuda.Stream() for _ in range(4)]
    for turn in range(5):
        given = []
        for n, (apart, alone) in enumerate(zip(*sides)):
            g = torch.Generator().manual_seed(10 * turn + n)
            parents = torch.randint(0, apart.rows, (apart.rows,), generator=g).int().cuda()
            counts = torch.randint(0, 3, (apart.rows,), generator=g).int().cuda()
            torch.cuda.synchronize()
            tq.cache_advance(*alone.pools, alone.table, alone.lengths, alone.references, counts, parents, True)
            given.append((counts, parents))
        torch.cuda.synchronize()
        for stream, apart, numbers in zip(streams, sides[0], given):
            with torch.cuda.stream(stream):
                tq.cache_advance(*apart.pools, apart.table, apart.lengths, apart.references, *numbers, True)
        torch.cuda.synchronize()
        assert status() == 0
    for apart, alone in zip(*sides):
        assert all(torch.equal(x, y) for x, y in zip((apart.table, apart.lengths, apart.references), (alone.table, alone.lengths, alone.references)))
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(apart.pools, alone.pools))


def test_no_rows_and_no_blocks(tq):
    books = filled(tq)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    got = tq.cache_advance(*books.pools, books.table[:0], none, books.references, none)
    assert got[0].shape == (0, 6) and torch.equal(got[2], books.references) and got[2] is not books.references
    got = tq.cache_advance(*books.pools, books.table[:, :0], torch.zeros(6, dtype=torch.int32, device="cuda"), books.references, torch.zeros(6, dtype=torch.int32, device="cuda"))
    assert got[0].shape == (6, 0) and torch.equal(got[2], books.references) and not got[3].any() and status() == 0


def test_advance_in_graphs_and_recorded(tq):
    from tessiq_b200 import _lib

    a, b = filled(tq, pages=60), filled(tq, pages=60)
    counts, parents = torch.ones(6, dtype=torch.int32, device="cuda"), torch.tensor([0, 0, 2, 2, 4, 4], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        starts = tq.cache_advance(*a.pools, a.table, a.lengths, a.references, counts, parents, True)[3]
    for turn in range(4):
        parents.copy_(torch.tensor([[0, 0, 2, 2, 4, 4], [1, 0, 3, 2, 5, 4], [5, 5, 5, 5, 5, 5], [0, 1, 2, 3, 4, -1]][turn]))
        graph.replay()
        expected = tq.cache_advance(*b.pools, b.table, b.lengths, b.references, counts, parents, True)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((a.table, a.lengths, a.references, starts), expected))
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a.pools, b.pools))
    handle = ctypes.c_void_p()
    _lib.check(_lib.lib.tq_recipe_create(ctypes.byref(handle)))
    _lib.check(_lib.lib.tq_recipe_begin_recording(handle))
    recorded = tq.cache_advance(*a.pools, a.table, a.lengths, a.references, counts, parents)
    _lib.check(_lib.lib.tq_recipe_end_recording(handle))
    _lib.check(_lib.lib.tq_recipe_run(handle, 0, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(recorded, tq.cache_advance(*b.pools, b.table, b.lengths, b.references, counts, parents)))
    _lib.check(_lib.lib.tq_recipe_destroy(handle))
    assert status() == 0


# ---- together ------------------------------------------------------------------------------------


def decoded(cache, layer, table_row, length):
    """[2, kv_heads, length, width] in f64: a row's keys and values as the cache has them."""
    page = cache.books.page_tokens
    pages = table_row[: -(-length // page)].long()
    both = []
    for codes, scales in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)):
        x = codes[layer].view(torch.uint8)[pages].view(E4M3).double() * scales[layer][pages].double()[..., None, None]
        both.append(x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :length])
    return torch.stack(both)


@pytest.mark.parametrize("captured", [False, True], ids=["eager", "captured"])
def test_a_search(tq, captured):
    """Two prompts, four beams each, forty steps: selection, books, store and attention of two layers, all on the device, or in a graph. Each row's cache has to be
    what its own tokens give, and attention what the definition gives of that; then beams become sequences and the rest goes back."""
    from tessiq_b200.cache import PagedCache

    layers, kv_heads, heads, width, vocab, beams, page = 2, 2, 4, 32, 997, 4, 16
    g = torch.Generator().manual_seed(11)
    k_of, v_of = (torch.randn(layers, vocab, kv_heads, width, generator=g).bfloat16().cuda() for _ in range(2))      # of a token
    q_of = torch.randn(layers, vocab, heads, width, generator=g).bfloat16().cuda()
    out_of = torch.randn(heads * width, vocab, generator=g).cuda()
    cache = PagedCache(layers, kv_heads, width, 400, page)
    prompts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (301, 144)]
    sequences = [cache.start() for _ in prompts]
    for sequence, prompt in zip(sequences, prompts):
        step = cache.extend([sequence], len(prompt))
        at = torch.tensor(prompt, device="cuda")
        for layer in range(layers):
            cache.store(step, layer, k_of[layer, at].transpose(0, 1)[None], v_of[layer, at].transpose(0, 1)[None])
    free_before = cache.books.free_pages
    search = cache.beams(sequences, beams, 41)
    with pytest.raises(RuntimeError, match="compact"):
        cache.compact()
    rows = search.rows
    scores = torch.zeros(2, beams, device="cuda")
    scores[:, 1:] = -math.inf
    parents, tokens = torch.arange(rows, dtype=torch.int32, device="cuda").reshape(2, beams), torch.tensor([p[-1] for p in prompts for _ in range(beams)], device="cuda").int().reshape(2, beams)
    attended = [torch.zeros(rows, heads, 1, width, device="cuda", dtype=torch.bfloat16) for _ in range(layers)]

    def go_on():
        step = search.step(parents)
        at = tokens.reshape(-1).long()
        for layer in range(layers):
            cache.store(step, layer, k_of[layer, at][:, :, None], v_of[layer, at][:, :, None])
            attended[layer].copy_(cache.attention(step, layer, q_of[layer, at][:, :, None]))
        logits = (attended[0] + attended[1]).float().reshape(2, beams, heads * width) @ out_of * 3.0
        chosen = tq.beam_select(logits, scores, beams)
        scores.copy_(chosen[0]), parents.copy_(chosen[1]), tokens.copy_(chosen[2])

    histories = [list(p) for p in prompts for _ in range(beams)]
    graph = None
    for turn in range(40):
        histories = [histories[p] + [t] for p, t in zip(parents.reshape(-1).tolist(), tokens.reshape(-1).tolist())]
        fed = tokens.reshape(-1).tolist()
        if captured and turn == 2:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                go_on()
        graph.replay() if graph is not None else go_on()
        if turn in (0, 1, 2, 15, 16, 17, 39):
            assert search.lengths.tolist() == [len(h) for h in histories]
            for row, history in enumerate(histories):
                for layer in range(layers):
                    have = decoded(cache, layer, search.table[row], len(history))
                    at = torch.tensor(history, device="cuda")
                    want = torch.stack([k_of[layer, at], v_of[layer, at]]).transpose(1, 2).double()
                    # e4m3 rounds by 2^-4 of a number, or by half of 2^-9 of the scale, which is at most max / 224; encoded again, once more for each time the scale grew
                    assert ((have - want).abs() <= want.abs() * 2.0**-4 + want.abs().max() / 224 * 2.0**-9).all()
                    q = q_of[layer, fed[row]].double().reshape(kv_heads, heads // kv_heads, width)
                    exact = (torch.softmax(q @ have[0].transpose(1, 2) / math.sqrt(width), -1) @ have[1]).reshape(heads, width)
                    # half a step of bf16 and of the probabilities' f16, and what f32 sums of scores of about 10 and less leave
                    spread = have[1].abs().amax(1).repeat_interleave(heads // kv_heads, 0)
                    assert ((attended[layer][row, :, 0].double() - exact).abs() <= exact.abs() * 2.0**-8 + spread * (2.0**-11 + 2.0**-16)).all()
    assert status() == 0
    if captured:      # (the graph was replayed where the search had two steps already: a step of it is the newest)
        return search.free()
    with pytest.raises(ValueError, match="over"):
        cache.store(stale(search), 0, k_of[0, :rows][:, :, None], v_of[0, :rows][:, :, None])
    best = [search.keep(0), search.keep(3), search.keep(beams)]
    for sequence, row in zip(best, (0, 3, beams)):
        assert cache.length(sequence) == len(histories[row])
        assert torch.equal(decoded(cache, 1, torch.tensor(cache.books.pages_of(sequence), device="cuda"), len(histories[row])), decoded(cache, 1, search.table[row], len(histories[row])))
    cache.free(sequences[1])
    search.free()
    with pytest.raises(ValueError, match="freed"):
        search.step()
    kept = [decoded(cache, 0, torch.tensor(cache.books.pages_of(s), device="cuda"), cache.length(s)) for s in best]
    cache.compact()
    step = cache.extend(best, 1)
    assert all(torch.equal(decoded(cache, 0, step.table[i], kept[i].shape[2]), kept[i]) for i in range(3))
    for sequence in (*best, sequences[0]):
        cache.free(sequence)
    assert cache.books.free_pages == 400 and free_before < 400 and status() == 0


def stale(search):
    old = search.step(None, 0)
    search.step(None, 0)
    return old


def test_a_search_that_is_longer_than_it_said(tq):
    from tessiq_b200.cache import PagedCache
    from tessiq_b200.kernel import DeviceWaitError, check_status

    cache = PagedCache(1, 1, 16, 20, 16)
    a = cache.start()
    step = cache.extend([a], 20)
    x = torch.randn(1, 1, 20, 16, device="cuda").bfloat16()
    cache.store(step, 0, x, x)
    search = cache.beams([a], 3, 12)
    search.step(torch.tensor([0, 0, 0], dtype=torch.int32, device="cuda"), 12)
    check_status()
    before = search.table.clone()
    step = search.step(None, 1)
    codes = cache.k_pages.clone()
    cache.store(step, 0, torch.ones(3, 1, 1, 16, device="cuda").bfloat16(), torch.ones(3, 1, 1, 16, device="cuda").bfloat16())
    assert torch.equal(search.table, before) and search.lengths.tolist() == [32] * 3 and torch.equal(cache.k_pages.view(torch.uint8), codes.view(torch.uint8))
    with pytest.raises(DeviceWaitError, match="was not made|longer"):
        check_status()
    with pytest.raises(MemoryError):
        cache.beams([a], 3, 100)
    search.free()
    assert cache.books.free_pages == 18


def test_forks_of_a_prompt_read_it_once(tq):
    """The host's books find out what the sequences of a step have in common; the result is the same attention."""
    from tessiq_b200.cache import PagedCache

    cache = PagedCache(1, 2, 64, 600, 16)
    a = cache.start()
    step = cache.extend([a], 2000)
    x = torch.randn(2, 1, 2, 2000, 64, device="cuda").bfloat16()
    cache.store(step, 0, x[0], x[1])
    rows = [cache.fork(a) for _ in range(24)]
    step = cache.extend(rows, 1, runs=1)
    assert step.shared.tolist() == [2000 // 16 * 16]
    new = torch.randn(2, 24, 2, 1, 64, device="cuda").bfloat16()
    cache.store(step, 0, new[0], new[1])
    q = torch.randn(24, 8, 1, 64, device="cuda").bfloat16()
    got, alone = cache.attention(step, 0, q), tq.cache_attention(q, *cache.layer(0), step.table, step.lengths)
    # each is off by half a step of bf16 and of f16 probabilities of values of at most 6
    assert (got.double() - alone.double()).abs().max() <= 2 * (2.0**-8 * alone.double().abs().max() + 2.0**-11 * 6)
    assert torch.equal(cache.attention(step, 0, q, window=100), tq.cache_attention(q, *cache.layer(0), step.table, step.lengths, 100))
    assert status() == 0


def test_a_row_that_is_kept_while_the_others_go_on(tq):
    """What a kept sequence has stays as it is while the rows write, part and leave pages behind, and while it is extended itself."""
    from tessiq_b200.cache import PagedCache

    g = torch.Generator().manual_seed(5)
    cache = PagedCache(1, 2, 32, 60, 16)
    a = cache.start()
    step = cache.extend([a], 37)
    x = torch.randn(1, 2, 37, 32, generator=g).bfloat16().cuda()
    cache.store(step, 0, x, -x)
    search = cache.beams([a], 4, 60)

    def go_on(parents):
        new = torch.randn(4, 2, 1, 32, generator=g).bfloat16().cuda()
        cache.store(search.step(torch.tensor(parents, dtype=torch.int32, device="cuda")), 0, new * 4, -new)

    for turn in range(9):
        go_on([0, 0, 1, 3] if turn % 3 == 0 else [0, 1, 2, 3])
    kept = search.keep(2)
    row = torch.tensor(cache.books.pages_of(kept), device="cuda")
    had = decoded(cache, 0, row, 46)
    for turn in range(20):      # (row 2 goes its own way first, then nobody has it)
        go_on([0, 1, 2, 3] if turn < 3 else [0, 0, 0, 0])
        assert torch.equal(decoded(cache, 0, row, 46), had)
    step = cache.extend([kept], 1)
    assert torch.equal(decoded(cache, 0, step.table[0], 46), had)
    rows = [decoded(cache, 0, search.table[r], 66) for r in range(4)]
    cache.store(step, 0, x[:, :, :1], x[:, :, :1])
    assert all(torch.equal(decoded(cache, 0, search.table[r], 66), rows[r]) for r in range(4))
    search.free()
    assert torch.equal(decoded(cache, 0, step.table[0], 32), had[:, :, :32]) and status() == 0      # (the store may have raised the last page's scale)
    cache.free(kept)
    cache.free(a)
    assert cache.books.free_pages == 60
