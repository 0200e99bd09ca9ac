"""The operators of a batch that shares its beginning, as cases: attention over a paged cache whose sequences have a long prefix in
common, beam search's selection over beams and vocabulary, and the tables of the cache built on the GPU as beams are reordered and grow.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs and the cache's tensors, on the GPU
    run(state)          one pass: the plain form in torch, or with `own` the call of the library's operator
    work(case)          bytes and flops that a pass cannot do without
    exact(case, seed)   the outputs of a pass in 64 bits, from the definition

The cache is the library's: pages of `page` tokens, [pages, kv_heads, page, width] in e4m3, an f32 scale a page and head, a table row of
page numbers for each sequence. Its codes are returned as what they are, float8 numbers.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
LARGEST_CODE = 448.0


def listed():
    return [
        # four beams of one short request, a step: latency is all there is
        {"name": "prefix_attention_1x4x12_300x64_bf16", "kind": "prefix", "groups": 1, "each": 4, "heads": 12, "kv_heads": 12, "q": 1, "prompt": 300,
         "tail": 20, "width": 64, "page": 16, "dtype": "bf16"},
        # the benchmark's heads and prompt length, sixteen requests of four beams
        {"name": "prefix_attention_16x4x12_1024x64_bf16", "kind": "prefix", "groups": 16, "each": 4, "heads": 12, "kv_heads": 12, "q": 1, "prompt": 1024,
         "tail": 128, "width": 64, "page": 64, "dtype": "bf16"},
        # sixty-four conversations behind one instruction text, shared heads
        {"name": "prefix_attention_1x64x32_8_8001x128_bf16", "kind": "prefix", "groups": 1, "each": 64, "heads": 32, "kv_heads": 8, "q": 1, "prompt": 8001,
         "tail": 500, "width": 128, "page": 64, "dtype": "bf16"},
        # three drafted tokens and the last one of 3 x 7 candidates, an odd prompt, small pages
        {"name": "prefix_attention_3x7x14_2_2501x96_f16", "kind": "prefix", "groups": 3, "each": 7, "heads": 14, "kv_heads": 2, "q": 4, "prompt": 2501,
         "tail": 90, "width": 96, "page": 32, "dtype": "f16"},
        # many samples of one long document: more arithmetic than bytes
        {"name": "prefix_attention_1x256x64_8_30000x128_bf16", "kind": "prefix", "groups": 1, "each": 256, "heads": 64, "kv_heads": 8, "q": 1, "prompt": 30000,
         "tail": 300, "width": 128, "page": 64, "dtype": "bf16"},
        # one request's step
        {"name": "beam_select_1x4x50257_bf16", "kind": "select", "requests": 1, "beams": 4, "vocab": 50257, "keep": 4, "finished": False, "dtype": "bf16"},
        # a batch of requests, some beams at their end
        {"name": "beam_select_64x4x50257_f32", "kind": "select", "requests": 64, "beams": 4, "vocab": 50257, "keep": 8, "finished": True, "dtype": "f32"},
        # wide beams over a large vocabulary, twice as many candidates as beams
        {"name": "beam_select_32x16x128000_bf16", "kind": "select", "requests": 32, "beams": 16, "vocab": 128000, "keep": 32, "finished": False,
         "dtype": "bf16"},
        # one request of four beams: which page is copied, which is new
        {"name": "cache_advance_1x4x12_layers", "kind": "advance", "requests": 1, "beams": 4, "layers": 12, "kv_heads": 12, "width": 64, "page": 16,
         "prompt": 300, "longest": 40, "spare": 64, "count": 1},
        # a batch of requests at its first parting from prompts that end inside a page: nearly every row copies
        {"name": "cache_advance_64x4x4_layers", "kind": "advance", "requests": 64, "beams": 4, "layers": 4, "kv_heads": 8, "width": 128, "page": 64,
         "prompt": 1000, "longest": 1, "spare": 400, "count": 1},
        # a thousand rows in a large pool, one layer: the books alone are the work
        {"name": "cache_advance_256x4x1_layer", "kind": "advance", "requests": 256, "beams": 4, "layers": 1, "kv_heads": 1, "width": 64, "page": 16,
         "prompt": 2000, "longest": 200, "spare": 60000, "count": 3},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["prefix", "prefix", "prefix", "select", "select", "advance"])
    if kind == "prefix":
        heads, kv_heads = rng.choice([(12, 12), (12, 12), (16, 4), (32, 8), (64, 8), (8, 1), (14, 2), (6, 3)])
        width, page, q = rng.choice([64, 64, 128, 128, 32, 80, 96]), rng.choice([16, 32, 64, 64, 128]), rng.choice([1, 1, 1, 1, 2, 4])
        groups, each, prompt = rng.choice([1, 1, 1, 2, 3, 8, 16]), _log(rng, 2, 256), _log(rng, 100, 30000)
        while each > 2 and (groups * each * q * heads * prompt * width > 256 * 64 * 30000 * 128 or groups * each * heads * q > 16384):
            each //= 2
        while groups * prompt * kv_heads * width > 4 * 8 * 30000 * 128:
            prompt //= 2
        return {"kind": "prefix", "groups": groups, "each": each, "heads": heads, "kv_heads": kv_heads, "q": q, "prompt": prompt, "tail": _log(rng, 4, 500),
                "width": width, "page": page, "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "select":
        requests, beams, vocab = _log(rng, 1, 64), rng.randint(1, 16), _log(rng, 1000, 128000)
        while requests > 1 and requests * beams * vocab > 32 * 16 * 128000:
            requests //= 2
        return {"kind": "select", "requests": requests, "beams": beams, "vocab": vocab, "keep": beams * rng.choice([1, 2]), "finished": rng.random() < 0.3,
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    requests, beams, layers = _log(rng, 1, 128), rng.randint(2, 8), rng.randint(1, 12)
    kv_heads, width, page = rng.choice([1, 2, 8, 12]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    while requests > 1 and requests * beams * layers * kv_heads * width * page > 64 * 4 * 4 * 8 * 128 * 64:
        requests //= 2
    return {"kind": "advance", "requests": requests, "beams": beams, "layers": layers, "kv_heads": kv_heads, "width": width, "page": page,
            "prompt": _log(rng, 16, 2000), "longest": _log(rng, 1, 200), "spare": 5 * requests * beams + rng.randint(0, 200), "count": rng.choice([1, 1, 1, 2, 5])}


# ---- inputs ------------------------------------------------------------------------------------


def _tails(case, seed):
    """Each sequence's tokens behind the prompt: spread evenly from q to the longest, in an order made from the seed."""
    batch, low = case["groups"] * case["each"], case["q"]
    high = max(low, case["tail"])
    spread = [high if batch == 1 else low + (high - low) * i // (batch - 1) for i in range(batch)]
    order = torch.randperm(batch, generator=torch.Generator().manual_seed(int(seed)))
    return [spread[i] for i in order.tolist()]


def _pool(shape, generator):
    """Codes and scales of a pool in use: values of about one, larger in some heads and pages; [..., kv_heads, page, width]."""
    tensors = []
    for _ in range(2):
        codes = torch.empty(shape, dtype=E4M3, device="cuda")
        flat = codes.view(-1, *shape[-2:])
        for start in range(0, flat.shape[0], 8192):
            part = flat[start : start + 8192]
            part.copy_((torch.randn(part.shape, generator=generator, device="cuda") * 64.0).clamp_(-LARGEST_CODE, LARGEST_CODE))
        tensors.append((codes, torch.exp2(torch.randint(-8, -4, shape[:-2], generator=generator, device="cuda").float())))
    return tensors[0][0], tensors[1][0], tensors[0][1], tensors[1][1]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"prefix": _prepare_prefix, "select": _prepare_select, "advance": _prepare_advance}[case["kind"]](case, seed, g)


def _prepare_prefix(case, seed, g):
    groups, each, page = case["groups"], case["each"], case["page"]
    batch, whole = groups * each, case["prompt"] // page                   # pages of a prompt that all of a group have
    blocks = -(-(case["prompt"] + max(case["q"], case["tail"])) // page)
    pages = groups * whole + batch * (blocks - whole) + 5
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.empty(groups, each, blocks, dtype=torch.int32, device="cuda")
    table[:, :, :whole] = order[: groups * whole].reshape(groups, 1, whole)
    table[:, :, whole:] = order[groups * whole : groups * whole + batch * (blocks - whole)].reshape(groups, each, blocks - whole)
    shape = (batch, case["q"], case["heads"], case["width"])
    return {"case": case, "table": table.reshape(batch, blocks), "cache": _pool((pages, case["kv_heads"], page, case["width"]), g),
            "lengths": torch.tensor([case["prompt"] + tail for tail in _tails(case, seed)], dtype=torch.int32, device="cuda"),
            "shared": torch.full((groups,), whole * page, dtype=torch.int32, device="cuda"),
            "q": torch.randn(shape, generator=g, device="cuda").to(DTYPES[case["dtype"]]).transpose(1, 2)}


def _prepare_select(case, seed, g):
    shape = (case["requests"], case["beams"])
    logits = torch.randn(*shape, case["vocab"], generator=g, device="cuda") * 2.5
    # as a trained model's are: a few tokens stand out
    likely = torch.randint(0, case["vocab"], (*shape, 24), generator=g, device="cuda")
    logits.scatter_add_(2, likely, torch.randn(*shape, 24, generator=g, device="cuda").abs_() * 6.0)
    state = {"case": case, "logits": logits.to(DTYPES[case["dtype"]]), "scores": -torch.rand(shape, generator=g, device="cuda") * 4.0 - 10.0,
             "finished": None, "end": 0}
    if case["finished"]:
        state["finished"] = torch.rand(shape, generator=g, device="cuda") < 0.2
        state["finished"][:, 0] = False
        state["end"] = case["vocab"] - 1
    return state


def _prepare_advance(case, seed, g):
    requests, beams, page = case["requests"], case["beams"], case["page"]
    batch, whole = requests * beams, case["prompt"] // page
    # every request's beams have the prompt's whole pages together; behind them, each has pages of its own, or, with one token of its own at most, still
    # the page in which the prompt ends. Beams of a request are of one length.
    grown = torch.randint(0, case["longest"] + 1, (requests,), generator=torch.Generator().manual_seed(int(seed)))
    if case["longest"] == 1:
        grown.zero_()
    lengths = (case["prompt"] + grown).tolist()
    blocks = -(-(case["prompt"] + case["longest"] + case["count"]) // page)
    needed = [whole + ((-(-n // page)) - whole) * (1 if case["longest"] == 1 else beams) for n in lengths]
    pages = requests * (whole + (-(-(case["prompt"] + case["longest"]) // page) - whole) * beams) + case["spare"]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed) + 1)).tolist()
    rows, references, used = [], [0] * pages, 0
    for r in range(requests):
        own_pages, have = needed[r] - whole, -(-lengths[r] // page) - whole
        shared = order[used : used + whole]
        rest = order[used + whole : used + whole + own_pages]
        used += needed[r]
        for b in range(beams):
            mine = rest[b * have : (b + 1) * have] if own_pages != have else rest
            rows.append(shared + mine + [0] * (blocks - whole - have))
            for p in shared + mine:
                references[p] += 1
    # a step of the search: beams go on from any beam of their request, mostly from the better ones
    choice = (torch.rand(requests, beams, generator=g, device="cuda") ** 2 * beams).long().clamp_(max=beams - 1)
    parents = choice + torch.arange(requests, device="cuda")[:, None] * beams
    return {"case": case, "table": torch.tensor(rows, dtype=torch.int32).cuda(), "references": torch.tensor(references, dtype=torch.int32).cuda(),
            "lengths": torch.tensor(lengths, dtype=torch.int32).repeat_interleave(beams).cuda(), "parents": parents.reshape(-1).to(torch.int32),
            "counts": torch.full((batch,), case["count"], dtype=torch.int32, device="cuda"),
            "cache": _pool((case["layers"], pages, case["kv_heads"], page, case["width"]), g)}


# ---- one pass ----------------------------------------------------------------------------------


def _gather(codes, scales, pages):
    """[..., kv_heads, tokens, width] in f32: the pages [..., blocks] named, decoded and side by side."""
    pages = pages.long()
    values = codes.view(torch.uint8)[pages].view(E4M3).float() * scales[pages][..., None, None]
    values = values.transpose(-4, -3)
    return values.reshape(*values.shape[:-3], -1, values.shape[-1])


def _plain_prefix(state):
    case, q, table = state["case"], state["q"], state["table"]
    k_codes, v_codes, k_scales, v_scales = state["cache"]
    groups, each, kv_heads, width, tokens = case["groups"], case["each"], case["kv_heads"], case["width"], case["q"]
    whole, group = case["prompt"] // case["page"], case["heads"] // kv_heads
    out = torch.empty_like(q)
    for n in range(groups):
        rows = slice(n * each, (n + 1) * each)
        # [each, kv_heads, group * tokens, width]
        mine = q[rows].float().reshape(each, kv_heads, group * tokens, width) / math.sqrt(width)
        # the prefix once for all rows of the group, [kv_heads, each * group * tokens, keys] scores
        k, v = _gather(k_codes, k_scales, table[n * each, :whole]), _gather(v_codes, v_scales, table[n * each, :whole])
        near = (mine.transpose(0, 1).reshape(kv_heads, -1, width) @ k.transpose(-1, -2)).reshape(kv_heads, each, group * tokens, -1)
        tail_k, tail_v = _gather(k_codes, k_scales, table[rows, whole:]), _gather(v_codes, v_scales, table[rows, whole:])
        far = (mine @ tail_k.transpose(-1, -2)).transpose(0, 1)                # [kv_heads, each, group * tokens, keys]
        at = state["lengths"][rows].long()[:, None] + torch.arange(-tokens, 0, device=q.device)
        key = whole * case["page"] + torch.arange(far.shape[-1], device=q.device)
        visible = (key <= at[:, :, None])[:, None].expand(each, group, tokens, -1).reshape(each, group * tokens, -1)
        far = far.masked_fill(~visible, -math.inf)
        # (every query sees its own token, so each row has a finite maximum)
        top = torch.maximum(near.amax(-1, keepdim=True) if near.shape[-1] else far.amax(-1, keepdim=True), far.amax(-1, keepdim=True))
        near, far = torch.exp_(near.sub_(top)), torch.exp_(far.sub_(top))
        total = near.sum(-1, keepdim=True) + far.sum(-1, keepdim=True)
        found = (near.reshape(kv_heads, each * group * tokens, -1) @ v).reshape(kv_heads, each, group * tokens, width)
        found = found + (far.transpose(0, 1) @ tail_v).transpose(0, 1)
        out[rows] = (found / total).transpose(0, 1).reshape(each, case["heads"], tokens, width).to(q.dtype)
    return out


def _plain_select(state):
    """Over all beams and tokens of a request, the `keep` largest of score + log softmax: their values, the rows of logits they go on from, their tokens;
    in falling order, ties to the lower beam, then the lower token. In 64 bits: neighbours may be close. A finished beam has one candidate, `end`, at its
    score as it is."""
    case, logits = state["case"], state["logits"].double()
    shifted = logits - logits.amax(-1, keepdim=True)
    total = shifted - torch.log(torch.exp(shifted).sum(-1, keepdim=True)) + state["scores"].double()[..., None]
    if state["finished"] is not None:
        token = torch.arange(case["vocab"], device=logits.device)
        stays = torch.where(token == state["end"], state["scores"].double()[..., None], -math.inf)
        total = torch.where(state["finished"][..., None], stays, total)
    values, index = torch.sort(total.flatten(1), dim=1, descending=True, stable=True)
    values, index = values[:, : case["keep"]], index[:, : case["keep"]]
    first = torch.arange(case["requests"], device=logits.device)[:, None] * case["beams"]
    return values.float(), (index // case["vocab"] + first).int(), (index % case["vocab"]).int()


def _plain_advance(state):
    """Row b of the table goes on from row parents[b] and gets room for counts[b] tokens. A last page that is partly filled, and that another row has too, is
    copied for all that write into it, but for the last of them where no one else has it; new pages are the lowest free ones, row by row."""
    page, table, references = state["case"]["page"], state["table"].long(), state["references"].long()
    parents, counts, before = state["parents"].long(), state["counts"].long(), state["lengths"].long()
    batch, blocks = table.shape
    pages, row, block = references.shape[0], torch.arange(batch, device=table.device), torch.arange(blocks, device=table.device)
    starts = before[parents]
    held, has = (before + page - 1) // page, (starts + page - 1) // page
    had_it, has_it = block < held[:, None], block < has[:, None]
    now = torch.where(has_it, table[parents], table)
    references = references.scatter_add(0, table.flatten(), -had_it.long().flatten()).scatter_add(0, now.flatten(), has_it.long().flatten())
    # who writes into a page that is there already, and who of them is the last
    writes = (counts > 0) & (starts % page > 0)
    last = now.gather(1, (has - 1).clamp(min=0)[:, None])[:, 0]
    writers = torch.zeros(pages, dtype=torch.int64, device=table.device).scatter_add(0, last, writes.long())
    final = torch.full((pages,), -1, dtype=torch.int64, device=table.device).scatter_reduce(0, last, torch.where(writes, row, -1), "amax")
    copies = writes & ((references[last] > writers[last]) | (final[last] != row))
    lengths = starts + counts
    new = (lengths + page - 1) // page - has
    upto = (new + copies).cumsum(0)
    free = torch.sort((references > 0).long(), stable=True).indices
    first = upto - new - copies.long()
    targets = torch.where(copies, free[first], last)
    references = references.scatter_add(0, last, -copies.long())
    now = torch.where((block == has[:, None] - 1) & copies[:, None], targets[:, None], now)
    fresh = (block >= has[:, None]) & (block < (has + new)[:, None])
    taken = free[(first + copies.long())[:, None] + (block - has[:, None]).clamp(min=0).minimum(new.clamp(min=1)[:, None] - 1)]
    now = torch.where(fresh, taken, now)
    references = references.scatter_add(0, targets, copies.long()).scatter_add(0, taken.flatten(), fresh.long().flatten())
    # (a row that copies nothing copies a page onto itself; the sources are no targets)
    for t in state["cache"]:
        raw = t.view(torch.uint8) if t.dtype == E4M3 else t
        raw[:, targets] = raw[:, last]
    return [now.int(), lengths.int(), references.int(), starts.int(), *state["cache"]]


def _own(state):
    from tessiq_b200 import ops

    case = state["case"]
    if case["kind"] == "prefix":
        return ops.prefix_attention(state["q"], *state["cache"], state["table"], state["lengths"], state["shared"])
    if case["kind"] == "select":
        return ops.beam_select(state["logits"], state["scores"], case["keep"], state["finished"], state["end"])
    return [*ops.cache_advance(*state["cache"], state["table"], state["lengths"], state["references"], state["counts"], state["parents"]), *state["cache"]]


PLAIN = {"prefix": _plain_prefix, "select": _plain_select, "advance": _plain_advance}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    if case["kind"] == "select":
        rows, size = case["requests"] * case["beams"], {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
        # an exponential's argument, the exponential, its sum and a comparison for each logit
        return {"bytes": rows * (case["vocab"] * size + 4 + (1 if case["finished"] else 0)) + case["requests"] * case["keep"] * 12,
                "flops": 4 * rows * case["vocab"]}
    if case["kind"] == "advance":
        batch, page = case["requests"] * case["beams"], case["page"]
        blocks = -(-(case["prompt"] + case["longest"] // 2 + case["count"]) // page)
        pages = case["requests"] * (case["prompt"] // page) + case["spare"]
        # about half the beams of a request share their last page with another one, which is copied; at the first parting all but one
        inside = 1.0 if case["longest"] > 1 else float(case["prompt"] % page > 0)
        copied = case["requests"] * int((case["beams"] - 1) * (inside if case["longest"] == 1 else 0.5) * (page - 1) / page)
        return {"bytes": 4 * (2 * batch * blocks + 6 * batch + 2 * pages) + copied * case["layers"] * 4 * case["kv_heads"] * (page * case["width"] + 4),
                "flops": batch * blocks}
    whole = case["prompt"] // case["page"] * case["page"]
    rows, tails = case["groups"] * case["each"] * case["heads"] * case["q"], _tails(case, 0)
    keys = case["groups"] * whole + sum(case["prompt"] - whole + t for t in tails)
    pairs = sum(case["q"] * (case["prompt"] + t) - case["q"] * (case["q"] - 1) // 2 for t in tails)
    return {"bytes": 4 * case["width"] * rows + 2 * case["kv_heads"] * (keys * case["width"] + 4 * -(-keys // case["page"])) + 4 * -(-keys // case["page"]),
            "flops": 4 * pairs * case["heads"] * case["width"]}


# ---- the definition in 64 bits -------------------------------------------------------------------


def _exact_prefix(s, case):
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lengths = s["lengths"].tolist()
    for h in range(case["kv_heads"]):
        k_head, v_head = ((s["cache"][c].view(torch.uint8)[:, h].view(E4M3), s["cache"][c + 2][:, h]) for c in (0, 1))
        for b in range(case["groups"] * case["each"]):
            length = lengths[b]
            pages = s["table"][b, : -(-length // page)].long()
            k, v = ((codes.view(torch.uint8)[pages].view(E4M3).double() * scales[pages].double()[:, None, None]).reshape(-1, case["width"])[:length]
                    for codes, scales in (k_head, v_head))
            q = s["q"][b, h * group : (h + 1) * group].double().reshape(-1, case["width"])
            scores = (q @ k.T) * case["width"] ** -0.5
            at = torch.arange(length - case["q"], length, device="cuda").repeat(group)
            if case["q"] > 1:
                scores[torch.arange(length, device="cuda")[None] > at[:, None]] = -math.inf
            out[b, h * group : (h + 1) * group] = (torch.softmax(scores, 1) @ v).reshape(group, case["q"], case["width"])
    return out


def _exact_select(s, case):
    values, parents, tokens = [], [], []
    for r in range(case["requests"]):
        whole = s["logits"][r].double()
        total = whole - torch.logsumexp(whole, 1)[:, None] + s["scores"][r].double()[:, None]
        if s["finished"] is not None:
            for b in s["finished"][r].nonzero()[:, 0].tolist():
                total[b] = -math.inf
                total[b, s["end"]] = s["scores"][r, b].double()
        line = total.reshape(-1)
        # everything from the last one kept on, ties with it too, in the order of beam and token; then by value
        least = torch.topk(line, case["keep"]).values[-1]
        among = (line >= least).nonzero()[:, 0]
        among = among[torch.argsort(line[among], descending=True, stable=True)][: case["keep"]]
        values.append(line[among])
        parents.append(r * case["beams"] + torch.div(among, case["vocab"], rounding_mode="floor"))
        tokens.append(torch.remainder(among, case["vocab"]))
    return torch.stack(values), torch.stack(parents).int(), torch.stack(tokens).int()


def _exact_advance(s, case):
    """A page at a time on the host, as a serving loop without a GPU would keep its books."""
    page, table, references = case["page"], s["table"].tolist(), s["references"].tolist()
    lengths, parents, counts = s["lengths"].tolist(), s["parents"].tolist(), s["counts"].tolist()
    old = [row[: -(-n // page)] for row, n in zip(table, lengths)]
    rows = [list(old[p]) for p in parents]
    for row in rows:
        for p in row:
            references[p] += 1
    for row in old:
        for p in row:
            references[p] -= 1
    free = iter([p for p, n in enumerate(references) if n == 0])
    starts, pairs = [lengths[p] for p in parents], []
    for row, start, count in zip(rows, starts, counts):
        if count and start % page and references[row[-1]] > 1:
            references[row[-1]] -= 1
            pairs.append((row[-1], next(free)))
            row[-1] = pairs[-1][1]
            references[row[-1]] = 1
        while len(row) * page < start + count:
            row.append(next(free))
            references[row[-1]] = 1
    now = [row + before[len(row) :] for row, before in zip(rows, table)]
    tensors = [t.double() for t in s["cache"]]
    for t in tensors:
        for a, b in pairs:
            t[:, b] = t[:, a]
    whole = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (now, [a + c for a, c in zip(starts, counts)], references, starts)]
    return [*whole, *tensors]


def exact(case, seed):
    return {"prefix": _exact_prefix, "select": _exact_select, "advance": _exact_advance}[case["kind"]](prepare(case, seed), case)
