"""The serving operators as cases: attention with a sliding window and sinks, the paged cache in 8 bits (its writer and the
attention that reads it) and the copying of its pages, each with inputs, one pass and its outputs.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs and the cache's tensors, on the GPU
    run(state)          one pass: the plain form in torch, or with `own` the call of the library's operator
    work(case)          bytes and flops that a pass cannot do without
    exact(case, seed)   the outputs of a pass in 64 bits, from the definition

The cache: pages of `page` tokens, [pages, kv_heads, page, width] in e4m3, with one f32 scale a page and head; a table row names a
sequence's pages in order. Its codes are returned as what they are, float8 numbers, beside the scales they are multiplied by.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn
LARGEST_CODE = 448.0
SMALLEST_SCALE = 2.0**-126


def listed():
    return [
        # a prompt of the benchmark's heads under a window: the whole prefill of a window layer
        {"name": "window_prefill_8x12x4096x64_bf16", "kind": "window", "batch": 8, "heads": 12, "kv_heads": 12, "q": 4096, "kv": 4096, "width": 64,
         "window": 1024, "sinks": 4, "dtype": "bf16"},
        # wide shared heads, an odd length, a window that is no multiple of anything
        {"name": "window_prefill_2x32_8x2501x128_f16", "kind": "window", "batch": 2, "heads": 32, "kv_heads": 8, "q": 2501, "kv": 2501, "width": 128,
         "window": 333, "sinks": 16, "dtype": "f16"},
        # one new token of every sequence against a 16-bit cache
        {"name": "window_decode_32x32_8x4100x128_bf16", "kind": "window", "batch": 32, "heads": 32, "kv_heads": 8, "q": 1, "kv": 4100, "width": 128,
         "window": 2048, "sinks": 4, "dtype": "bf16"},
        # a single short conversation: latency is all there is
        {"name": "cache_attention_1x12x100x64_bf16", "kind": "attend", "batch": 1, "heads": 12, "kv_heads": 12, "q": 1, "shortest": 100, "longest": 100,
         "width": 64, "page": 16, "window": 0, "sinks": 0, "dtype": "bf16"},
        # the benchmark's decoding batch, sequences of all lengths
        {"name": "cache_attention_64x12x1000x64_bf16", "kind": "attend", "batch": 64, "heads": 12, "kv_heads": 12, "q": 1, "shortest": 1, "longest": 2000,
         "width": 64, "page": 64, "window": 0, "sinks": 0, "dtype": "bf16"},
        # long contexts with shared heads: the cache is what there is to read
        {"name": "cache_attention_16x64_8x30000x128_bf16", "kind": "attend", "batch": 16, "heads": 64, "kv_heads": 8, "q": 1, "shortest": 20001,
         "longest": 40000, "width": 128, "page": 64, "window": 0, "sinks": 0, "dtype": "bf16"},
        # three drafted tokens and the last one, under a window with sinks
        {"name": "cache_attention_drafts_48x32_8x128_f16", "kind": "attend", "batch": 48, "heads": 32, "kv_heads": 8, "q": 4, "shortest": 37,
         "longest": 9000, "width": 128, "page": 32, "window": 1024, "sinks": 4, "dtype": "f16"},
        # a decoding step's write: one token a sequence
        {"name": "cache_store_64x12x1x64_bf16", "kind": "store", "batch": 64, "kv_heads": 12, "tokens": 1, "shortest": 1, "longest": 1, "held": 999,
         "width": 64, "page": 64, "dtype": "bf16"},
        # prompts of several lengths in one padded batch, some behind a shared prefix
        {"name": "cache_store_8x8x2047x128_bf16", "kind": "store", "batch": 8, "kv_heads": 8, "tokens": 2047, "shortest": 100, "longest": 2047, "held": 300,
         "width": 128, "page": 64, "dtype": "bf16"},
        # a forked conversation's last page, in every layer
        {"name": "copy_pages_1x12_layers", "kind": "copy", "count": 1, "layers": 12, "kv_heads": 12, "width": 64, "page": 16},
        # a batch of beams that part
        {"name": "copy_pages_40x4_layers", "kind": "copy", "count": 40, "layers": 4, "kv_heads": 8, "width": 128, "page": 64},
        # compaction: a few hundred pages of each layer move
        {"name": "copy_pages_700x3_layers", "kind": "copy", "count": 700, "layers": 3, "kv_heads": 8, "width": 128, "page": 64},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["window", "window", "decode", "attend", "attend", "attend", "store", "copy"])
    heads, kv_heads = rng.choice([(12, 12), (12, 12), (16, 16), (16, 4), (32, 8), (64, 8), (8, 1), (14, 2), (6, 3)])
    width, dtype = rng.choice([64, 64, 128, 128, 32, 80, 96]), rng.choice(["bf16", "bf16", "f16"])
    if kind == "window":
        tokens = _log(rng, 20, 4200)
        batch = _log(rng, 1, 16)
        while batch > 1 and batch * heads * tokens * tokens > 8 * 12 * 4096 * 4096:
            batch -= 1
        heads, kv_heads = (heads, kv_heads) if heads * tokens * tokens <= 8 * 12 * 4096 * 4096 else (12, 12)
        more = rng.choice([0, 0, 0, rng.randint(1, 600)])
        return {"kind": "window", "batch": batch, "heads": heads, "kv_heads": kv_heads, "q": tokens, "kv": tokens + more, "width": width,
                "window": _log(rng, 1, 4200), "sinks": rng.choice([0, 1, 4, 16, 100]), "dtype": dtype}
    if kind == "decode":
        batch, kv = _log(rng, 1, 64), _log(rng, 1, 16384)
        while batch * kv_heads * kv * width > 32 * 8 * 16384 * 128:
            kv //= 2
        return {"kind": "window", "batch": batch, "heads": heads, "kv_heads": kv_heads, "q": rng.choice([1, 1, 1, 2, 5]), "kv": kv, "width": width,
                "window": _log(rng, 1, 16384), "sinks": rng.choice([0, 4, 4, 16, 100]), "dtype": dtype}
    page = rng.choice([16, 32, 64, 64, 128])
    if kind == "attend":
        batch, longest = _log(rng, 1, 128), _log(rng, 4, 40000)
        while batch * kv_heads * longest * width > 16 * 8 * 40000 * 128:
            longest //= 2
        return {"kind": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "q": rng.choice([1, 1, 1, 1, 2, 4]),
                "shortest": rng.choice([1, longest, max(1, longest // 2)]), "longest": longest, "width": width, "page": page,
                "window": rng.choice([0, 0, _log(rng, 16, 8192)]), "sinks": rng.choice([0, 4, 16]), "dtype": dtype}
    if kind == "store":
        tokens = rng.choice([1, 1, _log(rng, 2, 2047)])
        batch = _log(rng, 1, 128)
        while batch > 1 and batch * kv_heads * tokens * width > 8 * 8 * 2047 * 128:
            batch -= 1
        return {"kind": "store", "batch": batch, "kv_heads": kv_heads if tokens * kv_heads * width <= 8 * 8 * 2047 * 128 else 8, "tokens": tokens,
                "shortest": max(1, tokens // 2), "longest": tokens, "held": rng.randint(0, 1000), "width": width, "page": page, "dtype": dtype}
    kv_heads, width, layers = rng.choice([1, 2, 4, 8, 12]), rng.choice([64, 128]), rng.randint(1, 12)
    count = _log(rng, 1, 700)
    while count * layers * kv_heads * width * page > 700 * 3 * 8 * 128 * 64:
        count = max(1, count // 2)
        layers = max(1, layers // 2) if count == 1 else layers
    return {"kind": "copy", "count": count, "layers": layers, "kv_heads": kv_heads, "width": width, "page": page}


# ---- inputs ------------------------------------------------------------------------------------


def _lengths(case, seed):
    """The sequences' lengths: spread evenly from the shortest to the longest, in an order made from the seed."""
    batch, low, high = case["batch"], case["shortest"], case["longest"]
    spread = [high if batch == 1 else low + (high - low) * i // (batch - 1) for i in range(batch)]
    order = torch.randperm(batch, generator=torch.Generator().manual_seed(int(seed)))
    return [spread[i] for i in order.tolist()]


def _pool(case, seed, pages, generator):
    """Codes and scales of a pool in use: values of about one, larger in some heads and pages."""
    shape = (pages, case["kv_heads"], case["page"], case["width"])
    tensors = []
    for _ in range(2):
        codes = torch.empty(shape, dtype=E4M3, device="cuda")
        for start in range(0, pages, 1024):
            part = codes[start : start + 1024]
            part.copy_((torch.randn(part.shape, generator=generator, device="cuda") * 64.0).clamp_(-LARGEST_CODE, LARGEST_CODE))
        scales = torch.exp2(torch.randint(-8, -4, shape[:2], generator=generator, device="cuda").float())
        tensors.append((codes, scales))
    return tensors[0][0], tensors[1][0], tensors[0][1], tensors[1][1]


def _table(batch, blocks, pages, generator):
    """Every sequence's pages, scattered over the pool."""
    return torch.randperm(pages, generator=generator, device="cuda")[: batch * blocks].to(torch.int32).reshape(batch, blocks).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    state = {"case": case}
    if case["kind"] == "copy":
        pages = 2 * case["count"] + 3
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed))).tolist()
        state["sources"], state["targets"] = order[: case["count"]], order[case["count"] : 2 * case["count"]]
        state["source_index"], state["target_index"] = (torch.tensor(state[k], device="cuda") for k in ("sources", "targets"))
        shape = (case["layers"], pages, case["kv_heads"], case["page"], case["width"])
        noise = [torch.randint(0, 120, shape, generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
        scales = [torch.rand(shape[:3], generator=g, device="cuda") + 0.5 for _ in range(2)]
        state["tensors"] = [noise[0].view(E4M3), noise[1].view(E4M3), *scales]
        return state
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "window":
        # as a projection's [batch, tokens, heads, width] result is seen by heads
        def tokens_major(heads, tokens):
            return torch.randn(case["batch"], tokens, heads, case["width"], generator=g, device="cuda").to(dtype).transpose(1, 2)

        state["q"] = tokens_major(case["heads"], case["q"])
        state["k"], state["v"] = tokens_major(case["kv_heads"], case["kv"]), tokens_major(case["kv_heads"], case["kv"])
        return state
    if case["kind"] == "attend":
        lengths, blocks = _lengths(case, seed), -(-case["longest"] // case["page"])
        pages = case["batch"] * blocks + 5
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        state["q"] = torch.randn(case["batch"], case["q"], case["heads"], case["width"], generator=g, device="cuda").to(dtype).transpose(1, 2)
    else:
        counts, blocks = _lengths(case, seed), -(-(case["held"] + case["tokens"]) // case["page"])
        pages = case["batch"] * blocks + 5
        state["starts"] = torch.full((case["batch"],), case["held"], dtype=torch.int32, device="cuda")
        state["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
        shape = (case["batch"], case["tokens"], case["kv_heads"], case["width"])
        state["k"], state["v"] = (torch.randn(shape, generator=g, device="cuda").mul_(2.0).to(dtype).transpose(1, 2) for _ in range(2))
    state["cache"] = _pool(case, seed, pages, g)
    state["table"] = _table(case["batch"], blocks, pages, g)
    return state


# ---- one pass ----------------------------------------------------------------------------------


def _visible(positions, keys, window, sinks):
    """[..., queries, keys]: the keys a query at each of the positions sees."""
    p, j = positions.unsqueeze(-1), torch.arange(keys, device=positions.device)
    return (j <= p) & ((j > p - window) | (j < sinks))


def _plain_attention(q, k, v, visible, width):
    """softmax over the visible keys; q [batch, kv_heads, group, queries, width], k and v [batch, kv_heads, keys, width], f32."""
    batch, kv_heads, group, queries, _ = q.shape
    scores = (q.reshape(batch, kv_heads, group * queries, width) @ k.transpose(-1, -2)).reshape(batch, kv_heads, group, queries, -1)
    scores = (scores / math.sqrt(width)).masked_fill_(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp_(scores.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = weights.sum(-1, keepdim=True)
    out = (weights.reshape(batch, kv_heads, group * queries, -1) @ v).reshape(batch, kv_heads, group, queries, width)
    return out / torch.where(total == 0, 1.0, total)


def _grouped(q, kv_heads):
    batch, heads, queries, width = q.shape
    return q.reshape(batch, kv_heads, heads // kv_heads, queries, width)


def _plain_window(state):
    case, q = state["case"], state["q"]
    positions = torch.arange(case["q"], device=q.device) + (case["kv"] - case["q"])
    visible = _visible(positions, case["kv"], case["window"], case["sinks"])
    out = _plain_attention(_grouped(q.float(), case["kv_heads"]), state["k"].float(), state["v"].float(), visible, case["width"])
    return out.reshape(q.shape).to(q.dtype)


def _plain_gather(codes, scales, table):
    """[batch, kv_heads, tokens, width] in f32: a table's pages, decoded."""
    pages = table.long()
    values = codes.view(torch.uint8)[pages].view(E4M3).float() * scales[pages][..., None, None]
    batch, blocks, kv_heads, page, width = values.shape
    return values.permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, blocks * page, width)


def _plain_attend(state):
    case, q = state["case"], state["q"]
    k_codes, v_codes, k_scales, v_scales = state["cache"]
    k, v = _plain_gather(k_codes, k_scales, state["table"]), _plain_gather(v_codes, v_scales, state["table"])
    positions = state["lengths"].long()[:, None] + torch.arange(-case["q"], 0, device=q.device)
    visible = _visible(positions, k.shape[2], case["window"] or 1 << 30, case["sinks"])
    out = _plain_attention(_grouped(q.float(), case["kv_heads"]), k, v, visible[:, None, None], case["width"])
    return out.reshape(q.shape).to(q.dtype)


def _plain_store_one(x, codes, scales, state):
    case, table = state["case"], state["table"].long()
    page, (batch, kv_heads, tokens, width) = case["page"], x.shape
    starts, counts = state["starts"].long(), state["counts"].long()
    i = torch.arange(tokens, device=x.device)
    positions = starts[:, None] + i
    live = i < counts[:, None]
    first = starts // page
    relative = positions // page - first[:, None]                       # which of the touched blocks a token falls in
    touched = (tokens + page - 2) // page + 1
    values = x.float().transpose(1, 2)                                  # [batch, tokens, kv_heads, width]
    largest = torch.where(live[..., None], values.abs().amax(-1), 0.0)
    most = torch.zeros(batch, touched, kv_heads, device=x.device).scatter_reduce_(1, relative[..., None].expand_as(largest), largest, "amax")
    mantissa, exponent = torch.frexp(most)
    needed = torch.ldexp(torch.ones_like(most), exponent - torch.where(mantissa > 0.875, 8, 9)).clamp_(min=SMALLEST_SCALE)
    needed = torch.where(most > 0, needed, SMALLEST_SCALE)
    # the first block may hold earlier tokens: its scale only grows, and they are encoded again
    begun = starts % page
    first_pages = table.gather(1, first[:, None])[:, 0]
    old = scales[first_pages]
    needed[:, 0] = torch.where((begun > 0)[:, None], torch.maximum(needed[:, 0], old), needed[:, 0])
    earlier = codes.view(torch.uint8)[first_pages]
    again = (earlier.view(E4M3).float() * (old / needed[:, 0])[..., None, None]).to(E4M3).view(torch.uint8)
    keep = torch.arange(page, device=x.device)[None, :] < begun[:, None]
    codes.view(torch.uint8)[first_pages] = torch.where(keep[:, None, :, None], again, earlier)
    block_live = (torch.arange(touched, device=x.device) * page < (begun + counts)[:, None]) & (counts > 0)[:, None]
    b, r = block_live.nonzero(as_tuple=True)
    scales[table[b, first[b] + r]] = needed[b, r]
    own_scale = needed.gather(1, relative[..., None].expand(batch, tokens, kv_heads))
    encoded = (values / own_scale[..., None]).to(E4M3).view(torch.uint8)
    b, t = live.nonzero(as_tuple=True)
    at = positions[b, t]
    codes.view(torch.uint8)[table[b, at // page], :, at % page] = encoded[b, t]


def _plain_store(state):
    k_codes, v_codes, k_scales, v_scales = state["cache"]
    _plain_store_one(state["k"], k_codes, k_scales, state)
    _plain_store_one(state["v"], v_codes, v_scales, state)
    return list(state["cache"])


def _plain_copy(state):
    for tensor in state["tensors"]:
        raw = tensor.view(torch.uint8) if tensor.dtype == E4M3 else tensor
        raw[:, state["target_index"]] = raw[:, state["source_index"]]
    return state["tensors"]


def _own(state):
    from tessiq_b200 import ops

    case = state["case"]
    if case["kind"] == "window":
        return ops.window_attention(state["q"], state["k"], state["v"], case["window"], case["sinks"])
    if case["kind"] == "attend":
        return ops.cache_attention(state["q"], *state["cache"], state["table"], state["lengths"], case["window"] or None, case["sinks"])
    if case["kind"] == "store":
        ops.cache_store(state["k"], state["v"], *state["cache"], state["table"], state["starts"], state["counts"])
        return list(state["cache"])
    ops.copy_pages(state["tensors"], state["sources"], state["targets"], page_axis=1)
    return state["tensors"]


PLAIN = {"window": _plain_window, "attend": _plain_attend, "store": _plain_store, "copy": _plain_copy}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------


def _seen(length, queries, window, sinks):
    """(keys that any of the last `queries` of `length` positions sees, pairs of a query and a key it sees)."""
    pairs = 0
    for p in range(max(0, length - queries), length):
        low = max(0, p - window + 1)
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, max(0, length - queries) - window + 1)
    return length - low + min(sinks, low), pairs


def work(case):
    if case["kind"] == "copy":
        return {"bytes": 2 * case["count"] * case["layers"] * 2 * case["kv_heads"] * (case["page"] * case["width"] + 4), "flops": 0}
    if case["kind"] == "store":
        counts = _lengths(case, 0)
        tokens = sum(counts) * 2 * case["kv_heads"]
        blocks = sum((case["held"] % case["page"] + n - 1) // case["page"] + 1 for n in counts) * 2 * case["kv_heads"]
        return {"bytes": tokens * case["width"] * 3 + blocks * 4, "flops": 2 * tokens * case["width"]}
    rows = case["batch"] * case["heads"] * case["q"]
    if case["kind"] == "window":
        keys, pairs = _seen(case["kv"], case["q"], case["window"], case["sinks"])
        keys, pairs = keys * case["batch"], pairs * case["batch"]
        return {"bytes": 2 * case["width"] * (2 * rows + 2 * keys * case["kv_heads"]), "flops": 4 * pairs * case["heads"] * case["width"]}
    keys = pairs = scales = 0
    for length in _lengths(case, 0):
        seen = _seen(length, case["q"], case["window"] or 1 << 30, case["sinks"])
        keys, pairs, scales = keys + seen[0], pairs + seen[1], scales + -(-seen[0] // case["page"])
    return {"bytes": 4 * case["width"] * rows + 2 * case["kv_heads"] * (keys * case["width"] + 4 * scales) + 4 * scales,
            "flops": 4 * pairs * case["heads"] * case["width"]}


# ---- the definition in 64 bits -------------------------------------------------------------------


def _exact_rows(q, k, v, positions, window, sinks):
    """One sequence and one key head: q [rows, width] at `positions`, k and v [keys, width], all f64."""
    out = torch.zeros_like(q)
    for start in range(0, q.shape[0], 4096):
        at = positions[start : start + 4096]
        s = (q[start : start + 4096] @ k.T) / math.sqrt(q.shape[1])
        j = torch.arange(k.shape[0], device=q.device)
        sees = torch.logical_and(j[None] <= at[:, None], torch.logical_or(at[:, None] - j[None] < window, (j < sinks)[None]))
        s[~sees] = -math.inf
        some = sees.any(1)
        out[start : start + 4096][some] = torch.softmax(s[some], 1) @ v
    return out


def _exact_e4m3(x):
    """The nearest e4m3 number, ties to even, of each |x| <= 448."""
    power = torch.floor(torch.log2(x.abs().clamp(min=2.0**-30))).clamp(min=-6)
    step = torch.exp2(power - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        found = []
        for t in s["tensors"]:
            t = t.double()
            for a, b in zip(s["sources"], s["targets"]):
                t[:, b] = t[:, a]
            found.append(t)
        return found
    if case["kind"] == "store":
        found = [t.double() for t in s["cache"]]
        table, starts, counts = s["table"].tolist(), s["starts"].tolist(), s["counts"].tolist()
        for x, codes, scales in ((s["k"], found[0], found[2]), (s["v"], found[1], found[3])):
            for b in range(case["batch"]):
                new = x[b, :, : counts[b]].double()
                done = 0
                while done < counts[b]:
                    block, offset = divmod(starts[b] + done, case["page"])
                    n = min(case["page"] - offset, counts[b] - done)
                    part, page = new[:, done : done + n], table[b][block]
                    need = part.abs().flatten(1).amax(1) / LARGEST_CODE
                    scale = torch.exp2(torch.ceil(torch.log2(need.clamp(min=SMALLEST_SCALE))))
                    scale = torch.where(scale / 2 >= need, scale / 2, scale).clamp(min=SMALLEST_SCALE)
                    if offset:
                        scale = torch.maximum(scale, scales[page])
                        codes[page, :, :offset] = _exact_e4m3(codes[page, :, :offset] * (scales[page] / scale)[:, None, None])
                    codes[page, :, offset : offset + n] = _exact_e4m3(part / scale[:, None, None])
                    scales[page] = scale
                    done += n
        return found
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    window = case["window"] or 1 << 40
    for b in range(case["batch"]):
        length = case["kv"] if case["kind"] == "window" else int(s["lengths"][b])
        at = torch.arange(length - case["q"], length, device="cuda").repeat(group)
        for h in range(case["kv_heads"]):
            if case["kind"] == "window":
                k, v = s["k"][b, h].double(), s["v"][b, h].double()
            else:
                pages = s["table"][b, : -(-length // case["page"])].long()
                k, v = ((s["cache"][c].view(torch.uint8)[pages, h].view(E4M3).double() * s["cache"][c + 2][pages, h].double()[:, None, None])
                        .reshape(-1, case["width"])[:length] for c in (0, 1))
            q = s["q"][b, h * group : (h + 1) * group].double().reshape(-1, case["width"])
            out[b, h * group : (h + 1) * group] = _exact_rows(q, k, v, at, window, case["sinks"]).reshape(group, case["q"], case["width"])
    return out
