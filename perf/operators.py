"""What serving from a cache held in 8 bits is timed on: the maps of a step, the append to the cache, and attention over it.

A step brings `decode` requests with `each` new tokens behind `least` to `context` cached ones, and `prompts` portions of
`tokens` tokens behind `cached` ones (several: of half of that to all of it).

maps       from the requests' lengths and their pages: where each row of the step goes, the padded block tables, the blocks
           of 16 positions that the step writes, and the tiles of rows of the requests that bring more than a few.
append     the projections [q | k | v] of a step's rows: q and k turned by position, q rounded to bfloat16, k and v written
           into the cache as e4m3 codes with one scale for 16 positions, a key/value head and keys or values each.  A scale
           is a power of two, the smallest that keeps the block's largest entry within 448; where new tokens raise it, the
           codes that the block held are rounded anew.
attention  softmax attention of the step's queries over the cached codes, causal, optionally within a window and with a
           learned number per head in the denominator.
"""

from __future__ import annotations

import math
import random

import torch

own = False

F32, F64, I32, I64, BF16, F8 = torch.float32, torch.float64, torch.int32, torch.int64, torch.bfloat16, torch.float8_e4m3fn
BLOCK = 16                        # positions that share a scale
LEAST, MOST = -100, 119           # exponents a scale may have
LARGEST = 448.0                   # the largest e4m3 number
FEW_ROWS, TILE_ROWS = 16, 128     # the maps' tiles: requests of more than 16 packed rows, 128 rows a tile

# query heads, key/value heads, head size
HEADS = {"tinyllama": (32, 4, 64), "llama2-7b": (32, 32, 128), "llama3-8b": (32, 8, 128), "heads 14/2 of 64": (14, 2, 64),
         "heads 9/3 of 128": (9, 3, 128), "heads 16/1 of 128": (16, 1, 128)}


def _case(op, heads, decode=0, least=0, context=0, each=1, prompts=0, tokens=0, cached=0, page=64, **more):
    return {"op": op, "heads": heads, "decode": decode, "least": least, "context": context, "each": each, "prompts": prompts,
            "tokens": tokens, "cached": cached, "page": page, **more}


def listed():
    return [
        # a small chat server's decode step: eight requests, pages of 64
        dict(_case("maps", "llama3-8b", decode=8, least=100, context=2047), name="maps decode 8"),
        # a full server with long tables: 256 decoding requests and four prompts
        dict(_case("maps", "llama3-8b", decode=256, least=100, context=30000, prompts=4, tokens=2048, page=16), name="maps 256 + 4"),
        # the same eight requests' new keys and values
        dict(_case("append", "llama3-8b", decode=8, least=100, context=2047, partials=1, wide=False), name="append decode 8"),
        # 64 requests behind a product that split its sum three ways
        dict(_case("append", "tinyllama", decode=64, least=512, context=2047, partials=3, wide=True), name="append 64 partial"),
        # a prompt's portion
        dict(_case("append", "llama3-8b", prompts=1, tokens=2048, cached=1001, partials=1, wide=False), name="append prompt 2048"),
        # one person in a chat
        dict(_case("attention", "tinyllama", decode=1, least=1000, context=1000, window=0, sink=False), name="decode 1"),
        # eight requests at the end of the larger model's context
        dict(_case("attention", "llama3-8b", decode=8, least=8191, context=8191, window=0, sink=False), name="decode 8"),
        # a busy server with long texts: what the cache is held in 8 bits for
        dict(_case("attention", "llama3-8b", decode=64, least=2000, context=8191, window=0, sink=False), name="decode 64 long"),
        # a question behind a long text
        dict(_case("attention", "llama3-8b", prompts=1, tokens=61, cached=3001, window=0, sink=False), name="question 61"),
        # the longest prompt the small model takes
        dict(_case("attention", "tinyllama", prompts=1, tokens=2048, window=0, sink=False), name="prompt 2048"),
        # the second portion of a long prompt, a key/value head for each query head
        dict(_case("attention", "llama2-7b", prompts=1, tokens=2048, cached=2048, window=0, sink=False), name="7b prompt portion"),
        # continuous batching: decoding requests beside the prompts of new ones
        dict(_case("attention", "tinyllama", decode=24, least=100, context=1500, prompts=3, tokens=389, window=0, sink=False),
             name="mixed 24 + 3"),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is uniform."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("maps", "append", "attention", "attention", "attention"))
    heads = rng.choice(tuple(HEADS))
    page = rng.choice((16, 32, 48, 64, 128))
    kind = rng.choice(("decode", "decode", "prompt", "mixed"))
    least, each, decode, context, prompts, tokens, cached = 0, 1, 0, 0, 0, 0, 0
    if kind == "decode":
        decode, each = _spread(rng, 1, 64), rng.choice((1, 1, 1, 2, 3))
        _heads, kv_heads, dim = HEADS[heads]
        context = _spread(rng, 1, min(8000, (1 << 29) // (decode * kv_heads * dim)))
        least = int(context * rng.uniform(0.1, 1.0))
    elif kind == "prompt":
        prompts, tokens = 1, _spread(rng, 1, 2000)
        cached = _spread(rng, 1, 2000 if tokens > 256 else 8000) if rng.random() < 0.6 else 0
    else:
        decode, context, prompts, tokens = _spread(rng, 1, 24), _spread(rng, 16, 1800), rng.randrange(1, 4), _spread(rng, 2, 500)
        least = context // 3
    shape = dict(decode=decode, least=least, context=context, each=each, prompts=prompts, tokens=tokens, cached=cached, page=page)
    if op == "maps":
        return _case("maps", heads, **shape)
    if op == "append":
        wide = rng.random() < 0.4
        return _case("append", heads, **shape, partials=rng.randrange(1, 5) if wide and kind != "prompt" else 1, wide=wide)
    return _case("attention", heads, **shape, window=_spread(rng, 20, 3000) if rng.random() < 0.25 else 0, sink=rng.random() < 0.25)


# ----------------------------------------------------------------------------- a step's requests

def _requests(case, seed):
    """(cached tokens, new tokens) per request: the same ones for every seed, in another order."""
    rng = random.Random(str(sorted(case.items())))
    out = [(rng.randint(case["least"], case["context"]), case["each"]) for _ in range(case["decode"])]
    random.Random(f"decode {seed}").shuffle(out)
    new = [rng.randint(max(1, case["tokens"] // 2), case["tokens"]) if case["prompts"] > 1 else case["tokens"] for _ in range(case["prompts"])]
    random.Random(f"prompts {seed}").shuffle(new)
    return out + [(case["cached"], n) for n in new]


def _quantised(x, exponent):
    """Entries `x` (finite, 32 or 64 bits) times 2^-exponent as e4m3 codes, within the format's range."""
    return torch.ldexp(x, -exponent).clamp(-LARGEST, LARGEST).to(F32).to(F8)


def _exponents(largest):
    """The smallest e with largest <= 448 * 2^e, within bounds."""
    m, k = torch.frexp(largest)           # m in [0.5, 1); 448 = 0.875 * 2^9
    e = k - 9 + (m > 0.875).to(k.dtype)
    return torch.where(largest > 0, e, torch.full_like(e, LEAST)).clamp(LEAST, MOST)


def prepare(case, seed):
    """The step's lengths and pages; for append the projections and the cache before the step; for attention the queries and
    the cache with the step's own keys and values in it."""
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    requests = _requests(case, seed)
    heads, kv_heads, dim = HEADS[case["heads"]]
    page, S = case["page"], len(requests)
    blocks = [-(-(c + n) // page) for c, n in requests]
    n_pages = sum(blocks) + 3
    pages = torch.randperm(n_pages, generator=gen, device=dev)[: sum(blocks)].to(I32)
    rows = sum(n for _, n in requests)
    width = max(blocks) if case["op"] == "attention" else -(-max(c + n + 512 for c, n in requests) // page)
    state = {"case": case, "cached": torch.tensor([c for c, _ in requests], dtype=I32, device=dev), "pages": pages, "rows": rows,
             "q_len": torch.tensor([n for _, n in requests], dtype=I32, device=dev), "width": width,
             "longest": max(n for _, n in requests), "shortest": min(n for _, n in requests), "keys": max(c + n for c, n in requests)}
    if case["op"] == "maps":
        return state
    state["maps"] = _plain_maps(state)
    # keys with channels of their own size, as a trained model's have; values of one size, a few tokens far smaller
    size = torch.exp(torch.randn(2, kv_heads, 1, dim, generator=gen, device=dev) * torch.tensor([0.7, 0.1], device=dev).view(2, 1, 1, 1))
    codes = torch.empty(n_pages, 2, kv_heads, page, dim, dtype=torch.uint8, device=dev)
    scales = torch.empty(n_pages, 2, kv_heads, page // BLOCK, dtype=F32, device=dev)
    step = max(1, (1 << 26) // (2 * kv_heads * page * dim))
    for at in range(0, n_pages, step):
        n = min(step, n_pages - at)
        x = torch.randn(n, 2, kv_heads, page, dim, generator=gen, device=dev) * size
        x = x.view(n, 2, kv_heads, page // BLOCK, BLOCK, dim)
        e = _exponents(x.abs().amax((-1, -2)))
        codes[at: at + n] = _quantised(x, e[..., None, None]).view(torch.uint8).view(n, 2, kv_heads, page, dim)
        scales[at: at + n] = torch.ldexp(torch.ones((), device=dev), e)
    state |= {"codes": codes, "scales": scales}
    if case["op"] == "append":
        x = torch.randn(case["partials"], rows, heads + 2 * kv_heads, dim, generator=gen, device=dev) / math.sqrt(case["partials"])
        x[:, :, heads: heads + kv_heads] *= size[0, :, 0]
        x[:, :, heads + kv_heads:] *= size[1, :, 0]
        state["qkv"] = x.reshape(case["partials"], rows, -1).to(F32 if case["wide"] else BF16)
        state["inv_freq"] = (500000.0 ** (-torch.arange(0, dim, 2, dtype=F64) / dim)).to(F32).to(dev)
        state["q"] = torch.zeros(rows, heads * dim, dtype=BF16, device=dev)
        return state
    state["q"] = (torch.randn(rows, heads * dim, generator=gen, device=dev)).to(BF16)
    state["out"] = torch.zeros(rows, heads * dim, dtype=BF16, device=dev)
    state["sink"] = torch.randn(heads, generator=gen, device=dev) if case["sink"] else None
    return state


# ----------------------------------------------------------------------------- plain forms

def _listed_in(counts, n):
    """For entries 0 .. n - 1 of the lists of `counts` entries behind one another: whose entry it is (-1 behind the last) and
    its place in that list (0 behind the last)."""
    ends = counts.cumsum(0)
    i = torch.arange(n, device=counts.device)
    whose = torch.searchsorted(ends, i, right=True)
    inside = whose < counts.numel()
    safe = whose.clamp(max=counts.numel() - 1)
    return torch.where(inside, whose, -1), torch.where(inside, i - (ends - counts)[safe], 0)


def _plain_maps(state):
    case, page = state["case"], state["case"]["page"]
    heads, kv_heads, _dim = HEADS[case["heads"]]
    cached, q_len, pages, T = state["cached"].to(I64), state["q_len"].to(I64), state["pages"], state["rows"]
    S = cached.numel()
    kv_len = cached + q_len
    row_seq, within = _listed_in(q_len, T)
    positions = within + cached[row_seq]
    blocks = -(-kv_len // page)
    b = torch.arange(state["width"], device=cached.device)
    at = ((blocks.cumsum(0) - blocks)[:, None] + b).clamp(max=pages.numel() - 1)
    table = torch.where(b < blocks[:, None], pages[at], -1)
    slots = table[row_seq, positions // page].to(I64) * page + positions % page
    write_seq, write_at = _listed_in((kv_len - 1) // BLOCK - cached // BLOCK + 1, min(T, T // BLOCK + 2 * S))
    first = torch.where(write_seq >= 0, cached[write_seq.clamp(min=0)] // BLOCK, 0)
    packed = q_len * (heads // kv_heads)
    tile_seq, tile_index = _listed_in(torch.where(packed > FEW_ROWS, -(-packed // TILE_ROWS), 0), T * (heads // kv_heads) // TILE_ROWS + S)
    i32 = lambda x: x.to(I32)  # noqa: E731
    return {"q_start": i32(q_len.cumsum(0) - q_len), "q_len": i32(q_len), "kv_len": i32(kv_len), "positions": i32(positions),
            "row_seq": i32(row_seq), "slots": slots, "block_table": table, "write_seq": i32(write_seq),
            "write_block": i32(write_at + first), "tile_seq": i32(tile_seq), "tile_index": i32(tile_index)}


def _plain_append(state):
    case, maps, codes, scales = state["case"], state["maps"], state["codes"], state["scales"]
    heads, kv_heads, dim = HEADS[case["heads"]]
    n_pages, _two, _kv, page, _dim = codes.shape
    per_page = page // BLOCK
    T = state["rows"]
    x = state["qkv"].to(F64).sum(0).view(T, heads + 2 * kv_heads, dim)
    angle = maps["positions"].to(F64)[:, None, None] * state["inv_freq"].to(F64)
    lo, hi = x[:, : heads + kv_heads, : dim // 2], x[:, : heads + kv_heads, dim // 2:]
    turned = torch.cat([lo * angle.cos() - hi * angle.sin(), hi * angle.cos() + lo * angle.sin()], -1)
    state["q"].copy_(turned[:, :heads].reshape(T, -1))
    kv = torch.stack([turned[:, heads:], x[:, heads + kv_heads:]], 1)          # [T, K|V, kv head, dim]
    # the largest new entry of every block of the pool
    page_of, in_page = maps["slots"] // page, maps["slots"] % page
    block = page_of * per_page + in_page // BLOCK
    finite = kv.isfinite()
    largest = torch.where(finite, kv.abs(), 0).amax(-1)
    new = torch.zeros(n_pages * per_page, 2, kv_heads, dtype=F64, device=kv.device)
    new.scatter_reduce_(0, block[:, None, None].expand_as(largest), largest, "amax")
    spoilt = torch.zeros(n_pages * per_page, kv_heads, device=kv.device)
    spoilt.scatter_reduce_(0, block[:, None].expand(T, kv_heads), (~finite.all(-1)).any(1).to(F32), "amax")
    # the written blocks: their scales before and after, and what they held
    used = maps["write_seq"] >= 0
    seq = maps["write_seq"].clamp(min=0).to(I64)
    first = torch.where(used, maps["write_block"], maps["write_block"][0]).to(I64)
    seq = torch.where(used, seq, seq[0])                                       # padding names the first block again
    w_page = maps["block_table"][seq, first * BLOCK // page].to(I64)
    w_block = first % per_page
    opened = (state["cached"][seq] > first * BLOCK)[:, None, None]
    e = _exponents(new[w_page * per_page + w_block])
    before = scales[w_page, :, :, w_block]
    e_before = torch.where(opened & before.isfinite(), torch.frexp(before)[1] - 1, LEAST)
    e_after = torch.maximum(e, e_before)
    held = codes.view(n_pages, 2, kv_heads, per_page, BLOCK, dim)
    old = held[w_page, :, :, w_block]
    again = _quantised(old.view(F8).to(F32), (e_after - e_before)[..., None, None]).view(torch.uint8)
    grown = opened & before.isfinite() & (e_after > e_before)
    filled = torch.arange(BLOCK, device=kv.device) < (state["cached"][seq] - first * BLOCK)[:, None]      # positions of earlier steps
    held[w_page, :, :, w_block] = torch.where(grown[..., None, None] & filled[:, None, None, :, None], again, old)
    after = torch.ldexp(torch.ones((), device=kv.device), e_after)
    bad = (spoilt[w_page * per_page + w_block] > 0) | (opened[..., 0] & before[:, 0].isnan())
    after[:, 0] = torch.where(bad, math.nan, after[:, 0])
    scales[w_page, :, :, w_block] = after
    # the new codes
    exponent = torch.frexp(torch.where(scales.isnan(), 1.0, scales))[1] - 1
    mine = exponent[page_of, :, :, in_page // BLOCK]
    codes[page_of, :, :, in_page] = _quantised(torch.where(finite, kv, 0), mine[..., None]).view(torch.uint8)
    return {"q": state["q"], "codes": codes.view(F8), "scales": scales}


def _plain_attention(state):
    case, maps = state["case"], state["maps"]
    heads, kv_heads, dim = HEADS[case["heads"]]
    group, page, L, Q = heads // kv_heads, case["page"], state["keys"], state["longest"]
    dev = state["q"].device
    key = torch.arange(L, device=dev)
    held = maps["block_table"][:, key // page].clamp(min=0).to(I64)           # [S, L]

    def values(which):
        x = state["codes"][held, which, :, key % page].view(F8).to(F32)         # [S, L, kv head, dim]
        return (x * state["scales"][held, which, :, key % page // BLOCK][..., None]).permute(0, 2, 1, 3)

    i = torch.arange(Q, device=dev)
    row = (maps["q_start"][:, None] + i).clamp(max=state["rows"] - 1)           # [S, Q]
    q = state["q"].view(-1, kv_heads, group, dim)[row].to(F32)                  # [S, Q, kv head, group, dim]
    q = q.permute(0, 2, 1, 3, 4).reshape(-1, kv_heads, Q * group, dim)
    score = (q @ values(0).transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    position = (state["cached"][:, None] + i)[:, :, None]                       # [S, Q, 1]
    visible = (key <= position) & (key < maps["kv_len"][:, None, None])
    if case["window"]:
        visible &= key > position - case["window"]
    visible = visible.repeat_interleave(group, 1)[:, None]                      # [S, 1, Q * group, L]
    score = torch.where(visible, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    if state["sink"] is not None:
        sink = state["sink"].view(1, kv_heads, 1, group, 1).expand(-1, -1, Q, -1, -1).reshape(1, kv_heads, Q * group, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(score - torch.where(top.isfinite(), top, 0))
    total = p.sum(-1, keepdim=True)
    if state["sink"] is not None:
        total = total + torch.exp(sink - top)
    o = torch.where(total > 0, (p @ values(1)) / total, 0)
    o = o.view(-1, kv_heads, Q, group, dim).permute(0, 2, 1, 3, 4).reshape(-1, Q, heads * dim)
    seq = maps["row_seq"].to(I64)
    state["out"].copy_(o[seq, maps["positions"] - state["cached"][seq]])
    return state["out"]


# ----------------------------------------------------------------------------- one pass

def _handle(state):
    """What a program keeps beside its cache: the step's maps and the view of the cache."""
    from bare_cuda_4gib_b200.kernels import cache8, step_maps
    case = state["case"]
    heads, kv_heads, dim = HEADS[case["heads"]]
    tile_rows = TILE_ROWS if case["op"] == "maps" else cache8.tile_rows(dim)
    maps = step_maps.StepMaps(state["rows"], state["cached"].numel(), state["width"], case["page"], group=heads // kv_heads,
                              tile_rows=tile_rows, few_rows=FEW_ROWS, device="cuda")
    if case["op"] == "maps":
        return maps, None
    maps.build(state["cached"], state["q_len"], state["pages"], state["rows"], state["longest"], state["shortest"])
    return maps, cache8.view(state["codes"], state["scales"], maps.block_table)


def run(state):
    if not own:
        return {"maps": _plain_maps, "append": _plain_append, "attention": _plain_attention}[state["case"]["op"]](state)
    from bare_cuda_4gib_b200.kernels import cache8
    from bare_cuda_4gib_b200.kernels.lib import AttentionExtras, Partials
    case = state["case"]
    if "handle" not in state:
        state["handle"] = _handle(state)
    maps, cache = state["handle"]
    heads, _kv, dim = HEADS[case["heads"]]
    if case["op"] == "maps":
        maps.build(state["cached"], state["q_len"], state["pages"], state["rows"], state["longest"], state["shortest"])
        return {"q_start": maps.seq_q_start, "q_len": maps.seq_q_len, "kv_len": maps.seq_kv_len, "positions": maps.positions,
                "row_seq": maps.row_seq, "slots": maps.slots, "block_table": maps.block_table, "write_seq": maps.write_seq,
                "write_block": maps.write_block, "tile_seq": maps.tile_seq, "tile_index": maps.tile_index}
    if case["op"] == "append":
        cache8.append(Partials(state["qkv"], case["partials"]), state["q"], cache, maps, state["inv_freq"], heads)
        return {"q": state["q"], "codes": state["codes"].view(F8), "scales": state["scales"]}
    cache8.attention(state["q"], state["out"], cache, maps, heads, 1.0 / math.sqrt(dim), case["window"],
                     AttentionExtras(sink=state["sink"]) if state["sink"] is not None else None)
    return state["out"]


# ----------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    requests = _requests(case, 0)
    heads, kv_heads, dim = HEADS[case["heads"]]
    S, T = len(requests), sum(n for _, n in requests)
    if case["op"] == "maps":
        blocks = sum(-(-(c + n) // case["page"]) for c, n in requests)
        width = -(-max(c + n + 512 for c, n in requests) // case["page"])
        tiles = T * (heads // kv_heads) // TILE_ROWS + S
        return {"bytes": 4.0 * (2 * S + blocks + 3 * S + 4 * T + S * width + 2 * min(T, T // BLOCK + 2 * S) + 2 * tiles), "flops": 0.0}
    if case["op"] == "append":
        row = (heads + 2 * kv_heads) * dim
        written = sum((c + n - 1) // BLOCK - c // BLOCK + 1 for c, n in requests)
        return {"bytes": float(T * (row * case["partials"] * (4 if case["wide"] else 2) + heads * dim * 2 + 2 * kv_heads * dim)
                               + written * 2 * kv_heads * 4), "flops": 3.0 * T * (heads + kv_heads) * dim}
    nbytes = flops = 0.0
    for c, n in requests:
        w = case["window"] or c + n
        first = max(0, c - w + 1)
        nbytes += (c + n - first) * 2 * kv_heads * (dim + 4 / BLOCK) + n * heads * dim * 4
        flops += 4.0 * heads * dim * sum(min(c + i + 1, w) for i in range(n))
    return {"bytes": nbytes, "flops": flops}


# ----------------------------------------------------------------------------- the same from the definitions, in 64 bits

def _e4m3_values(dev):
    """The number that each of the 256 codes stands for: 1 sign, 4 exponent and 3 fraction bits, bias 7."""
    c = torch.arange(256, device=dev)
    exponent, fraction = (c >> 3) & 15, (c & 7).to(F64)
    size = torch.where(exponent == 0, fraction / 8 * 2.0 ** -6, (1 + fraction / 8) * 2.0 ** (exponent - 7).to(F64))
    size = torch.where((c & 127) == 127, math.nan, size)
    return torch.where(c >= 128, -size, size)


def _exact_append(state):
    """Block by block of 16 positions, each as the definition of the cache has it."""
    case = state["case"]
    heads, kv_heads, dim = HEADS[case["heads"]]
    page, half = case["page"], dim // 2
    dev = state["qkv"].device
    number = _e4m3_values(dev)
    steps = torch.sort(number[:127]).values                # the magnitudes that a code can have
    held = number[state["codes"].long()]
    scales = state["scales"].to(F64)

    def nearest(x):
        """x rounded to the nearest magnitude, ties to the even code."""
        size = x.abs()
        up = torch.searchsorted(steps, size).clamp(1, 126)
        below, above = steps[up - 1], steps[up]
        take_above = (size - below > above - size) | ((size - below == above - size) & (up % 2 == 0))
        return torch.where(take_above, above, below) * torch.where(x < 0, -1.0, 1.0)

    x = state["qkv"].to(F64).sum(0).view(state["rows"], heads + 2 * kv_heads, dim)
    q_out, row, page_start = [], 0, 0
    for c, n in _requests(case, state["seed"]):
        position = torch.arange(c, c + n, device=dev, dtype=F64)
        turn = torch.polar(torch.ones(n, half, dtype=F64, device=dev), position[:, None] * state["inv_freq"].to(F64))[:, None]
        mine = x[row: row + n]
        z = torch.complex(mine[:, : heads + kv_heads, :half], mine[:, : heads + kv_heads, half:]) * turn
        turned = torch.cat([z.real, z.imag], -1)
        q_out.append(turned[:, :heads].reshape(n, -1))
        kv = torch.stack([turned[:, heads:], mine[:, heads + kv_heads:]], 0)                       # [2, n, kv head, dim]
        for first in range(c // 16 * 16, c + n, 16):
            lo, hi = max(first, c), min(first + 16, c + n)
            p = int(state["pages"][page_start + first // page])
            new = kv[:, lo - c: hi - c]
            largest = new.abs().amax((1, 3))                                                    # [2, kv head]
            e = torch.ceil(torch.log2(largest / 448)).clamp(-100, 119)
            scale = 2.0 ** e
            at, b = first % page, first % page // 16
            if c > first:
                was = scales[p, :, :, b]
                scale = torch.maximum(scale, was)
                old = held[p, :, :, at: at + c - first]
                held[p, :, :, at: at + c - first] = nearest(old * (was / scale)[..., None, None])
            scales[p, :, :, b] = scale
            held[p, :, :, at + lo - first: at + hi - first] = nearest(new.transpose(1, 2) / scale[..., None, None])
        row, page_start = row + n, page_start + -(-(c + n) // page)
    return {"q": torch.cat(q_out), "codes": held, "scales": scales}


def _exact_attention(state):
    case = state["case"]
    heads, kv_heads, dim = HEADS[case["heads"]]
    page, group = case["page"], heads // kv_heads
    number = _e4m3_values(state["q"].device)
    out, row, page_start = [], 0, 0
    for c, n in _requests(case, state["seed"]):
        count = -(-(c + n) // page)
        p = state["pages"][page_start: page_start + count].long()
        kv = number[state["codes"][p].long()] * state["scales"][p].to(F64).repeat_interleave(16, -1)[..., None]
        k, v = kv.permute(1, 2, 0, 3, 4).reshape(2, kv_heads, count * page, dim)[:, :, : c + n]
        q = state["q"][row: row + n].to(F64).view(n, kv_heads, group, dim)
        s = torch.einsum("nhgd,hld->hgnl", q, k) / dim ** 0.5
        distance = torch.arange(c, c + n, device=q.device)[:, None] - torch.arange(c + n, device=q.device)
        hidden = (distance < 0) | ((distance >= case["window"]) if case["window"] else False)
        s.masked_fill_(hidden, -math.inf)
        if state["sink"] is not None:      # one more column, whose value is zero
            s = torch.cat([s, state["sink"].to(F64).view(kv_heads, group, 1, 1).expand(-1, -1, n, 1)], -1)
        w = torch.softmax(s, -1)[..., : c + n]
        out.append(torch.einsum("hgnl,hld->nhgd", w, v).reshape(n, heads * dim))
        row, page_start = row + n, page_start + count
    return torch.cat(out)


def exact(case, seed):
    if case["op"] == "maps":
        return None                        # whole numbers only
    state = prepare(case, seed)
    state["seed"] = seed
    return _exact_append(state) if case["op"] == "append" else _exact_attention(state)
