"""Rotary positions, a key-value cache held in 4 bits, and attention against
it: the calls that stand before and behind window attention in a language
model's layers, as cases to time and to compare.

Operands are [tokens, heads, d]; ``query_heads`` is a multiple of
``key_heads`` and consecutive query heads share a key head.

``rotary``    pairs of each head's elements turned by angles that positions
              of one or several axes and the pairs' frequencies give.
``turn_back`` the same's gradients: a turn by the angles' negatives.
``write``     packed tokens' keys and values quantised into the cache's pages,
              and read back as the attention of the same tokens takes them.
``read``      what sequences hold in the cache, as packed keys and values.
``decode``    one query for each sequence against the cache, over a sliding
              window with sinks.

A cache of 4 bits holds a row of d elements as d / 2 bytes of codes (element
2 j in the low half of byte j) and d / 32 scale bytes.  A code is a sign and
one of eight sizes, LEVELS; a scale byte b stands for 2^(b - 127), 255 for a
block that holds an infinity or NaN, all of which reads as NaN.  A block's
scale is the smallest power of two, from 2^-125 to 2^125, that 7 times covers
its largest size; values go to the nearest code, ties to the even one.

Lengths follow from a case alone, values from the seed.
"""
import math
import random

import torch

own = False

DEV = "cuda"
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

# what draw() spreads over: logarithms of sizes where the range passes a
# factor of ten
RANGES = {
    "tokens": (1, 65536),        # of a rotary call
    "write_tokens": (1, 32768),
    "context": (0, 4096),        # keys that were there before a call's tokens
    "sequences": (1, 64),
    "read_capacity": (1, 131072),  # longest sequence that is read back
    "batch": (1, 256),           # sequences of a token step
    "capacity": (1, 262144),     # longest sequence of a token step
    "window": (64, 262144),
    "elements": 4.0e8,           # of all operands of a rotary call, the most
    "cache": 6.0e8,              # elements of a key cache, the most
}


def listed():
    return [
        # The token step of a serving batch: one token of each of 64.
        {"name": "rotary_step", "op": "rotary", "dtype": "bf16", "tokens": 64,
         "axes": 1, "query_heads": 32, "key_heads": 8, "d": 128, "pairs": 64,
         "interleaved": False},
        # A long clip's patches: time, height and width.
        {"name": "rotary_video", "op": "rotary", "dtype": "bf16",
         "tokens": 32760, "axes": 3, "query_heads": 32, "key_heads": 8,
         "d": 128, "pairs": 64, "interleaved": False},
        # Gradients of an image model's step, in fp32: two axes, a part of
        # each head turned, neighbours in pairs.
        {"name": "turn_back_image", "op": "turn_back", "dtype": "f32",
         "tokens": 4097, "axes": 2, "query_heads": 12, "key_heads": 12,
         "d": 80, "pairs": 32, "interleaved": True},
        # A training step of packed documents.
        {"name": "turn_back_packed", "op": "turn_back", "dtype": "bf16",
         "tokens": 16384, "axes": 1, "query_heads": 16, "key_heads": 4,
         "d": 128, "pairs": 64, "interleaved": False},
        # One new token of each of 64 conversations.
        {"name": "write_step", "op": "write", "dtype": "bf16",
         "sequences": 64, "tokens": 64, "context": 8192, "page": 64,
         "key_heads": 8, "d": 128},
        # A serving batch of prompts of different lengths, one of them empty.
        {"name": "write_prompts", "op": "write", "dtype": "bf16",
         "sequences": 12, "tokens": 32768, "context": 0, "page": 64,
         "key_heads": 8, "d": 128},
        # Pieces of prompts of a small fp32 model, odd lengths, heads of 96.
        {"name": "write_pieces", "op": "write", "dtype": "f32",
         "sequences": 5, "tokens": 3001, "context": 1000, "page": 24,
         "key_heads": 3, "d": 96},
        # The earlier turns of two conversations of a small model.
        {"name": "read_turns", "op": "read", "dtype": "bf16", "batch": 2,
         "capacity": 700, "page": 16, "key_heads": 2, "d": 64},
        # The long contexts behind four prompts' next pieces.
        {"name": "read_context", "op": "read", "dtype": "bf16", "batch": 4,
         "capacity": 65536, "page": 64, "key_heads": 8, "d": 128},
        # One token of one conversation of a small model.
        {"name": "decode_one", "op": "decode", "dtype": "bf16", "batch": 1,
         "capacity": 500, "page": 0, "query_heads": 8, "key_heads": 2,
         "d": 64, "window": 256, "sinks": 4},
        # A token step of a serving batch over a paged cache; the largest.
        {"name": "decode_pages", "op": "decode", "dtype": "bf16", "batch": 64,
         "capacity": 20000, "page": 64, "query_heads": 32, "key_heads": 8,
         "d": 128, "window": 20000, "sinks": 0},
        # A few long conversations in fp32: odd heads, a window with sinks.
        {"name": "decode_f32", "op": "decode", "dtype": "f32", "batch": 5,
         "capacity": 100001, "page": 48, "query_heads": 12, "key_heads": 4,
         "d": 96, "window": 65537, "sinks": 7},
    ]


def _log(rng, lo, hi):
    """A whole number in lo..hi, spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(max(lo, 1)),
                                                      math.log(hi))))))


def draw(rng):
    case = {"op": rng.choice(("rotary", "turn_back", "write", "write", "read",
                              "decode", "decode", "decode")),
            "dtype": rng.choice(("bf16", "bf16", "f32"))}
    key_heads = rng.choice((1, 2, 3, 4, 8))
    query_heads = key_heads * rng.choice((1, 2, 3, 4, 8))
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("rotary", "turn_back"):
        d = rng.choice((8, 40, 64, 64, 80, 96, 128, 128, 128))
        pairs = d // 2 if rng.random() < 0.6 else rng.randint(1, d // 2)
        row = (query_heads + key_heads) * d * size // 2
        tokens = min(_log(rng, *RANGES["tokens"]),
                     int(RANGES["elements"] / row))
        return case | {"tokens": tokens, "axes": rng.choice((1, 1, 2, 3)),
                       "query_heads": query_heads, "key_heads": key_heads,
                       "d": d, "pairs": pairs,
                       "interleaved": rng.random() < 0.4}
    d = rng.choice((32, 64, 64, 96, 128, 128, 128))
    page = rng.choice((0, 16, 16, 24, 64, 64, 256))
    if case["op"] == "write":
        tokens = _log(rng, *RANGES["write_tokens"])
        return case | {"sequences": min(tokens,
                                        _log(rng, *RANGES["sequences"])),
                       "tokens": tokens,
                       "context": 0 if rng.random() < 0.4 else
                       _log(rng, 1, RANGES["context"][1]),
                       "page": page, "key_heads": key_heads, "d": d}
    batch = _log(rng, *RANGES["batch"])
    room = RANGES["cache"] / (batch * key_heads * d)
    if case["op"] == "read":
        room /= 4 * size // 2
        return case | {"batch": batch, "capacity": max(1, min(
            int(room), _log(rng, *RANGES["read_capacity"]))), "page": page,
            "key_heads": key_heads, "d": d}
    if case["dtype"] == "f32":
        room /= 2
    return case | {"batch": batch, "capacity": max(1, min(
        int(room), _log(rng, *RANGES["capacity"]))), "page": page,
        "query_heads": query_heads, "key_heads": key_heads, "d": d,
        "window": _log(rng, *RANGES["window"]),
        "sinks": rng.choice((0, 0, 1, 4, 16, 64))}


# ---- lengths, which follow from the case alone ------------------------------

def _lengths(case):
    """(tokens, keys) of each sequence: those of a call, and of its cache once
    they are in it.  Written: a ragged split of the tokens, the second of
    four and more sequences empty; one each where there are as many tokens as
    sequences.  Read and attended: all keys, the first sequence the longest."""
    if case["op"] == "write":
        n, total = case["sequences"], case["tokens"]
        rng = random.Random(f"{n} {total} {case['context']}")
        if n == total:
            tokens = [1] * n
        else:
            shares = [rng.uniform(0.2, 1.0) for _ in range(n)]
            if n >= 4:
                shares[1] = 0.0
            ends, run, whole = [], 0.0, sum(shares)
            for s in shares:
                run += s
                ends.append(min(total, int(total * run / whole)))
            ends[-1] = total
            tokens = [e - b for b, e in zip([0] + ends[:-1], ends)]
        return tokens, [t + rng.randint(case["context"] // 2, case["context"])
                        for t in tokens]
    rng = random.Random(f"{case['batch']} {case['capacity']}")
    cap = case["capacity"]
    keys = [cap] + [rng.randint((cap + 3) // 4, cap)
                    for _ in range(case["batch"] - 1)]
    return keys, keys


def _visible_keys(case):
    return [min(n, case["window"]) +
            min(case["sinks"], max(0, n - case["window"]))
            for n in _lengths(case)[1]]


# ---- inputs -----------------------------------------------------------------

def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _values(gen, dtype, *shape, spread=0.0):
    """Normal values, some channels wider than others where a projection's
    output is meant."""
    x = torch.empty(*shape, device=DEV, dtype=dtype)
    x.normal_(generator=gen)
    if spread:
        x *= torch.exp(spread * torch.randn(shape[-1], device=DEV,
                                            generator=gen)).to(x.dtype)
    return x


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=DEV)


def _positions(gen, case):
    """[axes, tokens]: places of a text that goes on from anywhere, or time,
    height and width of a clip's patches."""
    n, axes = case["tokens"], case["axes"]
    at = torch.arange(n, device=DEV)
    if axes == 1:
        start = torch.randint(0, 131072, (n,), device=DEV, generator=gen)
        return (start if n <= 256 else at + start[0])[None].to(torch.int32)
    wide = max(1, int(math.sqrt(n / (1 if axes == 2 else 16))))
    first = torch.randint(0, 4096, (axes, 1), device=DEV, generator=gen)
    grid = [at // (wide * wide), at // wide % wide, at % wide]
    return (torch.stack(grid[3 - axes:]) + first).to(torch.int32)


def _prepare_rotary(case, gen):
    n, h, hk, d = (case[k] for k in ("tokens", "query_heads", "key_heads", "d"))
    pairs, t = case["pairs"], _dtype(case)
    i = torch.arange(pairs, device=DEV)
    s = {"op": case["op"], "interleaved": case["interleaved"],
         "positions": _positions(gen, case),
         "frequencies": (10000.0 ** (-i.double() / pairs)).float(),
         # each axis takes a run of the pairs
         "pair_axes": None if case["axes"] == 1 else
         (i * case["axes"] // pairs).to(torch.int32),
         "query": _values(gen, t, n, h, d, spread=0.3),
         "key": _values(gen, t, n, hk, d, spread=0.3)}
    for name in ("query", "key"):
        s[name + "_output"] = torch.zeros_like(s[name])
    return s


def _prepare_pages(case, gen, keys):
    """A page table (None: a page for each sequence), and an empty cache whose
    pages hold a head's rows together."""
    hk, d = case["key_heads"], case["d"]
    if case["page"]:
        need = [-(-n // case["page"]) for n in keys]
        pages, width, page = sum(need), max(need), case["page"]
        order = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
        table = torch.full((len(keys), width), -1, dtype=torch.int32,
                           device=DEV)
        live = (torch.arange(width, device=DEV) <
                torch.tensor(need, device=DEV)[:, None])
        table[live] = order
    else:
        table, pages, page = None, len(keys), max(keys)

    def rows(n):
        return torch.zeros(pages, hk, page, n, dtype=torch.uint8,
                           device=DEV).transpose(1, 2)
    return {"page_table": table, "key_cache": (rows(d // 2), rows(d // 32)),
            "value_cache": (rows(d // 2), rows(d // 32))}


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if case["op"] in ("rotary", "turn_back"):
        return _prepare_rotary(case, gen)
    tokens, keys = _lengths(case)
    hk, d, t = case["key_heads"], case["d"], _dtype(case)
    s = {"op": case["op"], **_prepare_pages(case, gen, keys),
         "key_lengths": torch.tensor(keys, dtype=torch.int32, device=DEV)}
    if case["op"] != "write":
        # the cache holds normal values, channels of keys of several widths
        for name, spread in (("key", 0.3), ("value", 0.0)):
            codes, scales = s[name + "_cache"]
            step = max(1, (1 << 25) // (hk * codes.shape[1] * d))
            for a in range(0, len(codes), step):
                part = slice(a, a + step)
                codes[part], scales[part] = _quantise(_values(
                    gen, torch.float32, *codes[part].shape[:3], d,
                    spread=spread))
    if case["op"] == "decode":
        s["query"] = _values(gen, t, case["batch"], case["query_heads"], d,
                             spread=0.3)
        s |= {"output": torch.zeros_like(s["query"]),
              "alpha": 1.0 / math.sqrt(d), "window": case["window"],
              "sinks": case["sinks"]}
        return s
    n = sum(tokens)
    s["token_offsets"] = _offsets(tokens)
    if case["op"] == "write":
        s["new_key"] = _values(gen, t, n, hk, d, spread=0.3)
        s["new_value"] = _values(gen, t, n, hk, d)
        s["starts"] = s["key_lengths"] - torch.tensor(
            tokens, dtype=torch.int32, device=DEV)
    for name in ("key", "value"):
        s[name] = torch.zeros(n, hk, d, dtype=t, device=DEV)
    return s


# ---- one pass ---------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"rotary": _plain_rotary, "turn_back": _plain_rotary,
            "write": _plain_write, "read": _plain_read,
            "decode": _plain_decode}[s["op"]](s)


def _run_own(s):
    import sparsewavecomp_amd as sw
    if s["op"] in ("rotary", "turn_back"):
        call = sw.rotary if s["op"] == "rotary" else sw.rotary_backward
        call(s["positions"], s["frequencies"], s["pair_axes"], s["query"],
             s["key"], s["query_output"], s["key_output"], s["interleaved"])
        return {"query": s["query_output"], "key": s["key_output"]}
    if s["op"] == "decode":
        return {"output": sw.window_attention_decode_fp4(
            s["key_lengths"], s["page_table"], s["query"], s["key_cache"],
            s["value_cache"], s["output"], s["alpha"], s["window"],
            s["sinks"])}
    if s["op"] == "write":
        sw.fp4_cache_write(s["token_offsets"], s["key_lengths"],
                           s["page_table"], s["new_key"], s["new_value"],
                           s["key_cache"], s["value_cache"])
    sw.fp4_cache_read(s["token_offsets"], s.get("starts"), s["page_table"],
                      s["key_cache"], s["value_cache"], s["key"], s["value"])
    return {"key": s["key"], "value": s["value"]}


def _plain_rotary(s):
    pos, f = s["positions"], s["frequencies"]
    # (angles in 64 bits: far positions lose their turns in 32)
    if s["pair_axes"] is None:
        angle = pos[0].double()[:, None] * f.double()
    else:
        angle = pos.double()[s["pair_axes"].long()].t() * f.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if s["op"] == "turn_back":
        sin = -sin
    pairs, out = len(f), {}
    for name in ("query", "key"):
        x = s[name].float()
        if s["interleaved"]:
            a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        else:
            a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        y = x.clone()
        first, second = a * cos - b * sin, a * sin + b * cos
        if s["interleaved"]:
            y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = first, second
        else:
            y[..., :pairs], y[..., pairs:2 * pairs] = first, second
        out[name] = y.to(s[name].dtype)
    return out


def _power(e):
    """2^e as fp32, e whole numbers from -126 to 127."""
    return ((e + 127) << 23).view(torch.float32)


def _quantise(x):
    """Codes [..., d / 2] and scales [..., d / 32] of x [..., d]."""
    blocks = x.float().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    bad = ~torch.isfinite(blocks).all(-1)
    top = torch.where(bad, 1.0, top)
    # top = m 2^e, m in 1/2 .. 1: the scale is 2^(e - 3), or twice that where
    # m passes 7/8
    m, e = torch.frexp(top)
    e = (e - 3 + (m > 0.875).int()).clamp(-125, 125)
    e = torch.where(top == 0, -125, e)
    # (in two steps: 2^125 is a factor that fp32 holds, 2^-125 too)
    y = torch.where(bad[..., None], 0.0, blocks) * _power(-e)[..., None]
    size = y.abs()
    code = torch.zeros_like(size, dtype=torch.uint8)
    for i in range(1, 8):
        middle = (LEVELS[i - 1] + LEVELS[i]) / 2
        code += (size >= middle) if i % 2 == 0 else (size > middle)
    code += 8 * torch.signbit(y).to(torch.uint8)
    code = code.flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4),
            torch.where(bad, 255, e + 127).to(torch.uint8))


def _dequantise(codes, scales):
    """The fp32 values of codes [..., d / 2] and scales [..., d / 32]."""
    levels = torch.arange(8, device=codes.device)
    # 0, 1/2, then (2 + last bit) 2^(the others - 2)
    levels = torch.where(levels < 2, levels * 0.5,
                         (2.0 + levels % 2) * _power(levels.int() // 2 - 2))
    levels = torch.cat([levels, -levels])
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    x = levels[both.int()].unflatten(-1, (-1, 32))
    scale = scales.int()
    factor = torch.where(scale == 0, 0.5 * _power(scale - 126),
                         _power(scale.clamp(1, 254) - 127))
    factor = torch.where(scale == 255, math.nan, factor)
    return (x * factor[..., None]).flatten(-2)


def _places(s, j):
    """(page, slot) of the places j [sequences, n] of each sequence."""
    size = s["key_cache"][0].shape[1]
    table = s["page_table"]
    if table is None:
        page = torch.arange(len(j), device=j.device)[:, None].expand_as(j)
        return page, j.clamp(0, size - 1)
    page = torch.gather(table.long(), 1, (j // size).clamp(
        0, table.shape[1] - 1)).clamp(min=0)
    return page, j % size


def _token_places(s):
    """(page, slot) of each packed token, from its sequence's start on."""
    off = s["token_offsets"].long()
    token = torch.arange(s["key"].shape[0], device=off.device)
    seq = torch.searchsorted(off, token, right=True) - 1
    place = token - off[seq]
    if "starts" in s:
        place = place + s["starts"].long()[seq]
    size = s["key_cache"][0].shape[1]
    if s["page_table"] is None:
        return seq, place
    return s["page_table"].long()[seq, place // size], place % size


def _plain_write(s):
    at = _token_places(s)
    out = {}
    for name in ("key", "value"):
        codes, scales = s[name + "_cache"]
        codes[at], scales[at] = _quantise(s["new_" + name])
        out[name] = _dequantise(codes[at], scales[at]).to(s[name].dtype)
    return out


def _plain_read(s):
    at = _token_places(s)
    return {name: _dequantise(*(x[at] for x in s[name + "_cache"])).to(
        s[name].dtype) for name in ("key", "value")}


def _plain_decode(s):
    q, length = s["query"], s["key_lengths"].long()[:, None]
    b, h, d = q.shape
    size, hk = s["key_cache"][0].shape[1:3]
    table = s["page_table"]
    cap = size * (1 if table is None else table.shape[1])
    window, sinks = min(s["window"], cap), min(s["sinks"], cap)
    start = (length - window).clamp(min=0)
    i = torch.arange(sinks + window, device=q.device)
    j = torch.where(i < sinks, i, start + i - sinks)
    live = torch.where(i < sinks, j < start, j < length)
    page, slot = _places(s, j)

    def rows(cache):  # [b, hk, n, d]
        x = _dequantise(*(x[page, slot] for x in cache))
        return x.mul_(live[:, :, None, None]).transpose(1, 2)
    k = rows(s["key_cache"]).transpose(2, 3).contiguous()
    p = torch.matmul(q.float().view(b, hk, h // hk, d), k).mul_(s["alpha"])
    del k
    p = p.masked_fill_(~live[:, None, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == float("-inf"), 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1))
    o = torch.matmul(p, rows(s["value_cache"]).contiguous())
    return {"output": o.view(b, h, d).to(q.dtype)}


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("rotary", "turn_back"):
        n, heads = case["tokens"], case["query_heads"] + case["key_heads"]
        return {"bytes": 2 * n * heads * case["d"] * size +
                4 * n * case["axes"] + 4 * case["pairs"] * min(
                    2, case["axes"]),
                "flops": 6 * n * heads * case["pairs"]}
    tokens, keys = _lengths(case)
    row = case["key_heads"] * case["d"]
    held = row // 2 + row // 32  # bytes of a row of all heads in the cache
    if case["op"] == "read":
        return {"bytes": 2 * sum(tokens) * (held + row * size),
                "flops": 2 * sum(tokens) * row}
    if case["op"] == "write":
        # (codes and scales written and read back)
        return {"bytes": 2 * sum(tokens) * (2 * held + 2 * row * size),
                "flops": 6 * sum(tokens) * row}
    seen, wide = sum(_visible_keys(case)), case["query_heads"] * case["d"]
    return {"bytes": 2 * seen * held + 2 * case["batch"] * wide * size,
            "flops": 4 * seen * wide}


# ---- the definition in 64 bits ----------------------------------------------

def _exact_rotary(case, s):
    pairs, out = case["pairs"], {}
    axis = [0] * pairs if s["pair_axes"] is None else s["pair_axes"].tolist()
    pos = s["positions"].double()
    angle = torch.stack([pos[a] * f for a, f in zip(
        axis, s["frequencies"].double().tolist())], 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    if case["op"] == "turn_back":
        turn = turn.conj()
    for name in ("query", "key"):
        x = s[name].double()
        head, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
        shape = (pairs, 2) if case["interleaved"] else (2, pairs)
        z = head.unflatten(-1, shape)
        if not case["interleaved"]:
            z = z.transpose(-1, -2)
        z = torch.complex(z[..., 0].contiguous(), z[..., 1].contiguous()) * turn
        z = torch.view_as_real(z)
        if not case["interleaved"]:
            z = z.transpose(-1, -2)
        out[name] = torch.cat([z.flatten(-2), rest], -1)
    return out


def _rounded(x):
    """What the cache makes of x, by the nearest of the sizes that a code has;
    no input here is infinite or NaN."""
    blocks = x.double().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 7))  # (a first guess, put right below)
    for _ in range(2):
        e = torch.where(top > 7 * torch.exp2(e), e + 1, e)
        e = torch.where(top <= 7 * torch.exp2(e - 1), e - 1, e)
    scale = torch.exp2(torch.where(top > 0, e.clamp(-125, 125), -125.0))
    y = blocks / scale
    size, out = y.abs(), torch.zeros_like(y)
    # steps of 1/2 up to 2, of 1 up to 4, of 2 up to 6, halves to the even one
    for low, step in ((0.0, 0.5), (2.0, 1.0), (4.0, 2.0)):
        out = torch.where(size >= low, torch.round(size / step) * step, out)
    return (torch.copysign(out.clamp(max=6.0), y) * scale).flatten(-2)


def _held(s, name, i, n):
    """The first n rows of sequence i, [n, hk, d]."""
    codes, scales = s[name + "_cache"]
    j = torch.arange(n, device=DEV)
    page, size = torch.full_like(j, i), codes.shape[1]
    if s["page_table"] is not None:
        page, j = s["page_table"][i, j // size].long(), j % size
    codes, scales = codes[page, j].long(), scales[page, j].double()
    x = torch.zeros(*codes.shape[:-1], codes.shape[-1] * 2,
                    dtype=torch.float64, device=DEV)
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS),
                         dtype=torch.float64, device=DEV)
    x[..., 0::2], x[..., 1::2] = table[codes % 16], table[codes // 16]
    return x * torch.exp2(scales - 127).repeat_interleave(32, -1)


def _exact_decode(case, s):
    h, hk, d = case["query_heads"], case["key_heads"], case["d"]
    out = torch.zeros(case["batch"], h, d, dtype=torch.float64, device=DEV)
    for i, n in enumerate(_lengths(case)[1]):
        j = torch.arange(n, device=DEV)
        j = j[(j >= n - case["window"]) | (j < case["sinks"])]
        k = _held(s, "key", i, n)[j].permute(1, 2, 0).contiguous()
        v = _held(s, "value", i, n)[j].transpose(0, 1).contiguous()
        q = s["query"][i].double().view(hk, h // hk, d)
        p = torch.softmax(torch.bmm(q, k) * s["alpha"], -1)
        out[i] = torch.bmm(p, v).reshape(h, d)
    return {"output": out}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rotary", "turn_back"):
        return _exact_rotary(case, s)
    if case["op"] == "decode":
        return _exact_decode(case, s)
    if case["op"] == "write":
        return {name: _rounded(s["new_" + name]) for name in ("key", "value")}
    tokens, _ = _lengths(case)
    return {name: torch.cat([_held(s, name, i, n)
                             for i, n in enumerate(tokens)])
            for name in ("key", "value")}
