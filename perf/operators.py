"""Attention over a sliding window with sinks, and over a shared prefix: the
calls that a language model's training step, prompt pass and token loop make,
as cases to time and to compare.

Four operators over [tokens, heads, d] operands, in which ``query_heads`` is a
multiple of ``key_heads`` and consecutive query heads share a key head:

``window``   a prompt pass: every query sees its own key, the ``window - 1``
             keys before it and the first ``sinks`` keys of its sequence.
             Sequences lie packed behind each other; a sequence's queries are
             the last of its keys.
``train``    the same with its backward pass.
``decode``   one query for each sequence against a key-value cache of pages
             (``page`` > 0) or of one run of memory for each sequence.
``prefix``   one query for each sequence; all of them see the same prefix, and
             each the keys of its own cache behind it.

Lengths follow from a case alone, values from the seed.
"""
import math
import random

import torch

own = False

DEV = "cuda"
BLOCK = 128  # queries that the plain form takes together

# what draw() spreads over: logarithms of sizes where the range passes a
# factor of ten
RANGES = {
    "tokens": (1, 32768),        # packed queries of a prompt pass
    "sequences": (1, 64),
    "context": (0, 4096),        # keys that were there before a prompt's queries
    "window": (1, 8192),
    "train_tokens": (64, 16384),
    "train_window": (16, 2048),
    "batch": (1, 256),           # sequences of a token step
    "capacity": (1, 131072),     # longest sequence of a token step
    "decode_window": (64, 131072),
    "prefix": (1, 16384),
    "suffix": (1, 4096),
    "pairs_d": 1.0e11,           # visible pairs * query heads * d, the most
    "train_pairs_d": 3.0e10,
    "cache": 2.6e8,              # elements of a key cache, the most
}


def listed():
    return [
        # A short prompt of a small model, one sequence: the time of a call.
        {"name": "window_short", "op": "window", "dtype": "bf16",
         "sequences": 1, "tokens": 200, "context": 0, "query_heads": 8,
         "key_heads": 2, "d": 64, "window": 128, "sinks": 4},
        # A serving batch of prompts of different lengths, one of them empty.
        {"name": "window_ragged", "op": "window", "dtype": "bf16",
         "sequences": 12, "tokens": 16384, "context": 0, "query_heads": 32,
         "key_heads": 8, "d": 128, "window": 1024, "sinks": 4},
        # Pieces of long prompts, their earlier keys in place; odd lengths
        # and a head of 96.
        {"name": "window_pieces", "op": "window", "dtype": "bf16",
         "sequences": 5, "tokens": 2501, "context": 3001, "query_heads": 12,
         "key_heads": 4, "d": 96, "window": 2000, "sinks": 16},
        # One long document; the largest case.
        {"name": "window_long", "op": "window", "dtype": "bf16",
         "sequences": 1, "tokens": 65536, "context": 0, "query_heads": 16,
         "key_heads": 4, "d": 128, "window": 4096, "sinks": 16},
        # A training step's attention: packed documents, shared key heads.
        {"name": "train_packed", "op": "train", "dtype": "bf16",
         "sequences": 6, "tokens": 16384, "context": 0, "query_heads": 16,
         "key_heads": 4, "d": 128, "window": 1024, "sinks": 4},
        # The sequence and head of the sparse attention benchmark (8192, 64),
        # in fp32, eight heads of their own keys.
        {"name": "train_f32", "op": "train", "dtype": "f32", "sequences": 1,
         "tokens": 8192, "context": 0, "query_heads": 8, "key_heads": 8,
         "d": 64, "window": 512, "sinks": 0},
        # A small odd model in bf16: lengths and heads of no power of two.
        {"name": "train_odd", "op": "train", "dtype": "bf16", "sequences": 3,
         "tokens": 3001, "context": 0, "query_heads": 6, "key_heads": 2,
         "d": 80, "window": 300, "sinks": 3},
        # One token of one conversation of a small model.
        {"name": "decode_one", "op": "decode", "dtype": "bf16", "batch": 1,
         "capacity": 500, "page": 0, "query_heads": 8, "key_heads": 2,
         "d": 64, "window": 256, "sinks": 4},
        # A token step of a serving batch over a paged cache.
        {"name": "decode_pages", "op": "decode", "dtype": "bf16", "batch": 64,
         "capacity": 16384, "page": 64, "query_heads": 32, "key_heads": 8,
         "d": 128, "window": 4096, "sinks": 4},
        # A few long conversations, each cache one run of memory.
        {"name": "decode_long", "op": "decode", "dtype": "bf16", "batch": 4,
         "capacity": 131072, "page": 0, "query_heads": 32, "key_heads": 8,
         "d": 128, "window": 65536, "sinks": 4},
        # A few answers to one question, in fp32.
        {"name": "prefix_few", "op": "prefix", "dtype": "f32", "batch": 4,
         "prefix": 1000, "capacity": 60, "page": 16, "query_heads": 8,
         "key_heads": 2, "d": 64},
        # Many requests behind one long system prompt.
        {"name": "prefix_many", "op": "prefix", "dtype": "bf16",
         "batch": 128, "prefix": 16384, "capacity": 2048, "page": 64,
         "query_heads": 32, "key_heads": 8, "d": 128},
    ]


def _log(rng, lo, hi):
    """A whole number in lo..hi, spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(max(lo, 1)),
                                                      math.log(hi))))))


def draw(rng):
    case = {"op": rng.choice(("window", "window", "train", "train", "decode",
                              "decode", "prefix")),
            "dtype": rng.choice(("bf16", "bf16", "f32"))}
    key_heads = rng.choice((1, 2, 3, 4, 8))
    heads = {"query_heads": key_heads * rng.choice((1, 2, 3, 4, 8)),
             "key_heads": key_heads,
             "d": rng.choice((8, 40, 64, 64, 80, 96, 128, 128, 128))}
    hd = heads["query_heads"] * max(64, heads["d"])
    sinks = rng.choice((0, 0, 1, 4, 16, 64))
    if case["op"] in ("window", "train"):
        training = case["op"] == "train"
        lo, hi = RANGES["train_tokens" if training else "tokens"]
        tokens = _log(rng, lo, hi)
        window = _log(rng, *RANGES["train_window" if training else "window"])
        most = RANGES["train_pairs_d" if training else "pairs_d"] / hd
        if case["dtype"] == "f32":
            most /= 8
        context = 0 if training or rng.random() < 0.6 else \
            _log(rng, 1, RANGES["context"][1])
        seen = min(window + sinks, tokens + context)
        tokens = max(1, min(tokens, int(most / seen)))
        case |= {"sequences": min(tokens, _log(rng, *RANGES["sequences"])),
                 "tokens": tokens, "context": context, **heads,
                 "window": window, "sinks": sinks}
        return case
    batch = _log(rng, *RANGES["batch"])
    row = heads["key_heads"] * heads["d"] * (2 if case["dtype"] == "f32" else 1)
    room = max(1, int(RANGES["cache"] / (batch * row)))
    page = rng.choice((0, 16, 16, 24, 64, 256))
    if case["op"] == "decode":
        capacity = min(room, _log(rng, *RANGES["capacity"]))
        case |= {"batch": batch, "capacity": capacity, "page": page, **heads,
                 "window": _log(rng, *RANGES["decode_window"]),
                 "sinks": sinks}
    else:
        case |= {"batch": batch, "prefix": _log(rng, *RANGES["prefix"]),
                 "capacity": min(room, _log(rng, *RANGES["suffix"])),
                 "page": page, **heads}
    return case


# ---- lengths, which follow from the case alone ------------------------------

def _packed_lengths(case):
    """(queries, keys) of each sequence: a ragged split of the tokens, the
    second of four and more sequences empty."""
    n, total = case["sequences"], case["tokens"]
    rng = random.Random(f"{n} {total} {case['context']}")
    shares = [rng.uniform(0.2, 1.0) for _ in range(n)]
    if n >= 4:
        shares[1] = 0.0
    ends, run, whole = [], 0.0, sum(shares)
    for s in shares:
        run += s
        ends.append(min(total, int(total * run / whole)))
    ends[-1] = total
    queries = [e - b for b, e in zip([0] + ends[:-1], ends)]
    keys = [q + (rng.randint(case["context"] // 2, case["context"])
                 if q else 0) for q in queries]
    return queries, keys


def _cache_lengths(case):
    """Keys of each sequence of a token step, the first the longest."""
    rng = random.Random(f"{case['batch']} {case['capacity']}")
    cap = case["capacity"]
    return [cap] + [rng.randint((cap + 3) // 4, cap)
                    for _ in range(case["batch"] - 1)]


def _visible_pairs(case):
    pairs = 0
    w, s = case["window"], case["sinks"]
    for q, k in zip(*_packed_lengths(case)):
        for p in range(k - q, k):
            first = max(0, p - w + 1)
            pairs += p + 1 - first + min(s, first)
    return pairs


def _visible_keys(case):
    return [min(n, case["window"]) +
            min(case["sinks"], max(0, n - case["window"]))
            for n in _cache_lengths(case)]


# ---- inputs -----------------------------------------------------------------

def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _values(gen, case, *shape, spread=0.0):
    """Normal values, some channels wider than others where a projection's
    output is meant."""
    x = torch.empty(*shape, device=DEV, dtype=_dtype(case))
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


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    h, hk, d = case["query_heads"], case["key_heads"], case["d"]
    s = {"op": case["op"], "alpha": 1.0 / math.sqrt(d),
         "window": case.get("window", 0), "sinks": case.get("sinks", 0)}
    if case["op"] in ("window", "train"):
        queries, keys = _packed_lengths(case)
        tq, tk = sum(queries), sum(keys)
        s["query_offsets"] = _offsets(queries)
        s["key_offsets"] = (s["query_offsets"] if queries == keys
                            else _offsets(keys))
        s["query"] = _values(gen, case, tq, h, d, spread=0.3)
        s["key"] = _values(gen, case, tk, hk, d, spread=0.3)
        s["value"] = _values(gen, case, tk, hk, d)
        s["output"] = torch.zeros_like(s["query"])
        if case["op"] == "train":
            s["output_gradient"] = _values(gen, case, tq, h, d)
            s["log_sum"] = torch.zeros(h, tq, device=DEV)
            for name in ("query", "key", "value"):
                s[name + "_gradient"] = torch.zeros_like(s[name])
        return s
    batch, lengths = case["batch"], _cache_lengths(case)
    s["key_lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    s["query"] = _values(gen, case, batch, h, d, spread=0.3)
    s["output"] = torch.zeros_like(s["query"])
    if case["page"]:
        need = [-(-n // case["page"]) for n in lengths]
        pages, width = sum(need), max(need)
        order = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
        table = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
        live = (torch.arange(width, device=DEV) <
                torch.tensor(need, device=DEV)[:, None])
        table[live] = order
        s["page_table"], shape = table, (pages, case["page"], hk, d)
    else:
        s["page_table"], shape = None, (batch, case["capacity"], hk, d)
    s["key_cache"] = _values(gen, case, *shape, spread=0.3)
    s["value_cache"] = _values(gen, case, *shape)
    if case["op"] == "prefix":
        s["prefix_key"] = _values(gen, case, case["prefix"], hk, d, spread=0.3)
        s["prefix_value"] = _values(gen, case, case["prefix"], hk, d)
    return s


# ---- one pass ---------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    return {"window": _plain_window, "train": _plain_window,
            "decode": _plain_decode, "prefix": _plain_prefix}[s["op"]](s)


def _run_own(s):
    import sparsewavecomp_amd as sw
    if s["op"] == "decode":
        return {"output": sw.window_attention_decode(
            s["key_lengths"], s["page_table"], s["query"], s["key_cache"],
            s["value_cache"], s["output"], s["alpha"], s["window"],
            s["sinks"])}
    if s["op"] == "prefix":
        return {"output": sw.shared_prefix_attention(
            s["key_lengths"], s["page_table"], s["query"], s["prefix_key"],
            s["prefix_value"], s["key_cache"], s["value_cache"], s["output"],
            s["alpha"])}
    out = {"output": sw.window_attention(
        s["query_offsets"], s["key_offsets"], s["query"], s["key"],
        s["value"], s["output"], s.get("log_sum"), s["alpha"], s["window"],
        s["sinks"])}
    if s["op"] == "train":
        sw.window_attention_backward(
            s["query_offsets"], s["key_offsets"], s["query"], s["key"],
            s["value"], s["output"], s["log_sum"], s["output_gradient"],
            s["query_gradient"], s["key_gradient"], s["value_gradient"],
            s["alpha"], s["window"], s["sinks"])
        out |= {k: s[k] for k in ("log_sum", "query_gradient", "key_gradient",
                                  "value_gradient")}
    return out


def _heads_first(x, hk):
    """[n, rows, heads, d] as contiguous fp32 [n, hk, heads / hk * rows, d]."""
    n, rows, h, d = x.shape
    x = x.float().view(n, rows, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    return x.reshape(n, hk, h // hk * rows, d)


def _rows_first(x, h):
    """The inverse of _heads_first: [n, rows, h, d]."""
    n, hk, gr, d = x.shape
    g = h // hk
    return x.view(n, hk, g, gr // g, d).permute(0, 3, 1, 2, 4).reshape(
        n, gr // g, h, d)


def _plain_window(s):
    """Blocks of BLOCK queries of one sequence each, against the gathered
    keys of their windows and the sinks before them."""
    q, k, v = s["query"], s["key"], s["value"]
    tq, h, d = q.shape
    tk, hk, _ = k.shape
    g, dev = h // hk, q.device
    window, sinks = min(s["window"], tk), min(s["sinks"], tk)
    qo, ko = s["query_offsets"].long(), s["key_offsets"].long()
    n = qo.numel() - 1
    # sequence i has the blocks from qo[i] // BLOCK + i on
    first = qo[:-1] // BLOCK + torch.arange(n, device=dev)
    block = torch.arange(tq // BLOCK + n, device=dev)
    seq = torch.searchsorted(first, block, right=True) - 1
    row = ((block - first[seq]) * BLOCK)[:, None] + torch.arange(
        BLOCK, device=dev)
    live = row < (qo[1:] - qo[:-1])[seq][:, None]
    at = torch.where(live, qo[seq][:, None] + row, 0)
    lk = (ko[1:] - ko[:-1])[seq][:, None]
    pos = row + lk - (qo[1:] - qo[:-1])[seq][:, None]
    # keys: the sinks, then the run from the first query's window on
    j = torch.cat([torch.arange(sinks, device=dev).expand(len(block), -1),
                   pos[:, :1] - window + 1 + torch.arange(
                       window + BLOCK - 1, device=dev)], 1)
    sink = torch.arange(j.shape[1], device=dev) < sinks
    jj, pp = j[:, None, :], pos[:, :, None]
    see = (jj >= 0) & (jj <= pp) & live[:, :, None] & torch.where(
        sink, jj <= pp - window, jj > pp - window)
    src = (ko[seq][:, None] + j.clamp(min=0)).clamp(max=tk - 1)
    inside = ((j >= 0) & (j < lk))[:, :, None, None]
    qb = _heads_first(q[at], hk)
    kb = _heads_first(torch.where(inside, k[src], 0), hk)
    vb = _heads_first(torch.where(inside, v[src], 0), hk)
    shape = (len(block), hk, g, BLOCK, j.shape[1])
    p = torch.matmul(qb, kb.transpose(2, 3).contiguous())
    p = p.mul_(s["alpha"]).view(shape).masked_fill_(
        ~see[:, None, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0, top)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1)).view(
        len(block), hk, g * BLOCK, -1)
    o = _rows_first(torch.matmul(p, vb), h)
    out = torch.zeros_like(q)
    to = at[live]
    out[to] = o[live].to(q.dtype)
    if s["op"] == "window":
        return {"output": out}
    log_sum = torch.zeros(h, tq, device=dev)
    lse = (top + total.log()).view(len(block), h, BLOCK).transpose(1, 2)
    log_sum[:, to] = lse[live].t()
    do = _heads_first(s["output_gradient"][at] * live[:, :, None, None], hk)
    ds = torch.matmul(do, vb.transpose(2, 3).contiguous())
    ds = ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(s["alpha"])
    dq = torch.zeros_like(q)
    dq[to] = _rows_first(torch.matmul(ds, kb), h)[live].to(q.dtype)
    grads = {}
    for name, left, right in (("key", ds, qb), ("value", p, do)):
        x = torch.matmul(left.transpose(2, 3).contiguous(), right)
        x = x.transpose(1, 2).reshape(-1, hk, d)
        grads[name] = torch.zeros(tk, hk, d, device=dev).index_add_(
            0, src.view(-1), x).to(q.dtype)
    return {"output": out, "log_sum": log_sum, "query_gradient": dq,
            "key_gradient": grads["key"], "value_gradient": grads["value"]}


def _cached(cache, table, j, live):
    """Rows j [batch, n] of each sequence's cache, [batch, n, hk, d]; zero
    where not live."""
    j = j.clamp(min=0)
    if table is None:
        page = torch.arange(j.shape[0], device=j.device)[:, None].expand_as(j)
        slot = j.clamp(max=cache.shape[1] - 1)
    else:
        slot = j % cache.shape[1]
        page = torch.gather(table.long(), 1, (j // cache.shape[1]).clamp(
            max=table.shape[1] - 1)).clamp(min=0)
    return torch.where(live[:, :, None, None], cache[page, slot], 0)


def _capacity(s):
    table = s["page_table"]
    return s["key_cache"].shape[1] * (1 if table is None else table.shape[1])


def _softmax(p):
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == float("-inf"), 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total > 0, total, 1))


def _plain_decode(s):
    q, length = s["query"], s["key_lengths"].long()[:, None]
    b, h, d = q.shape
    hk, cap = s["key_cache"].shape[2], _capacity(s)
    window, sinks = min(s["window"], cap), min(s["sinks"], cap)
    start = (length - window).clamp(min=0)
    i = torch.arange(sinks + window, device=q.device)
    j = torch.where(i < sinks, i, start + i - sinks)
    live = torch.where(i < sinks, j < start, j < length)
    k = _heads_first(_cached(s["key_cache"], s["page_table"], j, live), hk)
    v = _heads_first(_cached(s["value_cache"], s["page_table"], j, live), hk)
    p = torch.matmul(q.float().view(b, hk, h // hk, d),
                     k.transpose(2, 3).contiguous()).mul_(s["alpha"])
    p = _softmax(p.masked_fill_(~live[:, None, None], float("-inf")))
    return {"output": torch.matmul(p, v).view(b, h, d).to(q.dtype)}


def _plain_prefix(s):
    q, length = s["query"], s["key_lengths"].long()[:, None]
    b, h, d = q.shape
    hk, g = s["key_cache"].shape[2], h // s["key_cache"].shape[2]
    j = torch.arange(_capacity(s), device=q.device).expand(b, -1)
    live = j < length
    k = _heads_first(_cached(s["key_cache"], s["page_table"], j, live), hk)
    v = _heads_first(_cached(s["value_cache"], s["page_table"], j, live), hk)
    qh = q.float().view(b, hk, g, d)
    tail = torch.matmul(qh, k.transpose(2, 3).contiguous()).masked_fill_(
        ~live[:, None, None], float("-inf"))
    # the prefix once for all: the queries of a key head are one matrix
    qp = qh.transpose(0, 1).reshape(hk, b * g, d)
    pk = s["prefix_key"].float().permute(1, 2, 0).contiguous()
    pv = s["prefix_value"].float().transpose(0, 1).contiguous()
    head = torch.matmul(qp, pk).view(hk, b, g, -1).transpose(0, 1)
    n = head.shape[-1]
    p = _softmax(torch.cat([head, tail], -1).mul_(s["alpha"]))
    o = torch.matmul(p[..., n:].contiguous(), v)
    o += torch.matmul(p[..., :n].transpose(0, 1).reshape(hk, b * g, n),
                      pv).view(hk, b, g, d).transpose(0, 1)
    return {"output": o.reshape(b, h, d).to(q.dtype)}


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    h, hk, d = case["query_heads"], case["key_heads"], case["d"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("window", "train"):
        queries, keys = _packed_lengths(case)
        tq, tk = sum(queries), sum(keys)
        pairs = _visible_pairs(case) * h * d
        rows = 2 * tq * h * d + 2 * tk * hk * d
        if case["op"] == "window":
            return {"bytes": rows * size, "flops": 4 * pairs}
        return {"bytes": 2 * rows * size + 4 * tq * h, "flops": 14 * pairs}
    lengths = (_visible_keys(case) if case["op"] == "decode"
               else _cache_lengths(case))
    pairs, keys = sum(lengths), sum(lengths)
    if case["op"] == "prefix":
        pairs += case["batch"] * case["prefix"]
        keys += case["prefix"]
    return {"bytes": size * (2 * case["batch"] * h * d + 2 * keys * hk * d),
            "flops": 4 * pairs * h * d}


# ---- the definition in 64 bits ----------------------------------------------

def _attend(q, k, v, see, alpha):
    """softmax(alpha q k^T) v of [heads, rows, d] operands in float64 over the
    pairs that `see` marks; also the probabilities and the logarithms of the
    sums."""
    score = torch.bmm(q, k.transpose(1, 2).contiguous()) * alpha
    score = score.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(score, -1, keepdim=True)
    p = torch.where(see, torch.exp(score - lse), 0.0)
    return torch.bmm(p, v), p, lse[..., 0]


def _exact_window(case, s):
    g = case["query_heads"] // case["key_heads"]
    grads = case["op"] == "train"
    out = {"output": torch.zeros_like(s["query"], dtype=torch.float64)}
    if grads:
        out["log_sum"] = torch.zeros_like(s["log_sum"], dtype=torch.float64)
        for name in ("query", "key", "value"):
            out[name + "_gradient"] = torch.zeros_like(
                s[name], dtype=torch.float64)
    q0 = k0 = 0
    for nq, nk in zip(*_packed_lengths(case)):
        for a in range(0, nq, 1024):
            b = min(nq, a + 1024)
            pos = torch.arange(nk - nq + a, nk - nq + b, device=DEV)
            low = max(0, int(pos[0]) - case["window"] + 1)
            lead = min(case["sinks"], low)
            j = torch.cat([torch.arange(lead, device=DEV),
                           torch.arange(low, int(pos[-1]) + 1, device=DEV)])
            see = (j <= pos[:, None]) & ((j > pos[:, None] - case["window"]) |
                                         (j < case["sinks"]))
            qd = s["query"][q0 + a:q0 + b].double()
            kd, vd = s["key"][k0 + j].double(), s["value"][k0 + j].double()
            for hk in range(case["key_heads"]):
                of = slice(hk * g, hk * g + g)
                qh = qd[:, of].transpose(0, 1).contiguous()
                kh = kd[:, hk].expand(g, -1, -1).contiguous()
                vh = vd[:, hk].expand(g, -1, -1).contiguous()
                o, p, lse = _attend(qh, kh, vh, see, s["alpha"])
                out["output"][q0 + a:q0 + b, of] = o.transpose(0, 1)
                if not grads:
                    continue
                out["log_sum"][of, q0 + a:q0 + b] = lse
                do = s["output_gradient"][q0 + a:q0 + b, of].double()
                do = do.transpose(0, 1).contiguous()
                dp = torch.bmm(do, vh.transpose(1, 2).contiguous())
                ds = p * (dp - (do * o).sum(-1, keepdim=True)) * s["alpha"]
                out["query_gradient"][q0 + a:q0 + b, of] = torch.bmm(
                    ds, kh).transpose(0, 1)
                for name, x, y in (("key", ds, qh), ("value", p, do)):
                    out[name + "_gradient"][k0 + j, hk] += torch.bmm(
                        x.transpose(1, 2).contiguous(), y).sum(0)
        q0, k0 = q0 + nq, k0 + nk
    return out


def _exact_step(case, s):
    g = case["query_heads"] // case["key_heads"]
    out = torch.zeros_like(s["query"], dtype=torch.float64)
    for i, n in enumerate(_cache_lengths(case)):
        j = torch.arange(n, device=DEV)
        if case["op"] == "decode":
            j = j[(j >= n - case["window"]) | (j < case["sinks"])]
        rows = []
        for name in ("key", "value"):
            cache = s[name + "_cache"]
            if case["page"]:
                x = cache[s["page_table"][i, j // case["page"]].long(),
                          j % case["page"]]
            else:
                x = cache[i, j]
            x = x.double()
            if case["op"] == "prefix":
                x = torch.cat([s["prefix_" + name].double(), x])
            rows.append(x.transpose(0, 1).contiguous())
        q = s["query"][i].double().view(case["key_heads"], g, case["d"])
        see = torch.ones(1, dtype=torch.bool, device=DEV)
        out[i] = _attend(q, *rows, see, s["alpha"])[0].reshape(out[i].shape)
    return {"output": out}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("window", "train"):
        return _exact_window(case, s)
    return _exact_step(case, s)
