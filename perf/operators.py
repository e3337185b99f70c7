"""The paged key/value cache in 8 bits and the attention that reads it, as measurable cases.

    update   appends the new tokens of several sequences: queries and keys are rotated to their positions, keys and values
             go to the sequences' pages as 8-bit codes with one scale for each page and head (PagedKVCache.Update), then the
             pages that were written are read back (PagedKVCache.read)
    read     pages back as values (PagedKVCache.read)
    attend   causal attention of the last tokens of every sequence over its pages (PagedKVCache.attention): one token for
             each (a decode step), a few (drafts), or many (a prompt, or a chunk of one behind a filled cache)

What a page holds: keys [kv_heads, page, head_dim] and values [kv_heads, head_dim, page] as e4m3 numbers, and for each head the
scales of its keys and of its values, powers of two.  A block's scale is the smallest one, 2^-40 at least, under which every
magnitude that entered the block since its first token fits 448; where it grows, the tokens that are there are rounded again.
Position p of sequence s is token p % page of page table[s, p / page]; `lengths` counts the tokens with the new ones.

Head counts are those of the two decoder configurations and of common grouped-query decoders.
"""
import math
import random

import torch

own = False

FLOOR = -40  # exponent of the smallest scale
SIZE = {"f32": 4, "bf16": 2}
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
HEADS = [(16, 8, 128), (32, 8, 128), (14, 2, 64), (8, 8, 64), (40, 8, 128), (24, 8, 128), (16, 1, 128), (12, 4, 64)]


def listed():
    return [
        # one chat: the newest token of one sequence enters the cache of one layer of the small model
        {"name": "update-one", "kind": "update", "heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "batch": 1, "ctx": 1000, "rows": 1, "type": "f32"},
        # a server's step: 64 sequences of their own lengths, one token each
        {"name": "update-batch", "kind": "update", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "batch": 64, "ctx": 4000, "rows": 1, "type": "bf16"},
        # three prompts of different lengths enter in one call
        {"name": "update-prompt", "kind": "update", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "batch": 3, "ctx": 3000, "rows": 2500, "type": "f32"},
        # one sequence's cache leaves for a snapshot
        {"name": "read-one", "kind": "read", "heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "batch": 1, "ctx": 2000, "rows": 1, "type": "f32"},
        # the caches of 32 sequences move to another place
        {"name": "read-many", "kind": "read", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "batch": 32, "ctx": 4096, "rows": 1, "type": "bf16"},
        # one chat with the small model: latency
        {"name": "decode-one", "kind": "attend", "heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "batch": 1, "ctx": 1000, "rows": 1, "window": 0, "type": "f32"},
        # one sequence with a long context: its work is split over the device
        {"name": "decode-long", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "batch": 1, "ctx": 30001, "rows": 1, "window": 0, "type": "f32"},
        # a full server: 64 sequences, the lengths from a few tokens to the longest
        {"name": "decode-batch", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "batch": 64, "ctx": 8000, "rows": 1, "window": 0, "type": "bf16"},
        # five drafted tokens for each of eight sequences, small pages and heads, an uneven group
        {"name": "draft", "kind": "attend", "heads": 14, "kv_heads": 2, "dim": 64, "page": 16, "batch": 8, "ctx": 1999, "rows": 5, "window": 0, "type": "bf16"},
        # an ordinary prompt in fp32
        {"name": "prompt-f32", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "batch": 1, "ctx": 777, "rows": 777, "window": 0, "type": "f32"},
        # a long prompt
        {"name": "prompt-long", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "batch": 1, "ctx": 6000, "rows": 6000, "window": 0, "type": "bf16"},
        # chunks of three prompts behind what is cached of them
        {"name": "prompt-chunks", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "batch": 3, "ctx": 5500, "rows": 512, "window": 0, "type": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    heads, kv_heads, dim = rng.choice(HEADS)
    case = {"kind": rng.choice(["update", "update", "read", "attend", "attend", "attend", "attend"]), "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": rng.choice([16, 32, 64]), "type": rng.choice(["f32", "bf16"])}
    if case["kind"] == "read":
        case |= {"batch": _spread(rng, 1, 32), "ctx": _spread(rng, 1, 4096), "rows": 1}
    elif case["kind"] == "update":
        if rng.random() < 0.5:  # a step
            case |= {"batch": _spread(rng, 1, 64), "rows": _spread(rng, 1, 6)}
        else:
            case |= {"batch": rng.randint(1, 3), "rows": _spread(rng, 17, 2500)}
        case["ctx"] = case["rows"] + _spread(rng, 1, 4000) - 1
    else:
        long = rng.random()
        if long < 0.5:
            case |= {"batch": _spread(rng, 1, 64), "rows": 1, "ctx": _spread(rng, 1, 8000)}
        elif long < 0.65:
            case |= {"batch": _spread(rng, 1, 16), "rows": rng.randint(2, 8)}
            case["ctx"] = case["rows"] + _spread(rng, 1, 4000)
        else:
            case |= {"batch": rng.randint(1, 3), "rows": _spread(rng, 17, 1500)}
            case["ctx"] = case["rows"] + _spread(rng, 1, 4000) - 1
        case["window"] = _spread(rng, 100, 2000) if rng.random() < 0.25 else 0
    return case


def _shape(case):
    """Rows and lengths of the sequences: the first has the sizes that the case names, the others less.  Where a batch of single tokens is
    large, its last slot is empty: a server fills its batch up."""
    r = random.Random("%(batch)s %(ctx)s %(rows)s" % case)
    rows, lens = [case["rows"]], [case["ctx"]]
    for _ in range(case["batch"] - 1):
        n = case["rows"] if case["rows"] <= 8 else r.randint(1, case["rows"])
        rows.append(n)
        lens.append(max(n, int(case["ctx"] * r.uniform(0.05, 1.0))))
    if case["rows"] == 1 and case["batch"] >= 8 and case["kind"] == "attend":
        lens[-1] = 0
    return rows, lens


def _pairs(case):
    """(query row, key) pairs that see each other, and keys that some row sees."""
    pairs = keys = 0
    window = case.get("window", 0)
    for n, length in zip(*_shape(case)):
        for p in range(length - n, length):
            if p >= 0:
                pairs += min(p + 1, window) if window else p + 1
        first = max(0, length - n + 1 - window) if window else 0
        keys += max(0, length - first)
    return pairs, keys


def work(case):
    rows, lens = _shape(case)
    total, size, dim, kvh = sum(rows), SIZE[case["type"]], case["dim"], case["kv_heads"]
    token = 2 * kvh * dim
    if case["kind"] == "attend":
        pairs, keys = _pairs(case)
        return {"bytes": keys * token + 8 * kvh * -(-keys // case["page"]) + 2 * total * case["heads"] * dim * size, "flops": 4.0 * pairs * case["heads"] * dim}
    if case["kind"] == "read":
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": pages * (case["page"] * token * (1 + size) + 8 * kvh), "flops": pages * case["page"] * token}
    pages = sum((n - 1) // case["page"] - (n - r) // case["page"] + 1 for r, n in zip(rows, lens))
    back = pages * (case["page"] * token * 3 + 8 * kvh)  # bytes and bfloat16 values of the pages that are read back
    return {"bytes": total * (token * (size + 1) + 2 * case["heads"] * dim * size) + back, "flops": 3.0 * total * dim * (kvh + case["heads"])}


# ------------------------------------------------------------------------------------------------ inputs from the seed
def _gen(seed, tag):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + tag)


def _randn(shape, seed, tag):
    return torch.randn(shape, generator=_gen(seed, tag), device="cuda")


def _exponent(amax):
    """Exponent of the smallest power of two, 2^-40 at least, under which amax fits 448 = 0.875 * 2^9."""
    m, e = torch.frexp(amax)
    return torch.clamp(e - 9 + (m > 0.875).to(e.dtype), min=FLOOR)


def _power(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _standing_out(kv_heads, dim, seed):
    """Keys have channels that stand out."""
    return torch.exp(0.6 * _randn((kv_heads, dim), seed, 90))


def prepare(case, seed):
    rows, lens = _shape(case)
    batch, page, kvh, dim, heads = case["batch"], case["page"], case["kv_heads"], case["dim"], case["heads"]
    width = max(1, -(-max(lens) // page))
    total = batch * width + 3
    dev = "cuda"
    order = torch.randperm(total, generator=_gen(seed, 1), device=dev)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    table = order[:batch * width].reshape(batch, width)
    # what the cache holds before the call: every token of a sequence, or (update) those before the new ones
    held = lengths - torch.tensor(rows, dtype=torch.int32, device=dev) if case["kind"] == "update" else lengths
    count = torch.zeros(total, dtype=torch.int64, device=dev)
    count[table.reshape(-1)] = (held[:, None] - page * torch.arange(width, device=dev)).clamp(0, page).reshape(-1).long()
    there = (torch.arange(page, device=dev) < count[:, None])[:, None, :, None]
    codes, scales = [], torch.empty((total, kvh, 2), device=dev)
    for i in range(2):
        x = _randn((total, kvh, page, dim), seed, 2 + i)
        if i == 0:
            x *= _standing_out(kvh, dim, seed)[:, None]
        x = x * there
        s = _power(_exponent(x.abs().amax((2, 3))))
        scales[:, :, i] = s
        codes.append((x / s[:, :, None, None]).to(torch.float8_e4m3fn))
        del x
    state = {"case": case, "k_pages": codes[0], "v_pages": codes[1].transpose(2, 3).contiguous(), "scales": scales, "table": table.to(torch.int32).contiguous(),
             "lengths": lengths, "max_len": max(lens), "max_rows": max(rows)}
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    state["row_start"] = None if case["rows"] == 1 else torch.tensor(starts, dtype=torch.int32, device=dev)
    t = TYPE[case["type"]]
    n = starts[-1]
    if case["kind"] != "read":
        state["q"] = _randn((n, heads, dim), seed, 4).to(t)
    if case["kind"] == "update":
        state["k"] = (_randn((n, kvh, dim), seed, 5) * _standing_out(kvh, dim, seed)).to(t)
        state["v"] = _randn((n, kvh, dim), seed, 6).to(t)
        angle = torch.arange(width * page, device=dev, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(dim // 2, device=dev, dtype=torch.float64) / (dim // 2))
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    first = [(length - r) // page if case["kind"] == "update" else 0 for r, length in zip(rows, lens)]
    state["pages"] = torch.cat([state["table"][s, first[s]:-(-lens[s] // page)] for s in range(batch)])
    if own:
        from sharpmind_b200 import paged

        state["cache"] = paged.PagedKVCache(_context(), state["k_pages"], state["v_pages"], state["scales"])
    return state


_contexts = []


def _context():
    if not _contexts:
        from sharpmind_b200 import ops

        _contexts.append(ops.CudaContext(0))
    return _contexts[0]


# ------------------------------------------------------------------------------------------------ plain forms
def _places(s):
    """Sequence and position of every new row."""
    lengths, start = s["lengths"].long(), s["row_start"]
    batch = lengths.shape[0]
    rows = s["q"].shape[0]
    at = torch.arange(rows, device=lengths.device)
    if start is None:
        return at, lengths - 1
    start = start.long()
    n = start[1:] - start[:-1]
    seq = torch.repeat_interleave(torch.arange(batch, device=lengths.device), n, output_size=rows)
    return seq, lengths[seq] - n[seq] + at - start[seq]


def _rotate(x, cos, sin):
    """x [rows, heads, dim] by the rows' angles; dimension i goes with i + dim / 2."""
    x = x.float()
    a, b = x.chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _values(s, ids, t):
    scale = s["scales"][ids][:, :, :, None, None]
    k = (s["k_pages"][ids].float() * scale[:, :, 0]).transpose(1, 2)
    v = (s["v_pages"][ids].float() * scale[:, :, 1]).permute(0, 3, 1, 2)
    return k.to(t), v.to(t)


def _append(s, x, pages, which, page, off, first, ids, size):
    """The block scales grow to the new rows' magnitudes, the tokens that are there are rounded to the new scale, the rows enter."""
    amax = torch.zeros(s["scales"].shape[:2], device=x.device)
    amax.scatter_reduce_(0, page[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    old = s["scales"][:, :, which]
    need = _power(_exponent(amax))
    new = torch.where((first == 0)[:, None], need, torch.maximum(old, need))
    stay = torch.arange(size, device=x.device) < first[ids][:, None]
    held, was = pages[ids].float(), pages[ids].view(torch.uint8)
    again = (held * (old[ids] / new[ids])[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    stay = stay[:, None, :, None] if which == 0 else stay[:, None, None, :]
    raw = pages.view(torch.uint8)
    raw[ids] = torch.where(stay, again, was)
    code = (x / new[page][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    if which == 0:
        raw[page, :, off] = code
    else:
        raw[page, :, :, off] = code
    s["scales"][ids, :, which] = new[ids]


def _update(s):
    seq, pos = _places(s)
    size = s["k_pages"].shape[2]
    page, off = s["table"].long()[seq, pos // size], pos % size
    cos, sin = s["cos"][pos], s["sin"][pos]
    ids = s["pages"].long()
    first = torch.full((s["k_pages"].shape[0],), size, device=page.device).scatter_reduce_(0, page, off, "amin")
    _append(s, _rotate(s["k"], cos, sin), s["k_pages"], 0, page, off, first, ids, size)
    _append(s, s["v"].float(), s["v_pages"], 1, page, off, first, ids, size)
    k, v = _values(s, ids, torch.bfloat16)
    return {"q": _rotate(s["q"], cos, sin).to(s["q"].dtype), "k": k, "v": v}


def _attend(s):
    case, q = s["case"], s["q"]
    kvh, dim, group = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    batch, width = s["table"].shape
    seq, pos = _places(s)
    k, v = _values(s, s["table"].long().reshape(-1), torch.float32)
    k = k.reshape(batch, -1, kvh, dim).permute(0, 2, 3, 1)
    v = v.reshape(batch, -1, kvh, dim).transpose(1, 2)
    keys, most = k.shape[-1], s["max_rows"]
    row = torch.arange(q.shape[0], device=q.device) - (0 if s["row_start"] is None else s["row_start"].long()[seq])
    if s["row_start"] is None:
        row = torch.zeros_like(seq)
    padded = q.new_zeros((batch, most, kvh, group, dim), dtype=torch.float32)
    padded[seq, row] = q.float().reshape(-1, kvh, group, dim)
    place = torch.full((batch, most), -1, device=q.device)
    place[seq, row] = pos
    x = torch.matmul(padded.permute(0, 2, 3, 1, 4).reshape(batch, kvh, group * most, dim), k) * dim ** -0.5
    at = torch.arange(keys, device=q.device)
    sees = at <= place[:, :, None]
    if case["window"]:
        sees &= at > place[:, :, None] - case["window"]
    x = x.reshape(batch, kvh, group, most, keys).masked_fill_(~sees[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(batch, kvh, group * most, keys), v).reshape(batch, kvh, group, most, dim) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4)[seq, row].reshape(q.shape).to(q.dtype)


def run(state):
    s = state
    kind = s["case"]["kind"]
    if own:
        cache = s["cache"]
        if kind == "read":
            return cache.read(s["pages"], TYPE[s["case"]["type"]])
        if kind == "attend":
            return cache.attention(s["q"], s["table"], s["lengths"], s["case"]["dim"] ** -0.5, row_start=s["row_start"], max_rows=s["max_rows"], max_len=s["max_len"],
                                   window=s["case"]["window"])
        q = cache.Update(s["k"], s["v"], s["table"], s["lengths"], row_start=s["row_start"], cos=s["cos"], sin=s["sin"], q=s["q"])
        k, v = cache.read(s["pages"], torch.bfloat16)
        return {"q": q, "k": k, "v": v}
    if kind == "read":
        return _values(s, s["pages"].long(), TYPE[s["case"]["type"]])
    return _update(s) if kind == "update" else _attend(s)


# ------------------------------------------------------------------------------------------------ from the definition, in 64 bits
def _numbers(s, i):
    x = s["v_pages"].transpose(2, 3) if i else s["k_pages"]
    return x.double() * s["scales"][:, :, i, None, None].double()


def _fit(x):
    """Power of two of a block of magnitudes, and its e4m3 rounding: steps of 2^-3 of the value's own power of two, 2^-9 at least."""
    amax = float(x.abs().max())
    e = FLOOR
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def _round(x):
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), torch.clamp(e - 4, min=-9))
    return torch.round(x / step) * step


def _turned(x, places, dim):
    x = x.double()
    freq = 1e6 ** (-torch.arange(dim // 2, device=x.device, dtype=torch.float64) * 2 / dim)
    z = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), places.double()[:, None] * freq)[:, None]
    y = torch.complex(x[..., :dim // 2], x[..., dim // 2:]) * z
    return torch.cat([y.real, y.imag], -1)


def exact(case, seed):
    s = prepare(case, seed)
    rows, lens = _shape(case)
    page, dim, kvh, heads = case["page"], case["dim"], case["kv_heads"], case["heads"]
    if case["kind"] == "read":
        ids = s["pages"].long()
        return tuple(_numbers({**s, "k_pages": s["k_pages"][ids], "v_pages": s["v_pages"][ids], "scales": s["scales"][ids]}, i).transpose(1, 2).contiguous() for i in range(2))
    table = s["table"].tolist()
    if case["kind"] == "attend":
        out, done = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
        for b, (n, length) in enumerate(zip(rows, lens)):
            if length:
                ids = torch.tensor(table[b][:-(-length // page)], device="cuda")
                part = {**s, "k_pages": s["k_pages"][ids], "v_pages": s["v_pages"][ids], "scales": s["scales"][ids]}
                k, v = (_numbers(part, i).transpose(0, 1).reshape(kvh, -1, dim)[:, :length] for i in range(2))
                p = torch.arange(length - n, length, device="cuda")[:, None]
                j = torch.arange(length, device="cuda")[None]
                hidden = (j > p) | ((j <= p - case["window"]) if case["window"] else (j < 0))
                for h in range(heads):
                    x = s["q"][done:done + n, h].double() @ k[h * kvh // heads].T / math.sqrt(dim)
                    out[done:done + n, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[h * kvh // heads]
            done += n
        return out
    if sum(rows) * kvh > 60000:
        return None
    places = torch.cat([torch.arange(length - n, length, device="cuda") for n, length in zip(rows, lens)])
    new = [_turned(s["k"], places, dim), s["v"].double()]
    result, done = [[], []], 0
    for b, (n, length) in enumerate(zip(rows, lens)):
        for c in range((length - n) // page, -(-length // page)):
            lo, hi = max(length - n, c * page), min(length, (c + 1) * page)
            for i in range(2):
                codes = (s["v_pages"].transpose(2, 3) if i else s["k_pages"])[table[b][c]].double()
                block = torch.empty_like(codes)
                for h in range(kvh):
                    x = new[i][done + lo - (length - n):done + hi - (length - n), h]
                    e = _fit(x)
                    if lo > c * page:
                        was = math.frexp(float(s["scales"][table[b][c], h, i]))[1] - 1
                        e, keep = max(e, was), codes[h, :lo - c * page]
                        codes[h, :lo - c * page] = keep if e == was else _round(keep * 2.0 ** (was - e))
                    codes[h, lo - c * page:hi - c * page] = _round(x * 2.0 ** -e)
                    block[h] = codes[h] * 2.0 ** e
                result[i].append(block.transpose(0, 1))
        done += n
    return {"q": _turned(s["q"], places, dim), "k": torch.stack(result[0]), "v": torch.stack(result[1])}
