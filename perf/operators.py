"""The operators of a cache held in 4 bits, as cases that can be timed and compared.

Keys and values lie in pages, every row of a token and KV head as ``head_dim`` codes of 4 bits with a step and a zero of its
own: value = (code - zero) * step.  With lo = min(x, 0) and hi = max(x, 0) over the row, step is the smallest number of four
significant bits (2^-126 at least) with 15 step >= hi - lo, zero = -round(lo / step), code = round(x / step) + zero within
0 .. 15; roundings are to the nearest, ties to even.  So every value is a bfloat16 number.  Byte b of a row holds the code of
element 2b in its low half and that of 2b + 1 in its high half; a 16-bit word holds the bits of the step as bfloat16 with the
zero in the lowest four.  The cases:

``rows``    keys and values of a step's tokens are written into their pages and read back;
``attend``  the step's queries over the pages of their requests: single tokens, portions of prompts and both together, with
            ``sums`` the weights that every cached token receives are added to a running sum per token and KV head;
``evict``   of every request and KV head the last ``recent`` tokens and those with the largest sums stay, ``keep`` in all, and
            move to the front of its pages in their order (pools of bfloat16, or held in 4 bits).

``exact`` states each in 64 bits, request by request.
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda:0"
LOWEST = -1e30


def _attend(requests, tokens, cached, heads, kv_heads, dim, ragged=False, decoding=0, page=64, dtype="bfloat16", window=0, sums=False, name=None):
    c = {"kind": "attend", "requests": requests, "tokens": tokens, "cached": cached, "ragged": ragged, "decoding": decoding, "heads": heads,
         "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "window": window, "sums": sums}
    return c if name is None else {**c, "name": name}


def _rows(requests, tokens, cached, kv_heads, dim, page=64, dtype="bfloat16", name=None):
    c = {"kind": "rows", "requests": requests, "tokens": tokens, "cached": cached, "ragged": requests > 1 and tokens > 1, "decoding": 0,
         "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}
    return c if name is None else {**c, "name": name}


def _evict(requests, length, keep, recent, kv_heads, dim, packed, page=64, name=None):
    c = {"kind": "evict", "requests": requests, "tokens": 1, "cached": length - 1, "ragged": requests > 1, "decoding": 0, "keep": keep,
         "recent": recent, "kv_heads": kv_heads, "dim": dim, "page": page, "packed": packed, "dtype": "bfloat16"}
    return c if name is None else {**c, "name": name}


def listed():
    return [
        # a busy server's decode step stores one token of each of 64 requests
        _rows(64, 1, 1040, 8, 128, name="rows of a decode step"),
        # prompts of unequal length enter the cache
        _rows(3, 4001, 0, 8, 128, name="rows of prompts"),
        # the latency of a lone request with a short context (Llama-3-8B's heads)
        _attend(1, 1, 128, 32, 8, 128, name="decode, one short request"),
        # the benchmark's decode step: 64 requests around 1,040 tokens
        _attend(64, 1, 1040, 32, 8, 128, ragged=True, name="decode, 64 requests"),
        # few requests with long contexts, what a smaller cache is for (Llama-3.2-3B's heads)
        _attend(8, 1, 32000, 24, 8, 128, ragged=True, name="decode, long contexts"),
        # the true 32-bit path (Llama-3.2-1B's heads)
        _attend(4, 1, 1900, 32, 8, 64, page=16, dtype="float32", name="decode, float32"),
        # time to the first token: a whole prompt
        _attend(1, 2048, 0, 32, 8, 128, name="prompt of 2,048 tokens"),
        # a portion of a long prompt beside decoding requests
        _attend(1, 512, 6001, 24, 8, 128, decoding=7, name="portion beside decoding requests"),
        # decode steps that keep count of which tokens are attended to
        _attend(16, 1, 4000, 32, 8, 128, ragged=True, sums=True, name="decode with sums"),
        # prompts that start the count
        _attend(2, 1500, 0, 32, 8, 64, ragged=True, sums=True, name="prompts with sums"),
        # a cache in bfloat16 cut to half
        _evict(32, 4160, 2048, 256, 8, 128, False, name="eviction, 32 requests"),
        # one request's packed cache cut by a little
        _evict(1, 700, 512, 64, 8, 64, True, name="eviction, one request"),
    ]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    page = rng.choice([16, 32, 64, 64])
    kind = rng.choice(["rows", "attend", "attend", "attend", "evict"])
    if kind == "rows":
        n, t = rng.choice([(spread(1, 128), 1), (rng.choice([1, 2, 3, 4]), spread(2, 2900))])
        return _rows(n, t, spread(1, 2000), rng.choice([1, 2, 8]), rng.choice([64, 128]), page, rng.choice(["bfloat16", "bfloat16", "float32"]))
    if kind == "evict":
        length = spread(130, 8000)
        keep = max(2, int(length * rng.uniform(0.2, 0.9)))
        n = spread(1, max(1.01, min(48, 130000 / length)))
        return _evict(n, length, keep, rng.choice([0, 1, keep // 8, keep // 2]), rng.choice([1, 2, 8]), rng.choice([64, 128]), rng.random() < 0.5, page)
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (24, 8, 128), (32, 8, 64), (16, 8, 128), (2, 1, 128), (8, 1, 64)])
    shape = rng.choice(["decode", "decode", "decode", "portion"])
    dtype = "float32" if rng.random() < 0.15 else "bfloat16"
    window = rng.choice([0, 0, 0, spread(100, 2000)])
    if shape == "decode":
        n = spread(1, 96)
        cached = spread(1, max(2, min(32000, (64 if dtype == "bfloat16" else 8) * 1500 // n)))
        return _attend(n, 1, cached, heads, kv_heads, dim, n > 1 and rng.random() < 0.7, 0, page, dtype, window, rng.random() < 0.3)
    n = rng.choice([1, 1, 2, 3])
    tokens = spread(2, (2048 if dtype == "bfloat16" else 160) // n)
    return _attend(n, tokens, rng.choice([0, spread(1, 4000)]), heads, kv_heads, dim, n > 1, rng.choice([0, 0, 5]) if n == 1 and tokens <= 512 else 0, page, dtype,
                   window, rng.random() < 0.3)


# ---- the step -------------------------------------------------------------------------------------------------------

def _lens(case):
    """(tokens brought, tokens held before) of every request."""
    r, t, c = case["requests"], case["tokens"], case["cached"]
    if not case["ragged"]:
        brought, held = [t] * r, [c] * r
    else:
        brought = [max(1, t - i * (t // (2 * r)) - i) if t > 1 else 1 for i in range(r)]
        held = [max(0, c - i * (c // (2 * r))) for i in range(r)]
    more = case["decoding"]
    return brought + [1] * more, held + [max(1, c // (2 + i)) for i in range(more)]


def _seen(case):
    """Cached tokens that each row's query sees, summed over the rows."""
    w = case.get("window", 0)
    total = 0
    for t, c in zip(*_lens(case)):
        if not w:
            total += t * c + t * (t + 1) // 2
        else:
            whole = max(0, min(t, w - c))                     # rows whose window reaches the first token
            total += whole * c + whole * (whole + 1) // 2 + (t - whole) * w
    return total


def _touched(case):
    """Cached tokens that any row's query sees."""
    w = case.get("window", 0)
    return sum(min(t + c, w + t - 1) if w else t + c for t, c in zip(*_lens(case)))


def work(case):
    brought, held = _lens(case)
    n, g, d = sum(brought), case["kv_heads"], case["dim"]
    e = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "rows":
        return {"bytes": 2 * n * g * (2 * d * e + 2 * (d // 2 + 2)), "flops": 2 * n * g * d * 6}
    if case["kind"] == "attend":
        row, touched = d + 4, _touched(case) * g                # a token and KV head: codes of key and value, two words
        return {"bytes": touched * (row + (8 if case["sums"] else 0)) + 2 * n * case["heads"] * d * e, "flops": 4 * _seen(case) * case["heads"] * d}
    row = d + 4 if case["packed"] else 4 * d
    moved = sum(min(case["keep"], c + t) for t, c in zip(brought, held) if c + t > case["keep"])
    back = sum(min(case["keep"], c + t) for t, c in zip(brought, held)) * g * (row + 4 * d) if case["packed"] else 0
    return {"bytes": sum(c + t for t, c in zip(brought, held)) * g * 4 + moved * g * (2 * row + 4 + 4) + back,
            "flops": 2 * sum(c + t for t, c in zip(brought, held)) * g}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _quantize(x):
    """(codes uint8, words int16) of rows ``x`` [..., dim], in 64 bits (values may stand next to a border)."""
    x = x.double()
    low, high = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    mantissa, exponent = torch.frexp((high - low) / 15)
    step = torch.ldexp((mantissa * 16).ceil(), exponent - 4).clamp(min=2.0 ** -126)
    zero = -(low / step).round()
    code = ((x / step).round() + zero).clamp(0, 15).to(torch.uint8)
    return code, step[..., 0].bfloat16().view(torch.int16) | zero[..., 0].to(torch.int16)


def _bytes_of(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _values(packed, words):
    """float32 values of packed rows [..., dim / 2] with their words [...]."""
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float()
    return (code - (words & 15)[..., None].float()) * (words & -16).view(torch.bfloat16)[..., None].float()


def _dtype(case):
    return torch.float32 if case["dtype"] == "float32" else torch.bfloat16


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
    brought, before = _lens(case)
    page, g, d = case["page"], case["kv_heads"], case["dim"]
    held = [b + t for b, t in zip(before, brought)]
    per = [-(-h // page) for h in held]
    pages, r = sum(per) + 2, len(held)
    perm = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    table, at = torch.full((r, max(per)), -1, dtype=torch.int32, device=DEV), 0
    for i, p in enumerate(per):
        table[i, :p] = perm[at:at + p]
        at += p
    starts = [0]
    for t in brought:
        starts.append(starts[-1] + t)
    pos = torch.cat([torch.arange(b, b + t, dtype=torch.int32, device=DEV) for b, t in zip(before, brought)])
    req = torch.repeat_interleave(torch.arange(r, dtype=torch.int32, device=DEV), torch.tensor(brought, device=DEV))
    s = {"case": {k: v for k, v in case.items() if k != "name"}, "table": table, "q_start": i32(starts), "positions": pos, "req": req,
         "lengths": i32(held), "longest": max(brought), "longest_context": max(held)}
    # keys have a few strong channels and an offset per channel, as a model's do; values have neither
    weight, offset = (normal(g, 1, d) * 0.5).exp(), normal(g, 1, d) * 0.3
    if case["kind"] == "evict" and not case["packed"]:
        s["k"], s["v"] = ((normal(pages, g, page, d) * weight + offset).bfloat16(), normal(pages, g, page, d).bfloat16())
    else:
        s["k"], s["v"] = (torch.empty((pages, g, page, d // 2), dtype=torch.uint8, device=DEV) for _ in range(2))
        s["words"] = torch.empty((pages, g, page, 2), dtype=torch.int16, device=DEV)
        for a in range(0, pages, 1024):
            b = min(pages, a + 1024)
            for to, x, j in ((s["k"], normal(b - a, g, page, d) * weight + offset, 0), (s["v"], normal(b - a, g, page, d), 1)):
                code, s["words"][a:b, ..., j] = _quantize(x)
                to[a:b] = _bytes_of(code)
    n = sum(brought)
    if case["kind"] == "rows":
        s["new_k"] = (normal(n, g, d) * weight[:, 0] + offset[:, 0]).to(_dtype(case)).flatten(1)
        s["new_v"] = normal(n, g * d).to(_dtype(case))
    if case["kind"] == "attend":
        s["q"] = normal(n, case["heads"] * d).to(_dtype(case))
    if case["kind"] == "evict" or case.get("sums"):
        # what attention leaves behind: a few tokens with most of the weight, many with little, some that were never seen
        u = torch.rand((pages, g, page), generator=gen, device=DEV)
        s["sums"] = torch.where(u < 0.1, torch.zeros_like(u), normal(pages, g, page).mul(2).exp() * 0.01)
        if case["kind"] == "attend" and case["cached"] == 0:
            s["sums"].zero_()                                                        # prompts start the count
    if case["kind"] == "evict" and case["packed"]:
        kept = [min(case["keep"], h) for h in held]
        s["kept_positions"] = torch.cat([torch.arange(k, dtype=torch.int32, device=DEV) for k in kept])
        s["kept_req"] = torch.repeat_interleave(torch.arange(r, dtype=torch.int32, device=DEV), torch.tensor(kept, device=DEV))
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(s):
    return {"rows": _run_rows, "attend": _run_attend, "evict": _run_evict}[s["case"]["kind"]](s)


def _pages(s):
    from yalis_b200.ops.packed import PackedPages
    return PackedPages(s["k"], s["v"], s["words"])


def _place(s, positions, req):
    """(page, row in the page) of cached tokens."""
    page = s["case"]["page"]
    return s["table"][req.long(), (positions // page).long()].long(), (positions % page).long()


def _read(s, positions, req, dtype):
    at, row = _place(s, positions, req)
    words = s["words"][at, :, row]
    return tuple(_values(s[n][at, :, row], words[..., j]).to(dtype).flatten(1) for n, j in (("k", 0), ("v", 1)))


def _run_rows(s):
    case = s["case"]
    if own:
        from yalis_b200.ops.packed import packed_kv_read, packed_kv_write
        pages = _pages(s)
        packed_kv_write(s["new_k"], s["new_v"], pages, s["positions"], s["req"], s["table"])
        return packed_kv_read(pages, s["positions"], s["req"], s["table"], dtype=_dtype(case))
    at, row = _place(s, s["positions"], s["req"])
    n = at.shape[0]
    k_code, k_word = _quantize(s["new_k"].view(n, case["kv_heads"], case["dim"]))
    v_code, v_word = _quantize(s["new_v"].view(n, case["kv_heads"], case["dim"]))
    s["k"][at, :, row], s["v"][at, :, row] = _bytes_of(k_code), _bytes_of(v_code)
    s["words"][at, :, row] = torch.stack([k_word, v_word], -1)
    return _read(s, s["positions"], s["req"], _dtype(case))


def _run_attend(s):
    case = s["case"]
    if own:
        from yalis_b200.ops.packed import packed_attention
        out = packed_attention(s["q"], _pages(s), s["positions"], s["q_start"], s["table"], s["longest"], case["heads"],
                               window=case["window"] or None, max_kv_len=s["longest_context"], weight_sums=s.get("sums"))
        return (out, s["sums"]) if case["sums"] else out
    g, d, heads, page = case["kv_heads"], case["dim"], case["heads"], case["page"]
    table, start, dev = s["table"], s["q_start"].long(), s["q"].device
    r, width, per, most = table.shape[0], table.shape[1], heads // g, s["longest"]
    at = table.clamp(min=0).long()
    flat = lambda x: x[at].transpose(1, 2).flatten(2, 3)                             # [R, kv_heads, width * page, ...]
    words = flat(s["words"])
    k, v = _values(flat(s["k"]), words[..., 0]), _values(flat(s["v"]), words[..., 1])
    brought = start[1:] - start[:-1]
    i = torch.arange(most, device=dev)
    real = i[None] < brought[:, None]                                                # rows of the padded batch that are tokens
    token = (start[:-1, None] + i[None]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float().view(-1, g, per, d)[token].permute(0, 2, 1, 3, 4).flatten(2, 3)          # [R, kv_heads, Q * per, d]
    pos = s["positions"].long()[token]
    j = torch.arange(width * page, device=dev)
    sees = (j <= pos[..., None]) & real[..., None]
    if case["window"]:
        sees &= j > pos[..., None] - case["window"]
    sees = sees[:, None].repeat_interleave(per, 2)                                   # [R, 1, Q * per, keys]
    score = ((q @ k.transpose(2, 3)) * (1.0 / math.sqrt(d))).masked_fill(~sees, LOWEST)
    weight = (score - score.amax(-1, keepdim=True)).exp() * sees
    weight = weight / weight.sum(-1, keepdim=True).clamp(min=1e-38)
    y = (weight @ v).view(r, g, most, per, d).permute(0, 2, 1, 3, 4).flatten(2)
    out = y[real].to(s["q"].dtype)
    if not case["sums"]:
        return out
    total = weight.sum(2).view(r, g, width, page).transpose(1, 2)                    # [R, width, kv_heads, page]
    s["sums"].index_add_(0, at[table >= 0], total[table >= 0])
    return out, s["sums"]


def _run_evict(s):
    case = s["case"]
    keep, recent, packed = case["keep"], case["recent"], case["packed"]
    if own:
        from yalis_b200.ops.packed import evict_tokens, packed_kv_read
        pages = _pages(s) if packed else None
        kept = evict_tokens(pages.pools() if packed else (s["k"], s["v"]), s["sums"], s["lengths"], s["table"], keep, recent=recent)
        if packed:
            return (kept, s["sums"]) + tuple(packed_kv_read(pages, s["kept_positions"], s["kept_req"], s["table"], dtype=torch.bfloat16))
        return kept, s["sums"], s["k"], s["v"]
    table, length, page, g = s["table"], s["lengths"].long(), case["page"], case["kv_heads"]
    r, width = table.shape
    at = table.clamp(min=0).long()
    flat = lambda x: x[at].transpose(1, 2).flatten(2, 3)
    j = torch.arange(width * page, device=table.device)
    inside = j[None] < length[:, None]
    newest = inside & (j[None] >= length[:, None] - recent)
    total = flat(s["sums"])                                                          # [R, kv_heads, tokens]
    rank = torch.where(newest[:, None], math.inf, torch.where(inside[:, None], total, -math.inf))
    chosen = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values       # [R, kv_heads, keep]
    short = length <= keep
    first = torch.arange(chosen.shape[-1], device=table.device)
    chosen = torch.where(short[:, None, None], first, chosen)
    there = (first[None] < length[:, None])[:, None].expand_as(chosen)
    pools = (s["k"], s["v"], s["words"]) if packed else (s["k"], s["v"])
    of_request = torch.arange(r, device=table.device)[:, None, None].expand_as(chosen)
    of_head = torch.arange(g, device=table.device)[None, :, None].expand_as(chosen)
    new = first.expand_as(chosen)
    place = lambda index: (at[of_request[there], index[there] // page], of_head[there], index[there] % page)
    source, target = place(chosen), place(new)
    rows = [x[source] for x in pools + (s["sums"],)]
    for x, row in zip(pools + (s["sums"],), rows):
        x[target] = row
    kept = torch.where(there, chosen, -1).to(torch.int32)
    if packed:
        return (kept, s["sums"]) + _read(s, s["kept_positions"], s["kept_req"], torch.bfloat16)
    return kept, s["sums"], s["k"], s["v"]


# ---- the same in 64 bits, request by request ----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    brought, before = _lens(case)
    page, g, d = case["page"], case["kv_heads"], case["dim"]
    if case["kind"] == "rows":
        out = []
        for x in (s["new_k"], s["new_v"]):
            x = x.double().view(-1, g, d)
            lo, hi = x.min(-1).values.clamp(max=0.0), x.max(-1).values.clamp(min=0.0)
            near, step = torch.floor(torch.log2((hi - lo) / 15.0)), torch.full_like(lo, math.inf)
            for e in (1, 0, -1):
                for c in range(15, 7, -1):                 # from the largest down: the last that is wide enough stays
                    candidate = torch.exp2(near + e) * (c / 8.0)
                    step = torch.where(15.0 * candidate >= hi - lo, torch.minimum(step, candidate), step)
            first = torch.round(lo / step)                 # the row's codes stand for the multiples first .. first + 15
            multiple = torch.round(x / step[..., None])
            multiple = torch.minimum(torch.maximum(multiple, first[..., None]), first[..., None] + 15.0)
            out.append((multiple * step[..., None]).flatten(1))
        return out
    if case["kind"] == "evict":
        return None                                        # rows are moved, not computed
    heads, per, w, at = case["heads"], case["heads"] // g, case["window"], 0
    out = torch.empty((sum(brought), heads * d), dtype=torch.float64, device=DEV)
    sums = s["sums"].double() if case["sums"] else None
    for i, (t, b) in enumerate(zip(brought, before)):
        n = b + t
        ids = s["table"][i, :-(-n // page)].long()
        rows = torch.arange(n, device=DEV)
        seen = rows[None] <= b + torch.arange(t, device=DEV)[:, None]
        if w:
            seen &= rows[None] + w > b + torch.arange(t, device=DEV)[:, None]
        for h in range(g):
            p = s["words"][ids, h].flatten(0, 1)[:n]
            step, zero = p.bitwise_and(-16).view(torch.bfloat16).double(), p.remainder(16).double()
            nibbles = [s[x][ids, h].flatten(0, 1)[:n] for x in ("k", "v")]
            k, v = (torch.stack((x.remainder(16), x.div(16, rounding_mode="floor")), 2).flatten(1).double() for x in nibbles)
            k, v = ((x - zero[:, j:j + 1]) * step[:, j:j + 1] for j, x in enumerate((k, v)))
            total = torch.zeros(n, dtype=torch.float64, device=DEV)
            for e in range(h * per, (h + 1) * per):
                q = s["q"][at:at + t, e * d:(e + 1) * d].double()
                weight = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill(~seen, -math.inf), -1)
                out[at:at + t, e * d:(e + 1) * d] = weight @ v
                total += weight.sum(0)
            if sums is not None:
                place = sums[ids, h].flatten()
                place[:n] += total
                sums[ids, h] = place.view(-1, page)
        at += t
    return (out, sums) if case["sums"] else out
