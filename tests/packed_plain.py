"""The cache held in 4 bits in plain torch and 64 bits, on the CPU: what the kernels over such pages are compared with."""

import math

import torch

NAN_WORD = 0x7FC0                   # the word of a row that holds no number


def quantize(x):
    """(codes [..., dim] int64, words [...] int16) of float64 rows: the smallest step of four significant bits that spans them."""
    x = x.double()
    bad = ~(x.abs() <= 2.0 ** 120).all(-1)
    y = torch.where(bad[..., None], torch.zeros_like(x), x)
    lo, hi = y.amin(-1).clamp(max=0), y.amax(-1).clamp(min=0)
    step = torch.full_like(lo, 2.0 ** -126)
    need = (hi - lo) / 15
    e = torch.floor(torch.log2(need.clamp(min=2.0 ** -126)))
    best = torch.full_like(lo, math.inf)
    for shift in (-1, 0, 1):
        for c in range(8, 16):
            candidate = torch.ldexp(torch.full_like(lo, c / 8), (e + shift).int())
            best = torch.where((15 * candidate >= hi - lo) & (candidate < best), candidate, best)
    step = torch.maximum(step, best)
    zero = -torch.round(lo / step)
    code = (torch.round(y / step[..., None]) + zero[..., None]).clamp(0, 15)
    word = step.float().bfloat16().view(torch.int16) | zero.to(torch.int16)
    return torch.where(bad[..., None], torch.zeros_like(code), code).long(), torch.where(bad, torch.tensor(NAN_WORD, dtype=torch.int16), word)


def pack(code):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8)


def unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2).double()


def step_zero(words):
    return (words & -16).view(torch.bfloat16).double(), (words & 15).double()


def values(packed, words):
    step, zero = step_zero(words)
    return (unpack(packed) - zero[..., None]) * step[..., None]


class Cache:
    """Requests of the given lengths in shuffled pages; every place that no request holds is not a number.  ``owned``: pages are
    each a request's own."""

    def __init__(self, lengths, g, dim, page, seed=0, spare=2):
        gen = torch.Generator().manual_seed(seed)
        per = [-(-n // page) for n in lengths]
        pages = sum(per) + spare
        self.lengths, self.g, self.dim, self.page = list(lengths), g, dim, page
        self.k, self.v = (torch.randint(0, 256, (pages, g, page, dim // 2), generator=gen, dtype=torch.uint8) for _ in range(2))
        self.words = torch.full((pages, g, page, 2), NAN_WORD, dtype=torch.int16)
        self.table = torch.full((len(per), max(per + [1]) + 1), -1, dtype=torch.int32)
        order, at = torch.randperm(pages, generator=gen).int(), 0
        for r, n in enumerate(per):
            self.table[r, :n] = order[at:at + n]
            at += n
        for r, n in enumerate(lengths):
            for j in range(n):
                mantissa = torch.randint(8, 16, (g, 2), generator=gen).float()
                step = mantissa * 2.0 ** torch.randint(-8, -4, (g, 2), generator=gen).float()
                zero = torch.randint(4, 12, (g, 2), generator=gen).to(torch.int16)
                self.words[int(self.table[r, j // page]), :, j % page] = step.bfloat16().view(torch.int16) | zero
        self.sums = torch.rand(pages, g, page, generator=gen)

    def rows(self, r, n, pool):
        """Rows 0 .. n - 1 of request r in a pool: [n, g, ...]."""
        j = torch.arange(n)
        return pool[self.table[r, j // self.page].long(), :, j % self.page]

    def to(self, device):
        from yalis_b200.ops.packed import PackedPages
        return PackedPages(self.k.to(device), self.v.to(device), self.words.to(device)), self.table.to(device)


def attention(cache, q, q_start, positions, heads, window=None, scale=None):
    """float64: out [N, heads * dim], the sum of weights per pool place, and per output the sum of P |v| and, per row and head, the
    largest score error that float32 products of the codes can make (31 times the step times the sum of |q|, a rounding an
    element).  The sum of P |v| of bfloat16 queries has 2^8 times this on top, which half a step of bfloat16 turns into what weights
    too small for float16 can lose: weights times steps are held as multiples of 2^-24 at least, at a scale at which the row's largest
    is 2^6 or more (where values' steps are 2^-80 or more); half of that, 2^-31 of the largest, times |code - zero| <= 15 for every key seen.  And what float32 sums
    lose when codes and zeros are multiplied out apart, sum P t c - sum P t z with each at most 15 sum P t: 300 roundings of 2^-24 of that."""
    n, dim, g = q.shape[0], cache.dim, cache.g
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out, size = torch.zeros(n, heads, dim).double(), torch.zeros(n, heads, dim).double()
    sums, slack, sum_slack = torch.zeros(cache.sums.shape).double(), torch.zeros(n, heads).double(), torch.zeros(cache.sums.shape).double()
    for r in range(len(q_start) - 1):
        for t in range(q_start[r], q_start[r + 1]):
            last = int(positions[t])
            first = 0 if window is None else max(0, last - window + 1)
            if last < first:
                continue
            j = torch.arange(first, last + 1)
            at, row = cache.table[r, j // cache.page].long(), j % cache.page
            k, v = values(cache.k[at, :, row], cache.words[at, :, row, 0]), values(cache.v[at, :, row], cache.words[at, :, row, 1])
            k_step = step_zero(cache.words[at, :, row, 0])[0]
            v_step = step_zero(cache.words[at, :, row, 1])[0].nan_to_num(0)
            for h in range(heads):
                kv = h // (heads // g)
                x = q[t].double()[h * dim:(h + 1) * dim]
                p = torch.softmax(k[:, kv] @ x * scale, 0)
                out[t, h], size[t, h] = p @ v[:, kv], p @ v[:, kv].abs()
                if q.dtype == torch.bfloat16:
                    weighted = (p * v_step[:, kv]).nan_to_num(0)
                    size[t, h] += 2.0 ** 8 * 15 * (len(j) * 2.0 ** -31 * weighted.max() + 300 * 2.0 ** -24 * weighted.sum())
                slack[t, h] = (dim + 16) * 2.0 ** -24 * 31 * k_step[:, kv].max() * x.abs().sum() * abs(scale)
                sums[at, kv, row] += p
                sum_slack[at, kv, row] += p * (2 * slack[t, h] + (len(j) + 32) * 2.0 ** -24)
    return out.flatten(1), sums, size.flatten(1), slack.repeat_interleave(dim, 1), sum_slack


def refusals(device):
    """(what is wrong, call) pairs; every call is refused on the host before anything is launched."""
    from yalis_b200.ops.packed import PackedPages, evict_tokens, packed_attention, packed_kv_read, packed_kv_write
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    c = Cache([40], 2, 64, 16)
    pages, table = c.to(device)
    f, pos, start = torch.zeros(3, 128, device=device), i32([0, 1, 2]), i32([0, 3])
    req, sums = i32([0, 0, 0]), c.sums.to(device)
    write = lambda k=f, v=f, p=pages, pos=pos, req=req, table=table: packed_kv_write(k, v, p, pos, req, table)
    attend = lambda q=torch.zeros(3, 256, device=device), p=pages, pos=pos, start=start, table=table, heads=4, **o: packed_attention(q, p, pos, start, table, 3, heads, **o)
    evict = lambda pools=pages.pools(), sums=sums, lengths=i32([40]), table=table, keep=10, recent=0: evict_tokens(pools, sums, lengths, table, keep, recent)
    bad = PackedPages(pages.k, pages.v, pages.words.float())
    odd = PackedPages(pages.k[..., :30].contiguous(), pages.v[..., :30].contiguous(), pages.words)
    return [
        ("half", lambda: write(k=f.half(), v=f.half())), ("types", lambda: write(v=f.bfloat16())), ("width", lambda: write(k=f[:, :64], v=f[:, :64])),
        ("rows", lambda: write(v=f[:2])), ("strides", lambda: write(k=f.t().contiguous().t())), ("positions", lambda: write(pos=pos.long())),
        ("count", lambda: write(req=req[:2])), ("table", lambda: write(table=table.long())), ("words", lambda: write(p=bad)), ("odd size", lambda: write(p=odd)),
        ("read half", lambda: packed_kv_read(pages, pos, req, table, dtype=torch.float16)),
        ("empty", lambda: PackedPages.empty(4, 2, 16, 20, device)), ("heads", lambda: attend(heads=3)), ("queries", lambda: attend(q=torch.zeros(3, 128, device=device))),
        ("attend half", lambda: attend(q=torch.zeros(3, 256, device=device).half())), ("window", lambda: attend(window=0)), ("scale", lambda: attend(scale=math.inf)),
        ("sums", lambda: attend(weight_sums=sums.double())), ("sums' shape", lambda: attend(weight_sums=sums[:, :1])), ("out", lambda: attend(out=f)),
        ("start", lambda: attend(start=start.long())), ("requests", lambda: attend(start=i32([0, 1, 2, 3]))), ("attend odd", lambda: attend(p=odd)),
        ("keep", lambda: evict(keep=0)), ("recent", lambda: evict(recent=11)), ("pools", lambda: evict(pools=pages.pools() + pages.pools())),
        ("pool's shape", lambda: evict(pools=(pages.k[:, :1],))), ("sums double", lambda: evict(sums=sums.double())), ("lengths", lambda: evict(lengths=i32([40]).long())),
        ("lengths' count", lambda: evict(lengths=i32([1, 2]))), ("odd bytes", lambda: evict(pools=(torch.zeros(c.k.shape[:3] + (3,), dtype=torch.uint8, device=device),))),
    ]
