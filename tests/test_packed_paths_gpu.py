"""Pages held in 4 bits where the kernels' ways part: values without numbers, keys without a page, places outside the table, shares of
keys, parts of rows and groups of requests, against plain torch in 64 bits."""

import pytest
import torch

from packed_plain import NAN_WORD, Cache, step_zero, values
from test_packed_cache_gpu import DEV, HALF, i32, step_of

pytestmark = pytest.mark.gpu
BAD_PAGE = 2


@pytest.fixture(params=["by the rule", "unpacked"])
def both_forms(request, monkeypatch):
    """Steps by whichever way their sizes choose, and every step of bfloat16 queries by unpacked rows; gives the list of the launches'
    names, to which a test that means to unpack adds "expects_unpacking"."""
    names = launches(monkeypatch, forced=request.param == "unpacked")
    yield names
    if request.param == "unpacked" and "expects_unpacking" in names:
        assert "yalis_packed_unpack" in names


def launches(monkeypatch, forced=False):
    from yalis_b200.ops import packed
    names, entry = [], packed._entry
    monkeypatch.setattr(packed, "_entry", lambda name, signature: names.append(name) or entry(name, signature))
    if forced:
        monkeypatch.setattr(packed, "UNPACK_ROWS", 0)
        monkeypatch.setattr(packed, "UNPACK_FEW", 0)
    return names


def plain_attention(cache, q, q_start, positions, heads, window=None):
    """As ``packed_plain.attention`` (its bounds are derived there), but keys without a page are left out of rows and sums."""
    n, dim, g = q.shape[0], cache.dim, cache.g
    per, scale, pages, columns = heads // g, dim ** -0.5, cache.k.shape[0], cache.table.shape[1]
    out, size, slack = torch.zeros(n, heads, dim).double(), torch.zeros(n, heads, dim).double(), torch.zeros(n, heads).double()
    sums, sum_slack = torch.zeros(cache.sums.shape).double(), torch.zeros(cache.sums.shape).double()
    for r in range(len(q_start) - 1):
        for t in range(q_start[r], q_start[r + 1]):
            last = min(int(positions[t]), columns * cache.page - 1)
            j = torch.arange(min(0 if window is None else max(0, int(positions[t]) - window + 1), last + 1), last + 1)
            j = j[(cache.table[r, j // cache.page] >= 0) & (cache.table[r, j // cache.page] < pages)]
            if not len(j):
                continue
            at, row = cache.table[r, j // cache.page].long(), j % cache.page
            k, v = values(cache.k[at, :, row], cache.words[at, :, row, 0]), values(cache.v[at, :, row], cache.words[at, :, row, 1])     # [keys, g, dim]
            x = q[t, :heads * dim].double().view(g, per, dim)
            p = torch.softmax(torch.einsum("jgd,ghd->ghj", k, x) * scale, -1)
            out[t] = torch.einsum("ghj,jgd->ghd", p, v).reshape(heads, dim)
            magnitude = torch.einsum("ghj,jgd->ghd", p, v.abs())
            if q.dtype == torch.bfloat16:
                weighted = (p * step_zero(cache.words[at, :, row, 1])[0].nan_to_num(0).t()[:, None]).nan_to_num(0)
                magnitude = magnitude + 2.0 ** 8 * 15 * (len(j) * 2.0 ** -31 * weighted.amax(-1) + 300 * 2.0 ** -24 * weighted.sum(-1))[..., None]
            size[t] = magnitude.reshape(heads, dim)
            off = (dim + 16) * 2.0 ** -24 * 31 * step_zero(cache.words[at, :, row, 0])[0].amax(0)[:, None] * x.abs().sum(-1) * scale
            slack[t] = off.reshape(heads)
            sums[at, :, row] += p.sum(1).t()
            sum_slack[at, :, row] += (p * (2 * off + (len(j) + 32) * 2.0 ** -24)[..., None]).sum(1).t()
    return out.flatten(1), sums, size.flatten(1), slack.repeat_interleave(dim, 1), sum_slack


def check(cache, q, pos, q_start, heads, window=None, sums=True, flag=0, **options):
    """One call against the plain form: a result is no number exactly where the plain one is none."""
    from yalis_b200.ops.packed import packed_attention
    pages, table = cache.to(DEV)
    total, word = cache.sums.to(DEV) if sums else None, torch.zeros(1, dtype=torch.int32, device=DEV)
    longest = max([b - a for a, b in zip(q_start[:-1], q_start[1:])] + [0])
    options = {"max_q_len": longest, **options}
    got = packed_attention(q.to(DEV), pages, pos.to(DEV), i32(q_start), table, num_heads=heads, window=window, weight_sums=total, error_flag=word, **options)
    assert int(word) == flag
    ref, a, size, slack, sum_slack = plain_attention(cache, q, q_start, pos, heads, window)
    y, half = got.cpu().double(), HALF[q.dtype]
    none = ref.isnan()
    assert torch.equal(y.isnan(), none), f"{int((y.isnan() != none).sum())} of {y.numel()}"
    bound = half * ref.abs() + (half + 2 * slack + 300 * 2.0 ** -24) * size + 1e-30
    off = ((y - ref).abs() / bound)[~none]
    assert bool((off <= 1).all()), float(off.max())
    if sums:
        ref_sums = cache.sums.double() + a
        err, room = (total.cpu().double() - ref_sums).abs(), sum_slack + 2.0 ** -23 * ref_sums
        assert bool((err <= room)[~ref_sums.isnan()].all()), float((err / room).nan_to_num(0).max())
        assert torch.equal(total.cpu().isnan(), ref_sums.isnan())
    return got


# ---- values without numbers -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,g,dim,page,window", [(4, 2, 64, 16, None), (4, 2, 64, 64, 40), (8, 1, 128, 16, 70), (4, 2, 128, 64, None), (4, 2, 24, 16, 40)])
def test_a_value_without_numbers_is_seen_only_by_those_that_see_it(both_forms, dtype, heads, g, dim, page, window):
    """One value row in the middle of a portion, one that some windows have passed, one before a window's first key: rows that do not
    see it keep their numbers, however many there are, and the weights' sums go by the keys alone."""
    c = Cache([100, 300, 200, 90], g, dim, page, seed=dim + page)
    for r, j in ((0, 50), (1, 160), (2, 3)):
        c.words[int(c.table[r, j // page]), g - 1, j % page, 1] = NAN_WORD
    q, pos, q_start = step_of(c, [100, 170, 130, 1], dtype=dtype, heads=heads)
    got = check(c, q, pos, q_start, heads, window)
    assert bool(got.isnan().any()) and bool((~got.isnan()).any())
    both_forms += ["expects_unpacking"] * (dtype == torch.bfloat16 and dim != 24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,n", [(64, 1), (128, 1), (128, 7), (24, 1)])
def test_sums_where_a_value_without_numbers_is_seen(dtype, dim, n):
    """Its weight and everybody else's are softmax weights as ever, though the row's result is none: here it gets nearly all of a
    row's weight, or none, and the others what is left."""
    c = Cache([300, 90], 2, dim, 16, seed=dim)
    for r, j in ((0, 5), (0, 200), (1, 70)):
        at = int(c.table[r, j // 16])
        c.words[at, 0, j % 16, 1] = NAN_WORD
        c.words[at, 0, j % 16, 0] = torch.tensor(2.0 ** -2).bfloat16().view(torch.int16) | 7
    q, pos, q_start = step_of(c, [n, n], dtype=dtype, heads=4)
    check(c, q, pos, q_start, 4)

# ---- keys without a page --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,g,dim", [(4, 2, 64), (8, 1, 128), (4, 2, 24)])
@pytest.mark.parametrize("page,window", [(16, None), (64, None), (16, 90), (5, None)])
@pytest.mark.parametrize("brought", [[1, 1, 1, 1], [5, 1, 3, 2], [100, 40, 150, 1]])
def test_keys_without_a_page_are_left_out(both_forms, dtype, heads, g, dim, page, window, brought):
    """At the start, in the middle (of keys that every row sees), at the end, and all of a request's: neither rows nor normaliser
    nor sums know them, and the error word tells."""
    c = Cache([333, 200, 150, 70], g, dim, page, seed=dim + page)
    at = lambda r, *places: [c.table[r, j // page].fill_(w) for j, w in places]
    at(0, (100, -1), (210, c.k.shape[0]), (332, -5))
    at(1, (0, -1), (10, c.k.shape[0] + 7))
    c.table[2] = -1
    q, pos, q_start = step_of(c, brought, dtype=dtype, heads=heads)
    got = check(c, q, pos, q_start, heads, window, flag=BAD_PAGE)
    assert bool((got[q_start[2]:q_start[3]] == 0).all())
    both_forms += ["expects_unpacking"] * (dtype == torch.bfloat16 and dim != 24)
    check(c, q, pos, q_start, heads, window, sums=False, flag=BAD_PAGE)


# ---- places outside the table ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,n", [(64, 1), (128, 1), (24, 1), (64, 7), (24, 5), (64, 90), (128, 70)])
@pytest.mark.parametrize("window", [None, 50])
def test_places_outside_the_table(both_forms, dtype, dim, n, window):
    """Rows at places that the table has no columns for, at the last place that there is and far before the first: what the table has
    of their places is seen, the error word tells, and every walk ends with the table."""
    c = Cache([112, 100, 60, 64, 112, 90], 2, dim, 16, seed=n)       # places 112 .. 127 have no page, 128 and on no column
    ends = [140, 100, -150, 3, 2 ** 31, 90]
    pos = torch.cat([torch.arange(end - n, end) for end in ends]).int()
    q, q_start = torch.randn(6 * n, 4 * dim, generator=torch.Generator().manual_seed(dim)).to(dtype), [n * i for i in range(7)]
    got = check(c, q, pos, q_start, 4, window, flag=BAD_PAGE)
    assert bool((got[2 * n:3 * n] == 0).all())
    check(c, q, pos, q_start, 4, window, sums=False, flag=BAD_PAGE)
    both_forms += ["expects_unpacking"] * (dtype == torch.bfloat16 and dim != 24)
    keep = torch.cat([torch.arange(n, 4 * n), torch.arange(5 * n, 6 * n)])       # without them no word is raised
    c.table[[0, 4]] = c.table[[4, 0]]
    check(c, q[keep], pos[keep], [0, 0, n, 2 * n, 3 * n, 3 * n, 4 * n], 4, window)


# ---- eviction -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("pools", [0, 1])
def test_a_cut_without_rows_to_move(pools):
    """No pools, or one whose rows have no bytes: the sums move all the same."""
    from yalis_b200.ops.packed import evict_tokens
    c = Cache([40, 9, 2000], 2, 8, 16)
    total = c.sums.to(DEV)
    kept = evict_tokens([torch.empty(c.k.shape[:3] + (0,), device=DEV)] * pools, total, i32(c.lengths), c.table.to(DEV), 12, 3)
    for r, n in ((0, 40), (2, 2000)):
        for h in range(2):
            score = c.rows(r, n, c.sums)[:, h].clone()
            score[n - 3:] = 2.0
            j = torch.sort(torch.topk(score, 12).indices).values
            assert torch.equal(kept[r, h].cpu().long(), j)
            assert torch.equal(c.rows(r, 12, total.cpu())[:, h], c.rows(r, n, c.sums)[j, h])
    assert torch.equal(c.rows(1, 9, total.cpu()), c.rows(1, 9, c.sums)) and kept[1, 0].tolist() == list(range(9)) + [-1] * 3


# ---- bounds ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("brought", [[1, 1], [3, 2], [90, 90], [90, 1]])
def test_generous_bounds(both_forms, brought):
    """Bounds far above what a step brings and sees, past 32 bits too, and bounds that fit; none of keys where nothing is seen."""
    c = Cache([200, 90], 2, 64, 16, seed=4)
    q, pos, q_start = step_of(c, brought, heads=8)
    for max_q_len in (max(brought), 5000, 1 << 31, 1 << 40):
        for max_kv_len in (None, 200, 1 << 31, 1 << 50):
            check(c, q, pos, q_start, 8, max_q_len=max_q_len, max_kv_len=max_kv_len)
    both_forms += ["expects_unpacking"]
    assert bool((check(c, q, torch.full_like(pos, -1), q_start, 8, max_kv_len=0) == 0).all())
