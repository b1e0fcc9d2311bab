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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,g,dim,page", [(4, 2, 64, 16), (8, 1, 128, 5), (4, 2, 24, 16)])
@pytest.mark.parametrize("brought", [[1, 1, 1], [9, 3, 1], [100, 130, 1]])
def test_pages_given_back_behind_windows(both_forms, dtype, heads, g, dim, page, brought):
    """Pages that lie behind the first row's window may be gone, or another request's: nobody is told."""
    c, window = Cache([333, 200, 170], g, dim, page, seed=dim), 37
    for r, n in enumerate(brought):
        gone = (c.lengths[r] - n - window + 1) // page
        c.table[r, :gone] = torch.arange(gone).int() % 3 - 1
    q, pos, q_start = step_of(c, brought, dtype=dtype, heads=heads)
    check(c, q, pos, q_start, heads, window)
    both_forms += ["expects_unpacking"] * (dtype == torch.bfloat16 and dim != 24)


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


@pytest.mark.parametrize("n,keep,recent", [(24577, 11000, 40), (30000, 25000, 0), (26000, 30, 30)])
def test_a_cut_of_more_tokens_than_shared_memory_has_keys_for(n, keep, recent):
    from yalis_b200.ops.packed import evict_tokens
    c = Cache([n, 0], 1, 8, 64)                                      # (its words are filled row by row: one head)
    c.sums[torch.rand(c.sums.shape, generator=torch.Generator().manual_seed(1)) < 0.3] = 0.25       # ties
    pages, table = c.to(DEV)
    total = c.sums.to(DEV)
    kept = evict_tokens(pages.pools(), total, i32(c.lengths), table, keep, recent)
    score = c.rows(0, n, c.sums)[:, 0].clone()
    score[n - recent:] = 2.0
    j = torch.sort(torch.sort(score, descending=True, stable=True).indices[:keep]).values
    assert torch.equal(kept[0, 0].cpu().long(), j)
    for before, after in zip((c.k, c.v, c.words, c.sums), pages.pools() + (total,)):
        assert torch.equal(c.rows(0, keep, after.cpu()), c.rows(0, n, before)[j])


def test_tokens_behind_a_cut_start_from_zero_where_the_caller_says_so():
    """A place that is written again keeps the sum that stood there: set to zero first, its new token is ranked by its own weights."""
    from yalis_b200.ops.packed import PackedPages, evict_tokens, packed_attention, packed_kv_write
    heads, g, dim, page, keep = 4, 2, 64, 16, 20
    gen = torch.Generator().manual_seed(5)
    pages, table = PackedPages.empty(4, g, page, dim, DEV), i32([[2, 0, 3, 1]])
    c, sums = Cache([60], g, dim, page, spare=0), torch.zeros(4, g, page, device=DEV)
    c.table = table.cpu()
    counted = torch.zeros(4, g, page).double()

    def step(n, at):
        nonlocal counted
        qkv = torch.randn(n, (heads + 2 * g) * dim, generator=gen).bfloat16().to(DEV)
        places = torch.arange(at, at + n, dtype=torch.int32, device=DEV)
        sums[table[0, places // page].long(), :, (places % page).long()] = 0.0
        packed_kv_write(qkv[:, heads * dim:(heads + g) * dim], qkv[:, (heads + g) * dim:], pages, places, torch.zeros_like(places), table)
        packed_attention(qkv, pages, places, i32([0, n]), table, n, heads, weight_sums=sums)
        c.k, c.v, c.words = (t.cpu() for t in pages.pools())
        for j in range(at, at + n):
            counted[int(c.table[0, j // page]), :, j % page] = 0
        counted += plain_attention(c, qkv.cpu(), [0, n], places.cpu(), heads)[1]

    step(60, 0)
    evict_tokens(pages.pools(), sums, i32([60]), table, keep, 4)
    counted = sums.cpu().double()
    step(7, keep)
    torch.testing.assert_close(c.rows(0, keep + 7, sums.cpu()).double(), c.rows(0, keep + 7, counted), rtol=1e-4, atol=1e-6)
    assert bool((c.rows(0, keep + 7, sums.cpu())[keep:].sum(0) <= 7 * heads // g).all())



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


# ---- how the work is divided ----------------------------------------------------------------------------------------

def deal(slots, pairs, most, total):
    """What the codes' kernel's ``choose_deal`` answers: pieces of a pair, 0 where chunks go out in equal shares."""
    if pairs > slots:
        return 1
    even = total // min(slots, -(-total // 8)) + 64
    k = max(1, min(slots // pairs, -(-most // 8)))
    return k if -(-most // k) + (32 if k > 1 else 0) <= even else 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,g,brought,dim,expected", [
    ([12000] + [40] * 60, 2, 1, 64, 0),                    # equal shares: one long request among short ones
    ([9000, 5, 4000, 64] + [33] * 40, 3, 1, 128, 0),
    ([30, 6000, 31] * 3 + [3] * 30, 2, 4, 64, 0),          # ... with two blocks of columns a pair
    ([100, 3, 40, 257] * 30, 6, 1, 64, 1),                 # more pairs than blocks: whole pairs
    ([9, 130] * 45, 4, 5, 128, 1)])
def test_shares_of_unequal_requests(monkeypatch, dtype, lengths, g, brought, dim, expected):
    from yalis_b200.ops import packed
    names = launches(monkeypatch)
    monkeypatch.setattr(packed, "UNPACK_ROWS", 1 << 20)
    c, heads = Cache(lengths, g, dim, 64, seed=len(lengths)), 4 * g
    bring = [min(brought, n) for n in lengths]
    rows = 4 * max(bring)
    tile = 8 if dtype == torch.float32 or rows <= 8 else 16
    pairs = [g * -(-4 * b // tile) for b in bring]
    chunks = [-(-n // 32) for n in lengths]
    slots = torch.cuda.get_device_properties(0).multi_processor_count * (4 if dtype == torch.bfloat16 and tile == 8 else 2)
    assert deal(slots, sum(pairs), max(chunks), sum(a * b for a, b in zip(pairs, chunks))) == expected
    q, pos, q_start = step_of(c, bring, dtype=dtype, heads=heads)
    check(c, q, pos, q_start, heads)
    assert names.count("yalis_packed_attention_mma") == 1 and "yalis_packed_unpack" not in names
    check(c, q, pos, q_start, heads, sums=False)


@pytest.mark.parametrize("heads,g,dim,window", [(8, 2, 64, None), (4, 1, 128, None), (8, 2, 64, 700)])
@pytest.mark.parametrize("portions", [[600, 1, 1], [600, 0, 300]])
def test_portions_that_see_thousands_of_keys(monkeypatch, heads, g, dim, window, portions):
    """Keys of a tile of queries in shares (without a window), several parts of an item's rows in the sums, single tokens beside them."""
    from yalis_b200.ops import packed
    names = launches(monkeypatch, forced=True)
    chosen, splits = [], packed._portion_splits
    monkeypatch.setattr(packed, "_portion_splits", lambda *a: chosen.append(splits(*a)) or chosen[-1])
    c = Cache([4500, 900, 3700], g, dim, 64, seed=dim)
    q, pos, q_start = step_of(c, portions, heads=heads)
    check(c, q, pos, q_start, heads, window)
    assert "yalis_packed_unpack" in names and "yalis_packed_sums_tcgen05" in names
    assert window is not None or chosen[0][0] > 1
    assert -(-600 // (128 // (heads // g))) > 16           # tiles of the longest portion: more than a part has


@pytest.mark.parametrize("heads,g,dim", [(8, 2, 64), (4, 1, 128)])
def test_marks_where_keys_are_shared_out(monkeypatch, heads, g, dim):
    """A value without numbers in the last share and missing pages in others, one of them a whole share's."""
    from yalis_b200.ops import packed
    launches(monkeypatch, forced=True)
    chosen, splits = [], packed._portion_splits
    monkeypatch.setattr(packed, "_portion_splits", lambda *a: chosen.append(splits(*a)) or chosen[-1])
    c = Cache([4500, 900, 3700], g, dim, 64, seed=dim)
    c.words[int(c.table[0, 4100 // 64]), 0, 4100 % 64, 1] = NAN_WORD
    c.table[0, 5], c.table[2, :30], c.table[2, 40] = -1, -1, c.k.shape[0]
    q, pos, q_start = step_of(c, [600, 1, 300], heads=heads)
    got = check(c, q, pos, q_start, heads, flag=BAD_PAGE)
    assert chosen[0][0] > 1
    assert not bool(got[:200].isnan().any()) and bool(got[200:600, :dim].isnan().all()) and not bool(got[600:].isnan().any())


def test_a_replayed_portion_follows_its_values():
    """A recording made without marks meets a value without numbers, a missing page and neither again."""
    from yalis_b200.ops.packed import packed_attention
    c = Cache([300, 80], 2, 64, 16, seed=1)
    pages, table = c.to(DEV)
    q, pos, q_start = step_of(c, [300, 80], heads=8)
    arguments = (q.to(DEV), pages, pos.to(DEV), i32(q_start), table, 300, 8)
    with pytest.MonkeyPatch.context() as patch:
        names = launches(patch, forced=True)
        packed_attention(*arguments)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = packed_attention(*arguments)
    assert names.count("yalis_packed_unpack") == 2
    at, word, page = (int(c.table[0, 9]), 1, 5, 1), c.words[int(c.table[0, 9]), 1, 5, 1].clone(), int(c.table[1, 2])
    whole = None
    for none, missing in ((False, False), (True, False), (False, True), (True, True), (False, False)):
        c.words[at] = NAN_WORD if none else word
        c.table[1, 2] = -1 if missing else page
        pages.words.copy_(c.words)
        table.copy_(c.table)
        graph.replay()
        torch.cuda.synchronize()
        ref, _, size, slack, _ = plain_attention(c, q, q_start, pos, 8)
        y = out.cpu().double()
        assert torch.equal(y.isnan(), ref.isnan()) and bool(ref.isnan().any()) == none
        off = (y - ref).abs() / (2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2 * slack + 300 * 2.0 ** -24) * size + 1e-30)
        assert bool((off[~ref.isnan()] <= 1).all())
        if not (none or missing):
            assert whole is None or torch.equal(out, whole)            # the same bits as before there were marks
            whole = out.clone()


def test_groups_of_requests(monkeypatch):
    """Pools for fewer requests at a time than the step has, sums and single tokens included."""
    from yalis_b200.ops import packed
    names = launches(monkeypatch, forced=True)
    c = Cache([500, 70, 300, 1, 640, 33, 128], 2, 64, 16, seed=3)
    for brought in ([90, 70, 0, 1, 200, 1, 128], [90, 70, 300, 1, 200, 33, 100]):
        q, pos, q_start = step_of(c, brought, heads=8)
        for bytes_held in (1, 3 * 4 * 11 * 2 * 64 * 64):
            monkeypatch.setattr(packed, "UNPACK_BYTES", bytes_held)
            del names[:]
            check(c, q, pos, q_start, 8)
            check(c, q, pos, q_start, 8, sums=False, max_kv_len=660)
            assert names.count("yalis_packed_unpack") > 4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,window", [(64, None), (128, 90)])
@pytest.mark.parametrize("brought", [[1, 1, 1], [3, 1, 2], [120, 1, 1]])
def test_sums_without_room_for_scores(monkeypatch, dtype, dim, window, brought):
    """Steps of few rows whose scores would take too much memory: their products are taken once more."""
    from yalis_b200.ops import packed
    names = launches(monkeypatch, forced=max(brought) > 3)
    monkeypatch.setattr(packed, "SCORE_BYTES", 1000)
    c = Cache([700, 90, 257], 2, dim, 16, seed=dim)
    q, pos, q_start = step_of(c, brought, dtype=dtype, heads=8)
    check(c, q, pos, q_start, 8, window)
    assert "yalis_packed_sums_of_scores" not in names and "yalis_packed_weight_sums" in names


@pytest.mark.parametrize("heads,g,dim,window", [(8, 2, 64, None), (12, 1, 128, 60)])
def test_scores_of_single_tokens_beside_a_portion(monkeypatch, heads, g, dim, window):
    """Room for the single tokens' scores is enough, however many rows the portion has."""
    from yalis_b200.ops import packed
    names = launches(monkeypatch, forced=True)
    c = Cache([70, 400, 1, 257, 300], g, dim, 16, seed=dim)
    monkeypatch.setattr(packed, "SCORE_BYTES", 4 * 5 * heads * 401)
    for brought in ([1, 350, 1, 0, 1], [1, 1, 1, 257, 300]):
        q, pos, q_start = step_of(c, brought, heads=heads)
        del names[:]
        check(c, q, pos, q_start, heads, window, max_kv_len=400)
        assert "yalis_packed_unpack" in names and "yalis_packed_sums_of_scores" in names and "yalis_packed_weight_sums" not in names


def test_the_same_bits_however_the_work_is_divided_from_run_to_run(monkeypatch):
    from yalis_b200.ops.packed import packed_attention
    launches(monkeypatch, forced=True)
    for lengths, brought in (([12000] + [40] * 60, [1] * 61), ([4500, 900, 3700], [600, 1, 300])):
        c = Cache(lengths, 2, 64, 64, seed=9)
        pages, table = c.to(DEV)
        q, pos, q_start = step_of(c, brought, heads=8)
        runs = []
        for _ in range(3):
            sums = c.sums.to(DEV)
            runs.append((packed_attention(q.to(DEV), pages, pos.to(DEV), i32(q_start), table, max(brought), 8, weight_sums=sums), sums))
        assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


# ---- masks by unpacked rows -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [64, 128])
def test_masks_and_extremes_by_unpacked_rows(monkeypatch, dim):
    """Steps of so few rows that the rule of sizes computes them from the codes: rows that see nothing, keys without numbers, scores far
    apart, rows of one value, values of another size, scales and windows at their limits."""
    import test_packed_cache_gpu as steps
    names = launches(monkeypatch, forced=True)
    for run in (lambda: steps.test_rows_that_see_nothing(torch.bfloat16),
                lambda: steps.test_large_scores_and_rows_of_one_value(torch.bfloat16, dim),
                lambda: steps.test_a_row_without_numbers_is_seen_only_by_those_that_see_it(64),
                lambda: steps.test_values_of_another_size_that_have_no_weight(torch.bfloat16, dim, 9, None),
                lambda: steps.test_values_of_another_size_that_have_no_weight(torch.bfloat16, dim, 5, 40),
                lambda: steps.test_queries_of_other_sizes(torch.bfloat16, dim, 9),
                lambda: steps.test_scales_and_windows_at_their_limits(torch.bfloat16, dim, 7),
                lambda: steps.test_portions(torch.bfloat16, 4, 2, dim),
                steps.test_attention_without_a_page):
        del names[:]
        run()
        assert "yalis_packed_unpack" in names
