"""Kernels over pages held in 4 bits against plain torch in 64 bits: rows written and read back, attention of single tokens,
portions and both, sums of weights, eviction, and what each refuses."""

import math

import pytest
import torch

from packed_plain import NAN_WORD, Cache, attention, pack, quantize, refusals, values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---- rows -----------------------------------------------------------------------------------------------------------

def awkward_rows(n, g, dim, dtype, seed):
    """Normal rows, and rows that try a border: constants, one sign only, ties, tiny and huge values, no numbers."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, g, dim, generator=gen) * torch.randn(n, g, 1, generator=gen).mul(3).exp()
    kinds = [torch.zeros(dim), torch.full((dim,), 5.0), torch.full((dim,), -0.3), torch.linspace(-7.5, 7.5, dim).mul(2).round() / 2,
             torch.arange(dim).float() % 16, torch.randn(dim, generator=gen) * 1e-38, torch.randn(dim, generator=gen) * 1e35,
             torch.full((dim,), 2.0 ** 120), torch.full((dim,), 2.0 ** 121), torch.full((dim,), math.nan), torch.full((dim,), -math.inf),
             torch.randn(dim, generator=gen).abs(), -torch.randn(dim, generator=gen).abs(), torch.randn(dim, generator=gen) * 1e-44]
    kinds[5][0] = 1.0
    for i, row in enumerate(kinds):
        x[i % n, (i // n) % g] = row
    x[n - 1, g - 1, dim - 1] = math.nan
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("g,dim,page", [(1, 8, 1), (2, 24, 5), (3, 64, 16), (8, 128, 64), (2, 96, 16), (1, 256, 32)])
def test_rows(dtype, g, dim, page):
    from yalis_b200.ops.packed import PackedPages, packed_kv_read, packed_kv_write
    lengths = [1, 37, 2 * page]
    c = Cache(lengths, g, dim, page)
    pages, table = c.to(DEV)
    before = [t.clone() for t in pages.pools()]
    pos, req = torch.cat([torch.arange(n) for n in lengths]).int(), torch.repeat_interleave(torch.arange(3), torch.tensor(lengths)).int()
    order = torch.randperm(len(pos), generator=torch.Generator().manual_seed(1))
    pos, req = pos[order], req[order]
    req[3] = -1                                                       # padding: nothing is written for it
    k, v = (awkward_rows(len(pos), g, dim, dtype, s) for s in (1, 2))
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    wide = torch.cat([k.flatten(1), torch.zeros(len(pos), 1, dtype=dtype), v.flatten(1)], 1).to(DEV)       # columns of a wider matrix, off any boundary
    kd, vd = wide[:, :g * dim], wide[:, g * dim + 1:]
    packed_kv_write(kd, vd, pages, pos.to(DEV), req.to(DEV), table, error_flag=flag)
    assert int(flag) == 0
    want = {}
    for name, x, pool, j in (("k", k, c.k, 0), ("v", v, c.v, 1)):
        code, word = quantize(x)
        for t in range(len(pos)):
            if req[t] >= 0:
                at, row = int(c.table[req[t], pos[t] // page]), int(pos[t] % page)
                pool[at, :, row], c.words[at, :, row, j] = pack(code[t]), word[t]
        want[name] = values(pack(code), word)
    assert torch.equal(pages.words.cpu(), c.words)                    # every row, those that no token has included
    assert torch.equal(pages.k.cpu(), c.k) and torch.equal(pages.v.cpu(), c.v)
    assert before[0].shape == pages.k.shape
    for out in (torch.float32, torch.bfloat16):
        got = packed_kv_read(pages, pos.to(DEV), req.to(DEV), table, dtype=out, error_flag=flag)
        for x, name in zip(got, ("k", "v")):
            ref = want[name].clone()
            ref[3] = 0                                                # a token of no request reads as zeros
            torch.testing.assert_close(x.cpu().double(), ref.flatten(1), rtol=0, atol=0, equal_nan=True)   # every value is a bfloat16 number
    assert int(flag) == 0
    # aligned rows take wide loads: the same bits
    again = PackedPages(*[t.clone() for t in before])
    packed_kv_write(k.flatten(1).to(DEV), v.flatten(1).to(DEV), again, pos.to(DEV), req.to(DEV), table)
    assert all(torch.equal(a, b) for a, b in zip(again.pools(), pages.pools()))


def test_rows_error_is_half_a_step():
    from yalis_b200.ops.packed import PackedPages, packed_kv_read, packed_kv_write
    x = torch.randn(500, 2 * 128, generator=torch.Generator().manual_seed(3)).to(DEV)
    pages = PackedPages.empty(500, 2, 1, 128, DEV)
    pos, req, table = torch.zeros(500, dtype=torch.int32, device=DEV), torch.arange(500, dtype=torch.int32, device=DEV), torch.arange(500, dtype=torch.int32, device=DEV)[:, None]
    packed_kv_write(x, -x, pages, pos, req, table)
    k, v = packed_kv_read(pages, pos, req, table, dtype=torch.float32)
    y = x.view(500, 2, 128)
    step = (y.amax(-1).clamp(min=0) - y.amin(-1).clamp(max=0)) / 15 * 1.125          # four significant bits, rounded up
    assert bool(((k.view_as(y) - y).abs() <= step[..., None] * (0.5 + 1e-6)).all()) and bool(((v.view_as(y) + y).abs() <= step[..., None] * (0.5 + 1e-6)).all())


def test_rows_without_a_page():
    from yalis_b200.ops.packed import packed_kv_read, packed_kv_write
    c = Cache([20, 20], 2, 64, 16)
    c.table[1, 1] = c.k.shape[0]                                      # past the pool
    pages, table = c.to(DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    pos, req = i32([19, 19, 1000, 5]), i32([0, 1, 0, 1])
    x = torch.ones(4, 128, device=DEV)
    packed_kv_write(x, x, pages, pos, req, table, error_flag=flag)
    assert int(flag) == 2
    flag.zero_()
    k, v = packed_kv_read(pages, pos, req, table, dtype=torch.float32, error_flag=flag)
    held = 14 * 9 / 128              # a row of ones: 1 / 15 rounded up to four bits is 9 / 128, of which 1 is 14.2
    assert int(flag) == 2 and k[:, 0].tolist() == [held, 0, 0, held] and v[:, 127].tolist() == [held, 0, 0, held]


# ---- attention ------------------------------------------------------------------------------------------------------

@pytest.fixture(params=["by the rule", "always unpacked"])
def portions_by_both(request, monkeypatch):
    """Portions by whichever way the step's sizes choose, and by the prompt kernel wherever they have more rows than 64."""
    from yalis_b200.ops import packed
    if request.param == "always unpacked":
        monkeypatch.setattr(packed, "UNPACK_FEW", 0)


def step_of(cache, brought, seed=0, dtype=torch.bfloat16, heads=4, empty=()):
    """Rows of the requests' last ``brought`` tokens (0: a request that brings none)."""
    gen = torch.Generator().manual_seed(seed)
    q_start, pos = [0], []
    for n, length in zip(brought, cache.lengths):
        pos += range(length - n, length)
        q_start.append(q_start[-1] + n)
    q = torch.randn(len(pos), heads * cache.dim, generator=gen).to(dtype)
    pos = torch.tensor(pos, dtype=torch.int32)
    for t in empty:
        pos[t] = -1
    return q, pos, q_start


def check_attention(cache, q, pos, q_start, heads, window=None, sums=True, max_q_len=None, scale=None):
    from yalis_b200.ops.packed import packed_attention
    pages, table = cache.to(DEV)
    n, width = q.shape
    before = cache.sums.to(DEV)
    total = before.clone() if sums else None
    # queries are columns of a wider matrix, results too, with a row more than there are tokens of requests
    wide = torch.full((n + 1, width + 24), math.nan, dtype=q.dtype, device=DEV)
    wide[:n, 8:8 + width] = q.to(DEV)
    result = torch.full((n + 1, width + 16), 7.0, dtype=q.dtype, device=DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    rows = torch.cat([pos, torch.zeros(1, dtype=torch.int32)]).to(DEV)
    longest = max([b - a for a, b in zip(q_start[:-1], q_start[1:])] + [0])
    got = packed_attention(wide[:, 8:8 + width], pages, rows, i32(q_start), table, longest if max_q_len is None else max_q_len, heads, window=window,
                           weight_sums=total, out=result[:, 8:8 + width], error_flag=flag, scale=scale)
    assert int(flag) == 0
    ref, a, size, slack, sum_slack = attention(cache, q, q_start, pos, heads, window, scale)
    y, half = got[:n].cpu().double(), HALF[q.dtype]
    # one rounding of the result, one of the weights, the scores' error twice (weight and normaliser), sums of float32
    bound = half * ref.abs() + (half + 2 * slack + 300 * 2.0 ** -24) * size + 1e-30
    off = ((y - ref).abs() / bound)
    assert bool((off <= 1).all()), float(off.max())
    assert bool((result[n] == 7).all()) and bool((result[:, :8] == 7).all()) and bool((result[:, -8:] == 7).all())
    if sums:
        ref_sums = cache.sums.double() + a
        err = (total.cpu().double() - ref_sums).abs()
        assert bool((err <= sum_slack + 2 * 2.0 ** -24 * ref_sums).all()), float((err / (sum_slack + 2.0 ** -23 * ref_sums)).max())
        assert torch.equal(total.cpu()[a == 0], cache.sums[a == 0])
    return got


LAYOUTS = [(1, 1, 64), (4, 2, 128), (8, 1, 64), (3, 1, 128), (12, 1, 64), (16, 1, 128), (20, 1, 64), (6, 2, 256), (4, 1, 24), (2, 2, 96), (4, 2, 8)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,g,dim", LAYOUTS)
def test_single_tokens(dtype, heads, g, dim):
    for page, window in ((16, None), (5, None), (64, 37), (16, 1)):
        c = Cache([1, 2, 15, 16, 17, 33, 64, 129, 300], g, dim, page, seed=page)
        q, pos, q_start = step_of(c, [1] * 9, dtype=dtype, heads=heads, seed=dim)
        check_attention(c, q, pos, q_start, heads, window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,g,dim", LAYOUTS)
@pytest.mark.usefixtures("portions_by_both")
def test_portions(dtype, heads, g, dim):
    for page, window in ((16, None), (64, 20)):
        c = Cache([1, 5, 40, 130], g, dim, page, seed=page)
        q, pos, q_start = step_of(c, [1, 5, 0, 33], dtype=dtype, heads=heads, seed=dim)
        check_attention(c, q, pos, q_start, heads, window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,g,dim,page", [(4, 1, 128, 64), (8, 2, 64, 16)])
@pytest.mark.parametrize("window", [None, 50])
@pytest.mark.usefixtures("portions_by_both")
def test_whole_prompts_beside_single_tokens(dtype, heads, g, dim, page, window):
    c = Cache([200, 1, 333, 64, 65], g, dim, page, seed=3)
    q, pos, q_start = step_of(c, [200, 1, 1, 64, 1], dtype=dtype, heads=heads)
    check_attention(c, q, pos, q_start, heads, window)
    check_attention(c, q, pos, q_start, heads, window, sums=False, scale=0.2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_long_request_and_many_short(dtype):
    c = Cache([5000], 1, 128, 64, seed=4)
    check_attention(c, *step_of(c, [1], dtype=dtype, heads=4), 4)
    c = Cache([900] + [3] * 70, 2, 64, 16, seed=5)
    check_attention(c, *step_of(c, [1] * 71, dtype=dtype, heads=4), 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.usefixtures("portions_by_both")
def test_rows_that_see_nothing(dtype):
    c = Cache([40, 3, 20], 2, 64, 16)
    q, pos, q_start = step_of(c, [1, 1, 1], dtype=dtype, heads=4, empty=(1,))
    got = check_attention(c, q, pos, q_start, 4)
    assert bool((got[1] == 0).all())
    check_attention(c, *step_of(c, [0, 0, 1], dtype=dtype, heads=4), 4, max_q_len=3)
    check_attention(c, q[:0], pos[:0], [0, 0, 0, 0], 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 24])
@pytest.mark.usefixtures("portions_by_both")
def test_large_scores_and_rows_of_one_value(dtype, dim):
    c = Cache([150, 70], 1, dim, 16, seed=6)
    q, pos, q_start = step_of(c, [1, 4], dtype=dtype, heads=4)
    check_attention(c, q * 30, pos, q_start, 4)                        # weights of one key, others far below the smallest number
    c.k[:] = 0x77
    check_attention(c, q, pos, q_start, 4)
    c.words[..., 0] = torch.where(c.words[..., 0] == NAN_WORD, c.words[..., 0], torch.tensor(0x0080 | 7, dtype=torch.int16))   # steps of 2^-126
    check_attention(c, q, pos, q_start, 4)


@pytest.mark.parametrize("dim", [64, 24])
@pytest.mark.usefixtures("portions_by_both")
def test_a_row_without_numbers_is_seen_only_by_those_that_see_it(dim):
    from yalis_b200.ops.packed import packed_attention
    c = Cache([40, 40], 2, dim, 16)
    at = int(c.table[0, 1])
    c.words[at, 1, 3, 0] = NAN_WORD                                    # key 19 of request 0, head 1
    pages, table = c.to(DEV)
    for n in (1, 30):
        q, pos, q_start = step_of(c, [n, n], heads=4)
        got = packed_attention(q.to(DEV), pages, pos.to(DEV), i32(q_start), table, n, 4).view(2, n, 4, dim)
        assert bool(got[0, -1, 2:].isnan().all()) and not bool(got[0, :, :2].isnan().any()) and not bool(got[1].isnan().any())
        if n == 30:
            assert not bool(got[0, :9].isnan().any())                  # positions 10 .. 18


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,n,window", [(64, 1, None), (128, 1, 40), (128, 5, None), (64, 9, 33), (24, 4, 20), (64, 40, None)])
@pytest.mark.usefixtures("portions_by_both")
def test_values_of_another_size_that_have_no_weight(dtype, dim, n, window):
    """Values 2^100 times as large as the others', at places that a row does not see (behind its window, after it, behind the last)
    or gives no weight, take nothing from its accuracy."""
    c = Cache([70 + n, 90 + n], 2, dim, 16, seed=dim + n)
    large = lambda r, j: c.words[int(c.table[r, j // 16]), :, j % 16, 1].copy_(torch.tensor(2.0 ** 100).bfloat16().view(torch.int16) | 7)
    q, pos, q_start = step_of(c, [n, n], dtype=dtype, heads=4)
    if n > 1:
        large(1, 90 + n - 1)                               # the last row's own place: its value is seen by nobody else
    if window is not None:
        large(0, 70 - window)                              # just behind the first row's window
    else:                                                  # a key of scores about 140 or -140: all of a row's weight or none
        c.words[int(c.table[0, 4]), :, 69 % 16, 0] = 0x4180
        large(0, 69)
    check_attention(c, q, pos, q_start, 4, window=window, sums=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,n", [(64, 1), (128, 5), (64, 9)])
def test_queries_of_other_sizes(dtype, dim, n):
    """Heads, and elements of a head, that lie many powers of two apart; rows of zeros."""
    c = Cache([n, 90 + n], 2, dim, 16, seed=n)
    q, pos, q_start = step_of(c, [n, n], dtype=dtype, heads=8)
    q = q.view(2 * n, 8, dim)
    q *= (2.0 ** torch.tensor([0, -60, -14, 3, -110, -24, 0, 1])).to(dtype)[:, None]
    q[:, 0, ::2] *= 2.0 ** -13
    q[:, 3, 5] = 2.0 ** 7
    q[0, 6] = 0
    check_attention(c, q.view(2 * n, 8 * dim), pos, q_start, 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,n", [(64, 1), (128, 7), (24, 3), (64, 70)])
@pytest.mark.usefixtures("portions_by_both")
def test_scales_and_windows_at_their_limits(dtype, dim, n):
    c = Cache([n, 90 + n], 2, dim, 16, seed=n)
    q, pos, q_start = step_of(c, [n, n], dtype=dtype, heads=4)
    for scale in (0.0, 1e-38, -0.2):                       # no weight differs from another; scales whose products with a step underflow
        check_attention(c, q, pos, q_start, 4, scale=scale)
    for window in (1, 2 ** 31 - 1, 2 ** 32 + 5):
        check_attention(c, q, pos, q_start, 4, window=window)


@pytest.mark.parametrize("dtype,n", [(torch.float32, 20), (torch.float32, 1), (torch.bfloat16, 1), (torch.bfloat16, 40)])
@pytest.mark.usefixtures("portions_by_both")
def test_a_table_for_many_more_tokens_than_there_are(dtype, n):
    c = Cache([30 + n, 90 + n], 2, 64, 64, seed=n)
    c.table = torch.cat([c.table, torch.full((2, 70000), -1, dtype=torch.int32)], 1)
    q, pos, q_start = step_of(c, [n, n], dtype=dtype, heads=4)
    check_attention(c, q, pos, q_start, 4)


@pytest.mark.usefixtures("portions_by_both")
def test_attention_without_a_page():
    from yalis_b200.ops.packed import packed_attention
    for dim, n in ((64, 1), (128, 1), (24, 1), (64, 20)):
        c = Cache([40, 40], 2, dim, 16)
        c.table[0, 1] = -1
        pages, table = c.to(DEV)
        q, pos, q_start = step_of(c, [n, n], heads=4)
        flag = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = packed_attention(q.to(DEV), pages, pos.to(DEV), i32(q_start), table, n, 4, error_flag=flag)
        assert int(flag) & 2
        ref = attention(c, q, q_start, torch.cat([torch.full((n,), -1, dtype=torch.int32), pos[n:]]), 4)[0]
        torch.testing.assert_close(got[n:].cpu().double(), ref[n:], rtol=2 ** -6, atol=2 ** -6)         # the other request is not touched


def test_a_replayed_step_follows_its_inputs():
    """One recording, replayed for other lengths, pages and queries; two recordings in flight on two streams."""
    from yalis_b200.ops.packed import packed_attention
    c = Cache([700, 90, 300], 2, 128, 64, seed=8)
    pages, table = c.to(DEV)
    q, pos, q_start = step_of(c, [1, 1, 1], heads=8)
    q, pos, start = q.to(DEV), pos.to(DEV), i32(q_start)
    sums = torch.zeros(c.sums.shape, device=DEV)
    call = lambda: packed_attention(q, pages, pos, start, table, 1, 8, weight_sums=sums)
    call()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for lengths in ([700, 90, 300], [1, 64, 299], [650, 1, 65]):
        pos.copy_(torch.tensor([n - 1 for n in lengths], dtype=torch.int32))
        q.copy_(torch.randn(3, 8 * 128, generator=torch.Generator().manual_seed(lengths[0])))
        sums.zero_()
        ref, a, _, _, _ = attention(c, q.cpu(), q_start, pos.cpu(), 8)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for out in outs:
            torch.testing.assert_close(out.cpu().double(), ref, rtol=2 ** -6, atol=2 ** -7)
        torch.testing.assert_close(sums.cpu().double(), 6 * a, rtol=1e-4, atol=1e-6)


def test_calls_on_two_streams_at_once():
    """Steps of different requests on two streams, neither waiting for the other, with workspaces that grow on the way."""
    from yalis_b200.ops.packed import packed_attention
    streams, want, got = [torch.cuda.Stream() for _ in range(2)], [], [[], []]
    inputs = []
    for i in range(2):
        c = Cache([900 + 300 * i, 90, 500], 2, 128, 16, seed=20 + i)
        for brought, heads in (([1, 1, 1], 4), ([1, 3, 2], 16), ([60, 1, 70], 8)):
            q, pos, q_start = step_of(c, brought, heads=heads, seed=i)
            pages, table = c.to(DEV)
            inputs.append((i, q.to(DEV), pages, pos.to(DEV), i32(q_start), table, max(brought), heads))
    for i, *args in inputs:
        want.append(packed_attention(*args))
    torch.cuda.synchronize()
    for _ in range(5):
        for i, *args in inputs:
            with torch.cuda.stream(streams[i]):
                got[i].append(packed_attention(*args))
    torch.cuda.synchronize()
    for i in range(2):
        for k, out in enumerate(got[i]):
            assert torch.equal(out, want[3 * i + k % 3])


@pytest.mark.usefixtures("portions_by_both")
def test_the_same_step_gives_the_same_bits():
    from yalis_b200.ops.packed import packed_attention
    c = Cache([1500, 7, 64, 800], 2, 64, 16, seed=9)
    pages, table = c.to(DEV)
    for brought in ([1, 1, 1, 1], [3, 7, 1, 100]):
        q, pos, q_start = step_of(c, brought, heads=8)
        runs = []
        for _ in range(3):
            sums = c.sums.to(DEV)
            runs.append((packed_attention(q.to(DEV), pages, pos.to(DEV), i32(q_start), table, max(brought), 8, weight_sums=sums), sums))
        assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


# ---- eviction -------------------------------------------------------------------------------------------------------

def evicted(cache, keep, recent, sums):
    """(kept, and what the pools hold afterwards) in plain torch."""
    pools = [t.clone() for t in (cache.k, cache.v, cache.words, sums)]
    kept = torch.full((len(cache.lengths), cache.g, keep), -1, dtype=torch.int32)
    for r, n in enumerate(cache.lengths):
        for h in range(cache.g):
            chosen = list(range(n))
            if n > keep:
                score = [float(x) for x in cache.rows(r, n, sums)[:, h]]
                rank = sorted(range(n - recent), key=lambda j: (-(score[j] if score[j] == score[j] else -math.inf), score[j] != score[j], j))
                chosen = sorted(rank[:keep - recent]) + list(range(n - recent, n))
            kept[r, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
            src = [(int(cache.table[r, j // cache.page]), h, j % cache.page) for j in chosen]
            held = [[p[s].clone() for s in src] for p in pools]
            for p, rows in zip(pools, held):
                for j, row in enumerate(rows):
                    p[int(cache.table[r, j // cache.page]), h, j % cache.page] = row
    return kept, pools


@pytest.mark.parametrize("g,dim,page", [(1, 8, 1), (2, 64, 16), (3, 24, 5), (8, 128, 64)])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (20, 0), (20, 7), (50, 50), (130, 31), (2000, 9)])
def test_eviction(g, dim, page, keep, recent):
    from yalis_b200.ops.packed import evict_tokens
    c = Cache([1, 19, 20, 21, 131, 300, 0], g, dim, page, seed=keep)
    sums = c.sums.clone()
    sums[sums < 0.2] = 0.0                                            # ties, zeros of both signs, and no numbers
    sums[(sums > 0.2) & (sums < 0.25)] = -0.0
    sums[(sums > 0.25) & (sums < 0.28)] = math.nan
    sums[(sums > 0.5) & (sums < 0.6)] = 0.5
    sums[(sums > 0.6) & (sums < 0.62)] = -1.0
    sums[(sums > 0.62) & (sums < 0.63)] = math.inf
    pages, table = c.to(DEV)
    total, flag = sums.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    kept = evict_tokens(pages.pools(), total, i32(c.lengths), table, keep, recent, error_flag=flag)
    want, pools = evicted(c, keep, recent, sums)
    assert int(flag) == 0 and torch.equal(kept.cpu(), want)
    for got, ref in zip(pages.pools() + (total,), pools):
        assert torch.equal(got.cpu().view(torch.int32 if got.dtype == torch.float32 else got.dtype), ref.view(torch.int32 if ref.dtype == torch.float32 else ref.dtype))


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 3), (torch.bfloat16, 1)])
def test_eviction_from_a_plain_cache(dtype, dim):
    from yalis_b200.ops.packed import evict_tokens
    c = Cache([2500, 1300], 2, 8, 16, seed=2)
    gen = torch.Generator().manual_seed(0)
    pools = [torch.randn(c.k.shape[:3] + (dim,), generator=gen).to(dtype) for _ in range(2)]
    on_gpu, total = [p.to(DEV) for p in pools], c.sums.to(DEV)
    kept = evict_tokens(on_gpu, total, i32(c.lengths), c.table.to(DEV), 1200, 100)
    for r, n in enumerate(c.lengths):
        for h in range(2):
            j = kept[r, h].cpu().long()
            score = c.rows(r, n, c.sums)[:, h].clone()
            score[n - 100:] = 2.0
            assert torch.equal(j, torch.sort(torch.topk(score, 1200).indices).values)
            for a, b in zip(pools + [c.sums], on_gpu + [total]):
                assert torch.equal(c.rows(r, 1200, b.cpu())[:, h], c.rows(r, n, a)[j, h])


def test_eviction_without_a_page():
    from yalis_b200.ops.packed import evict_tokens
    c = Cache([40, 40], 2, 64, 16)
    c.table[0, 2] = c.k.shape[0] + 5
    pages, table = c.to(DEV)
    total, flag = c.sums.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    kept = evict_tokens(pages.pools(), total, i32([40, 40]), table, 10, error_flag=flag)
    assert int(flag) == 2 and bool((kept[0] == -1).all()) and bool((kept[1] >= 0).all())
    assert torch.equal(c.rows(0, 32, total.cpu()), c.rows(0, 32, c.sums)) and torch.equal(c.rows(0, 32, pages.k.cpu()), c.rows(0, 32, c.k))
    flag.zero_()
    evict_tokens(pages.pools(), total, i32([1000, 5]), table, 10, error_flag=flag)       # longer than its row of the table
    assert int(flag) == 2


# ---- together -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.usefixtures("portions_by_both")
def test_a_request_through_all_of_them(dtype):
    """A prompt in two portions, tokens one by one with their weights counted, the cache cut, and tokens behind the cut: as one
    attention over the same rows in 64 bits."""
    from yalis_b200.ops.packed import PackedPages, evict_tokens, packed_attention, packed_kv_read, packed_kv_write
    heads, g, dim, page, keep, recent = 8, 2, 64, 16, 48, 8
    gen = torch.Generator().manual_seed(11)
    pages = PackedPages.empty(8, g, page, dim, DEV)
    table = torch.tensor([[5, 2, 7, 0, 1, 3, 6, 4]], dtype=torch.int32, device=DEV)
    sums = torch.zeros(8, g, page, device=DEV)
    c = Cache([100], g, dim, page, spare=1)
    c.table = table.cpu()
    held = torch.arange(0)
    counted = torch.zeros(8, g, page).double()

    def step(n, at):
        nonlocal counted
        qkv = torch.randn(n, (heads + 2 * g) * dim, generator=gen).to(dtype).to(DEV)
        pos, req = torch.arange(at, at + n, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
        k, v = qkv[:, heads * dim:(heads + g) * dim], qkv[:, (heads + g) * dim:]
        packed_kv_write(k, v, pages, pos, req, table)
        got = packed_attention(qkv, pages, pos, i32([0, n]), table, n, heads, weight_sums=sums)
        c.k, c.v, c.words = (t.cpu() for t in pages.pools())
        ref, a, size, slack, sum_slack = attention(c, qkv.cpu(), [0, n], pos.cpu(), heads)
        half = HALF[dtype]
        assert bool(((got.cpu().double() - ref).abs() <= half * ref.abs() + (half + 2 * slack + 300 * 2.0 ** -24) * size).all())
        counted += a
        written = values(c.rows(0, at + n, c.k), c.rows(0, at + n, c.words)[..., 0])[at:]
        code, word = quantize(k.cpu().view(n, g, dim))
        assert torch.equal(written, values(pack(code), word))

    step(40, 0)
    step(29, 40)
    for at in range(69, 75):
        step(1, at)
    torch.testing.assert_close(sums.cpu().double(), counted, rtol=1e-4, atol=1e-6)
    c.lengths, c.sums = [75], sums.cpu()
    want, pools = evicted(c, keep, recent, c.sums)
    kept = evict_tokens(pages.pools(), sums, i32([75]), table, keep, recent)
    assert torch.equal(kept.cpu(), want) and all(torch.equal(a.cpu(), b) for a, b in zip(pages.pools(), pools))
    counted = sums.cpu().double()
    for at in range(keep, keep + 3):
        step(1, at)
    torch.testing.assert_close(sums.cpu().double(), counted, rtol=1e-4, atol=1e-6)


# ---- refusals -------------------------------------------------------------------------------------------------------

def test_refusals():
    from yalis_b200.ops._lib import LAUNCHES, KernelError
    for what, call in refusals(DEV):
        before = LAUNCHES[0]
        with pytest.raises(KernelError):
            call()
            print("not refused:", what)
        assert LAUNCHES[0] == before, what


def test_empty_calls():
    from yalis_b200.ops.packed import evict_tokens, packed_kv_read, packed_kv_write
    c = Cache([40], 2, 64, 16)
    pages, table = c.to(DEV)
    none = i32([])
    f = torch.zeros(0, 128, device=DEV)
    before = [t.clone() for t in pages.pools()]
    packed_kv_write(f, f, pages, none, none, table)
    k, v = packed_kv_read(pages, none, none, table)
    assert k.shape == v.shape == (0, 128)
    assert evict_tokens(pages.pools(), c.sums.to(DEV), none, table, 4).shape == (0, 2, 4)
    assert all(torch.equal(a, b) for a, b in zip(before, pages.pools()))
