"""A paged cache held in 4 bits: rows written and read, attention over it, and eviction by accumulated weights.

The format (``csrc/packed.cuh``): a row of one token and KV head is one 4-bit code per element and a 16-bit word with the row's
step and zero, value = (code - zero) * step; every value is a bfloat16 number.  A token takes ``head_dim / 2 + 2`` bytes for its
key and as many for its value, per KV head.
"""

from __future__ import annotations

import ctypes
import functools
import itertools
import math
import struct
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from ._lib import BF16, F32, KernelError, check, dtype_code, lib, need
from .attention import (PREFILL_SPLIT_GAIN, PREFILL_SPLIT_MIN_TILES, PREFILL_SPLIT_START_UP, PREFILL_SPLIT_UNSHARED, _policy_lib,
                        sm_count)

_TYPES = {"i": ctypes.c_int, "s": ctypes.c_char_p}
_entries = {}


def _function(name: str, signature: str, result=ctypes.c_int):
    """The library's function with its argument types set."""
    fn = getattr(lib(), name)
    fn.argtypes, fn.restype = [_TYPES[c] for c in signature], result
    return fn


def _entry(name: str, signature: str):
    """The library's launch of that name, called with plain numbers in one array of slots (``csrc/slots.cuh``): these calls are made for
    every layer of a step, and handing thirty arguments over one by one takes longer than the smaller kernels run."""
    fn = _entries.get(name)
    if fn is None:
        launch = _function(name + "_slots", "s")
        pack = struct.Struct("".join("d" if c == "f" else "q" for c in signature)).pack
        fn = _entries[name] = lambda *arguments: launch(pack(*arguments))
    return fn


@dataclass(frozen=True)
class PackedPages:
    """Pages of keys and values in 4 bits: ``k`` and ``v`` uint8 [pages, kv_heads, page_size, head_dim / 2] (element 2b in the low
    half of byte b, 2b + 1 in the high half), ``words`` int16 [pages, kv_heads, page_size, 2] (of the key and of the value: the
    bits of the step as bfloat16, with the zero in the lowest four).  ``head_dim`` is a multiple of 8 up to 256."""

    k: torch.Tensor
    v: torch.Tensor
    words: torch.Tensor

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, device) -> "PackedPages":
        if head_dim < 8 or head_dim % 8 or head_dim > 256:
            raise KernelError(f"PackedPages: head_dim {head_dim} must be a multiple of 8 up to 256")
        make = lambda *last, dtype: torch.empty((num_pages, num_kv_heads, page_size) + last, dtype=dtype, device=device)
        return cls(make(head_dim // 2, dtype=torch.uint8), make(head_dim // 2, dtype=torch.uint8), make(2, dtype=torch.int16))

    @property
    def head_dim(self) -> int:
        return 2 * self.k.shape[3]

    @property
    def num_kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    def pools(self) -> Tuple[torch.Tensor, ...]:
        """The tensors that hold a token's rows (what ``evict_tokens`` moves)."""
        return self.k, self.v, self.words


def _need_here(name: str, *tensors: Optional[torch.Tensor]) -> int:
    """Every tensor on the current device, whose stream the kernels are launched on; returns its number."""
    here = -2
    for t in tensors:
        if t is not None:
            at = t.get_device()
            if at != here:
                if at < 0:
                    raise KernelError(f"{name}: every tensor must be on the GPU (there is no CPU path)")
                if here >= 0 or at != torch.cuda.current_device():
                    raise KernelError(f"{name}: every tensor must be on the current device")
                here = at
    return here


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _pages_arguments(name: str, pages: PackedPages):
    k, v, words = pages.k, pages.v, pages.words
    shape = k.shape
    if not (k.dtype is torch.uint8 and v.dtype is torch.uint8 and len(shape) == 4 and v.shape == shape and k.is_contiguous() and v.is_contiguous()):
        raise KernelError(f"{name}: codes must be contiguous uint8 [pages, kv_heads, page_size, head_dim / 2]")
    num_pages, g, page_size, half = shape
    if not (words.dtype is torch.int16 and words.shape == shape[:3] + (2,) and words.is_contiguous()):
        raise KernelError(f"{name}: words must be contiguous int16 [pages, kv_heads, page_size, 2]")
    if half % 4 or not 4 <= half <= 128:
        raise KernelError(f"{name}: head_dim {2 * half} must be a multiple of 8 up to 256")
    if num_pages * g * page_size >= 1 << 31:
        raise KernelError(f"{name}: {num_pages} pages of {g} x {page_size} rows are 2^31 rows or more")
    at = (k.data_ptr(), v.data_ptr(), words.data_ptr())
    if (at[0] | at[1] | at[2]) % 16:
        raise KernelError(f"{name}: pools must start on 16-byte boundaries")
    return at + (num_pages, page_size, g, 2 * half)


def _check_index(name: str, n: int, block_table: torch.Tensor, *per_token: torch.Tensor) -> Tuple[int, int]:
    """Checks the arrays of a step's tokens and the block table, whose (rows, columns) it returns."""
    for t in per_token:
        if not (t.dtype is torch.int32 and t.dim() == 1 and t.shape[0] == n and t.is_contiguous()):
            raise KernelError(f"{name}: positions/req_of_token: int32 [N]")
    if not (block_table.dtype is torch.int32 and block_table.dim() == 2 and block_table.is_contiguous()):
        raise KernelError(f"{name}: block_table must be contiguous int32 [R, width]")
    return block_table.shape


def _flag_address(name: str, error_flag: Optional[torch.Tensor]) -> int:
    if error_flag is None:
        return 0
    need(error_flag.dtype == torch.int32 and error_flag.numel() >= 1, name, "the error word must be int32")
    return error_flag.data_ptr()


_workspaces = {}


def _workspace(device: int, raw: int, counters: int, floats: int):
    """(zeroed int32 counters, which every launch leaves at zero, scratch memory) for a launch on the current stream: kept per
    stream, whose launches run one after the other; a recording, which may be replayed on any stream, gets its own with every
    launch."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(counters, dtype=torch.int32, device=device), torch.empty(floats, dtype=torch.float32, device=device)
    held = _workspaces.get((device, raw))
    if held is None or held[0].shape[0] < counters or held[1].shape[0] < floats:
        held = _workspaces[device, raw] = (torch.zeros(max(counters, 2048), dtype=torch.int32, device=device),
                                           torch.empty(floats, dtype=torch.float32, device=device))
    return held


_mma_launches = {}


def _mma_launch(device: int, code: int, dim: int, columns: int) -> Tuple[int, int]:
    """(blocks, floats of scratch memory) of the tensor-core kernel."""
    key = (device, code, dim, columns)
    found = _mma_launches.get(key)
    if found is None:
        blocks = _function("yalis_packed_attention_mma_blocks", "iii")(code, dim, columns)
        floats = _function("yalis_packed_attention_mma_scratch_floats", "iii", ctypes.c_longlong)(blocks, dim, columns)
        found = _mma_launches[key] = (blocks, floats)
    return found


def packed_kv_write(k: torch.Tensor, v: torch.Tensor, pages: PackedPages, positions: torch.Tensor, req_of_token: torch.Tensor,
                    block_table: torch.Tensor, error_flag: Optional[torch.Tensor] = None) -> None:
    """Store the keys and values of a step's tokens, [N, kv_heads * head_dim] in float32 or bfloat16 (column blocks of wider
    matrices are taken), in 4 bits: token n goes to place ``positions[n]`` of the request whose block-table row is
    ``req_of_token[n]`` (-1: nowhere).  No two tokens may share a place.  A token without a page is left out and raises the error
    word's bit.  Rows with a NaN, an infinity or a magnitude above 2^120 read back as NaN throughout."""
    name = "packed_kv_write"
    device = _need_here(name, k, v, pages.k, pages.v, pages.words, positions, req_of_token, block_table, error_flag)
    held, shape, size, code = _pages_arguments(name, pages), k.shape, k.element_size(), dtype_code(k.dtype)
    (k_step, k_unit), (v_step, v_unit) = (k.stride(), v.stride()) if k.dim() == v.dim() == 2 else ((0, 0), (0, 0))
    if not (k.dtype is v.dtype and k_unit == v_unit == 1 and v.shape == shape and shape[1] == held[5] * held[6]):
        raise KernelError(f"{name}: k and v must be [N, kv_heads * head_dim] of one dtype with unit inner stride")
    _, columns = _check_index(name, shape[0], block_table, positions, req_of_token)
    flag, k_at, v_at = _flag_address(name, error_flag), k.data_ptr(), v.data_ptr()
    check(_rows_entry()(1, k_at, v_at, k_step, v_step, code, *held, positions.data_ptr(), req_of_token.data_ptr(),
                        block_table.data_ptr(), columns, shape[0], (k_at | v_at | k_step * size | v_step * size) % 16 == 0, flag,
                        _raw_stream(device)), name)


def _rows_entry():
    return _entry("yalis_packed_rows", "ippllipppiiiipppiiipp")


def packed_kv_read(pages: PackedPages, positions: torch.Tensor, req_of_token: torch.Tensor, block_table: torch.Tensor,
                   dtype: torch.dtype = torch.bfloat16, error_flag: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values, each [N, kv_heads * head_dim] in ``dtype``, of the tokens at ``positions`` of the requests
    ``req_of_token``: what ``packed_kv_write`` left there, exactly.  Tokens of no request (-1) and tokens without a page (which
    raise the error word's bit) read as zeros."""
    name = "packed_kv_read"
    device = _need_here(name, pages.k, pages.v, pages.words, positions, req_of_token, block_table, error_flag)
    held, n, code = _pages_arguments(name, pages), positions.shape[0] if positions.dim() else -1, dtype_code(dtype)
    _, columns = _check_index(name, n, block_table, positions, req_of_token)
    flag, width = _flag_address(name, error_flag), held[5] * held[6]
    both = torch.empty(2, n, width, dtype=dtype, device=device)        # one allocation
    at = both.data_ptr()
    check(_rows_entry()(0, at, at + n * width * both.element_size(), width, width, code, *held, positions.data_ptr(), req_of_token.data_ptr(),
                        block_table.data_ptr(), columns, n, True, flag, _raw_stream(device)), name)
    return both.unbind(0)


_LONGEST = (1 << 31) - 1   # places are 32-bit numbers
# Query rows of a pair (tokens * heads of a KV head) beyond which portions are unpacked for the prompt kernel: 64, and more where there
# are few keys (of all KV heads and requests), since that way is two launches and 28 us at least.  By codes / unpacked, us, heads of
# 64: 16 requests of 8,000 tokens, 8 KV heads: 64 rows 150 / 160, 128 rows 284 / 150; of 1,000: 64 rows 34 / 40, 128 rows 65 / 39; one
# of 1,000: 256 rows 18 / 28.
UNPACK_ROWS, UNPACK_FEW = 64, 1 << 21
UNPACK_PAGE = 64          # keys of a page of the unpacked pools
UNPACK_BYTES = 2 << 30    # of unpacked keys and values at a time (one request may take more)
_unpackings = itertools.count(1)       # numbers by which a launch tells its own note that keys are marked from what the memory held before
SCORE_BYTES = 1 << 30     # of scores that a step of few rows may leave for its sums; beyond, the products are taken once more


def _unpacking_pays(rows: int, keys: int) -> bool:
    """Whether portions of up to ``rows`` query rows a pair, over up to ``keys`` keys in all, go by unpacked rows."""
    return rows > UNPACK_ROWS + UNPACK_FEW // max(1, keys)


@functools.lru_cache(maxsize=4096)
def _portion_splits(portions: int, q_len: int, kv_len: int, per: int, g: int, sms: int) -> Tuple[int, int]:
    """(shares of a tile's keys, tiles of keys of a share) for the prompt kernel, as the plain cache's steps choose them
    (``prefill_kv_splits``), for ``portions`` portions of ``q_len`` tokens that end at place ``kv_len``."""
    q_lens, before = (np.full(portions, v, dtype=np.int32) for v in (q_len, max(0, kv_len - q_len)))
    out = np.ones(2, dtype=np.int32)
    _policy_lib().ypol_kv_splits(q_lens.ctypes.data, before.ctypes.data, portions, 128 // per, max(1, 2 * sms // g), 0, PREFILL_SPLIT_MIN_TILES,
                                 PREFILL_SPLIT_START_UP, PREFILL_SPLIT_UNSHARED, PREFILL_SPLIT_GAIN, out.ctypes.data)
    return int(out[0]), int(out[1])


def _attend_unpacked(name, device, rows, held, at, n, max_q_len, max_kv_len, num_heads, scale, window, skip_single, lse2, weight_sums, flag, raw):
    """Portions of prompts: what they see is unpacked, as many requests at a time as ``UNPACK_BYTES`` hold, into pools of the call
    for the prompt kernel on the tcgen05 tensor cores (every value is a bfloat16 number, so nothing is rounded)."""
    g, dim = held[5:]
    positions, q_start, table, table_width, r = at
    width, per, sms = max(1, -(-max_kv_len // UNPACK_PAGE)), num_heads // g, sm_count(device)
    size = width * g * UNPACK_PAGE * dim                # of a request's keys, or values
    group = max(1, min(r, UNPACK_BYTES // (4 * size)))
    splits, share = (1, 1) if window else _portion_splits(max(1, min(r, n // max_q_len)), max_q_len, max_kv_len, per, g, sms)
    items = -(-max_kv_len // 128) * group * g if lse2 is not None else 0                # sums: 128 keys of a KV head each
    tiles = -(-max_q_len // (128 // per))               # tiles of rows that see an item, at most; about half of them on average
    each = max(16, items * tiles // (8 * sms))
    parts = -(-tiles // each)
    # pools; shares of outputs and of sums, counters (two of the prompt kernel's, one and four an item of the sums'), block table, marks of
    # keys and whether there are any
    floats = n * num_heads * splits * (dim + 2) if splits > 1 else 0
    pools = torch.empty(2 * group * size, dtype=torch.bfloat16, device=device)
    n_counters = (3 + 4 * items + 3) // 4 * 4
    pages = group * width
    work = torch.empty(floats + items * parts * 384 + n_counters + pages * (1 + g * 2048 // dim) + 1, dtype=torch.int32, device=device)
    k_at, scratch = pools.data_ptr(), work.data_ptr()
    v_at, partial = k_at + 2 * group * size, scratch + 4 * floats
    counters = partial + 4 * items * parts * 384
    table_at = counters + 4 * n_counters
    marks_at = table_at + 4 * pages
    some_marked_at, marked_by = marks_at + pages * g * 8192 // dim, next(_unpackings) & 0x7FFFFFFF
    for first in range(0, r, group):
        m = min(group, r - first)
        starts, row = q_start + 4 * first, table + 4 * first * table_width
        check(_entry("yalis_packed_unpack", "pppiiii" + "pppii" + "iii" + "ppppip" + "pipp")(
            *held, positions, starts, row, table_width, m, width, window, skip_single, k_at, v_at, marks_at, some_marked_at, marked_by, table_at,
            counters, 3 + 4 * items, flag, raw), name)
        check(_entry("yalis_prefill_attention_tcgen05_unpacked", "plpl" + "ppppi" + "pppiii" + "iiiiii" + "fiiiippppp")(
            *rows, k_at, v_at, marks_at, some_marked_at, marked_by, positions, starts, table_at, width, UNPACK_PAGE, m * width, n, m, max_q_len,
            num_heads, g, dim, scale, window, splits, share, skip_single, _address(lse2), scratch, counters, flag, raw), name)
        if lse2 is not None:
            check(_entry("yalis_packed_sums_tcgen05", "plpiiiii" + "pppiiiiifii" + "ppiipppp")(
                *rows[:2], k_at, width, held[3], held[4], g, dim, positions, starts, row, table_width, m, n, max_kv_len, num_heads, scale, window,
                skip_single, lse2.data_ptr(), weight_sums.data_ptr(), each, parts, partial, counters + 8, flag, raw), name)


def packed_attention(q: torch.Tensor, pages: PackedPages, positions: torch.Tensor, q_start: torch.Tensor, block_table: torch.Tensor,
                     max_q_len: int, num_heads: int, scale: Optional[float] = None, window: Optional[int] = None,
                     max_kv_len: Optional[int] = None, weight_sums: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                     error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a step's tokens over the packed cache of their requests: single tokens, portions of prompts and both together.

    ``q`` is [N, >= heads * head_dim] (the fused qkv matrix will do) in float32 or bfloat16; ``q_start`` int32 [R + 1] gives each
    request's rows, which stand at consecutive places of its cache; row n sees the places
    positions[n] - window < j <= positions[n] (all up to it without ``window``).  Place and position are one thing only as long as
    nothing was evicted: after ``evict_tokens`` a row sees by its place and was rotated by its position.  ``max_q_len`` bounds the
    rows of a request, ``max_kv_len`` the places seen (the block table's width bounds them otherwise).  ``weight_sums`` float32
    [pages, kv_heads, page_size]: the softmax weight that a token received, summed over the step's rows and the heads of the KV
    head, is added to it (pages of different requests must differ then).  It is never reset: a place that is written anew (in a page
    taken again, behind a cut) has the sum of the token that stood there until the caller sets it to zero.

    The result is [N, heads * head_dim] in q's dtype (``out`` may be a column block of a wider matrix); rows that see nothing are
    zeros, rows of no request stay as they are.  Places without a page are left out, as if the row did not see them, and raise the
    error word's bit.  A row that sees a key or a value without numbers is NaN; the weights' sums go by the keys alone.

    Scores, exponentials, normalisers and sums are float32, and with float32 queries so is every product.  With bfloat16 queries a weight
    is rounded where it meets the value: times the value's step to float16's eleven bits, relative to the row's largest such product,
    where codes are multiplied as they are (there, of a query what lies below 2^-28 of its row's largest is lost, and one of 2^119 or
    more gives NaN); to bfloat16 in portions whose rows are unpacked, or with a window to two bfloat16 parts."""
    name = "packed_attention"
    device = _need_here(name, q, pages.k, pages.v, pages.words, positions, q_start, block_table, weight_sums, out, error_flag)
    held = _pages_arguments(name, pages)
    page_size, g, dim = held[4:]
    dtype, width = q.dtype, num_heads * dim
    code = dtype_code(dtype)
    if num_heads < 1 or num_heads % g:
        raise KernelError(f"{name}: heads must be a multiple of kv_heads")
    if q.dim() != 2 or q.shape[1] < width:
        raise KernelError(f"{name}: q must be [N, >= heads*head_dim] with unit inner stride")
    n, (step, unit) = q.shape[0], q.stride()
    if unit != 1:
        raise KernelError(f"{name}: q must be [N, >= heads*head_dim] with unit inner stride")
    rows, columns = _check_index(name, n, block_table, positions)
    if q_start.dtype is not torch.int32 or q_start.dim() != 1 or not q_start.is_contiguous() or not 1 <= q_start.shape[0] <= rows + 1:
        raise KernelError(f"{name}: q_start must be int32 [R+1], and block_table have a row for every request")
    if max_q_len < 0 or (max_kv_len is not None and max_kv_len < 0) or (window is not None and window <= 0):
        raise KernelError(f"{name}: max_q_len and max_kv_len must not be negative, and the window must be positive")
    max_q_len = min(max_q_len, n)                       # (any bound will do)
    if scale is None:
        scale = dim ** -0.5
    elif not math.isfinite(scale):
        raise KernelError(f"{name}: the scale must be finite")
    r, reach, flag = q_start.shape[0] - 1, min(columns * page_size, _LONGEST), _flag_address(name, error_flag)
    if window is None or window >= reach:
        window = 0                                      # (every place that the table has)
    max_kv_len = reach if max_kv_len is None or max_kv_len > reach else int(max_kv_len)
    lse2 = scores = None
    if weight_sums is not None:
        need(weight_sums.dtype == torch.float32 and weight_sums.shape == pages.k.shape[:3] and weight_sums.is_contiguous(), name,
             "weight_sums must be contiguous float32 [pages, kv_heads, page_size]")
        lse2 = torch.empty((n, num_heads), dtype=torch.float32, device=device)
    if out is None:
        out = torch.empty_like(q) if step == width else torch.empty((n, width), dtype=dtype, device=device)
    elif out.shape != (n, width) or out.dtype is not dtype or out.stride(1) != 1:
        raise KernelError(f"{name}: bad out tensor")
    per, q_at, out_at, out_step, raw = num_heads // g, q.data_ptr(), out.data_ptr(), out.stride(0), _raw_stream(device)
    at = (positions.data_ptr(), q_start.data_ptr(), block_table.data_ptr(), columns, r)
    aligned = (q_at | step * (4 if code == F32 else 2)) % 16 == 0
    mma = (dim == 64 or dim == 128) and r <= 4096
    unpack = (code == BF16 and (dim == 64 or dim == 128) and per <= 128 and scale > 0 and aligned and (out_at | out_step * 2) % 16 == 0
              and _unpacking_pays(max_q_len * per, r * g * max_kv_len))
    # Single tokens beside the portions get a kernel of their own where there may be any: with one, the others have all rows but it.
    single = unpack and mma and max_q_len < n <= (r - 1) * max_q_len + 1
    if unpack:
        _attend_unpacked(name, device, (q_at, step, out_at, out_step), held, at, n, max_q_len, max_kv_len, num_heads, scale, window, single, lse2,
                         weight_sums, flag, raw)
    if mma and (single or not unpack):
        q_rows = per if single else max_q_len * per
        tile = 8 if code == F32 or q_rows <= 8 else 16
        n_scores = (r if single else n) * num_heads * max_kv_len               # (of the rows that this launch takes)
        if lse2 is not None and q_rows <= 16 and 4 * n_scores <= SCORE_BYTES:
            scores = torch.empty(n_scores, dtype=torch.float32, device=device)
        blocks, floats = _mma_launch(device, code, dim, tile)
        counters, scratch = _workspace(device, raw, blocks, floats)
        check(_entry("yalis_packed_attention_mma", "plipl" + "pppiiii" + "pppii" + "iiiifippliipppp")(
            q_at, step, code, out_at, out_step, *held, *at, num_heads, tile, aligned, single, scale, window, _address(lse2), _address(scores),
            max_kv_len, q_rows, blocks, scratch.data_ptr(), counters.data_ptr(), flag, raw), name)
    elif not unpack:
        check(_entry("yalis_packed_attention_general", "plipl" + "pppiiii" + "pppii" + "iifippp")(
            q_at, step, code, out_at, out_step, *held, *at, n, num_heads, scale, window, _address(lse2), flag, raw), name)
    if lse2 is None or (unpack and not single):
        return out
    to = (lse2.data_ptr(), weight_sums.data_ptr(), raw)
    if scores is not None:
        check(_entry("yalis_packed_sums_of_scores", "pliiii" + "pppii" + "iiiippp")(
            scores.data_ptr(), max_kv_len, *held[3:], *at, max_kv_len, num_heads, window, single, *to), name)
    elif mma:
        check(_entry("yalis_packed_weight_sums", "pli" + "pppiiii" + "pppii" + "iifiiippp")(
            q_at, step, code, *held, *at, max_kv_len, num_heads, scale, window, aligned, single, *to), name)
    else:
        check(_entry("yalis_packed_weight_sums_general", "pli" + "pppiiii" + "pppii" + "iifippp")(
            q_at, step, code, *held, *at, max_kv_len, num_heads, scale, window, *to), name)
    return out


def evict_tokens(pools: Sequence[torch.Tensor], weight_sums: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor, keep: int,
                 recent: int = 0, error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cut the caches of R requests to ``keep`` tokens, in place, for every KV head by itself.

    Of a request of ``lengths[r]`` tokens (int32 [R], row r of the block table) that holds more than ``keep``, every KV head keeps
    the last ``recent`` and, of the others, the keep - recent with the largest ``weight_sums`` (float32
    [pages, kv_heads, page_size]; of equal ones the earlier, NaN last).  They move, in their order, to the places 0 .. keep - 1 of
    the request's pages, in every tensor of ``pools`` (up to four, or none, [pages, kv_heads, page_size, ...]: ``PackedPages.pools()``,
    or the pools of keys and values of a plain cache) and in ``weight_sums``; what lies behind them stays as it was, and the pages
    there may be given back.  That holds for the sums as well: before the weights of tokens behind the cut are counted, the caller sets
    the sums of their places to zero (``weight_sums[block_table[r, place // page_size], :, place % page_size] = 0``), or they start
    with those of the tokens that stood there.  Requests of at most ``keep`` tokens, and requests with a token without a page (which
    raise the error word's bit), stay as they are.  The pages of the requests must differ.  Returns int32 [R, kv_heads, keep]: the
    place that each token had, ascending, -1 where there is none."""
    name = "evict_tokens"
    pools = tuple(pools)
    device = _need_here(name, *pools, weight_sums, lengths, block_table, error_flag)
    if len(pools) > 4:
        raise KernelError(f"{name}: at most four pools")
    if not (weight_sums.dtype is torch.float32 and weight_sums.dim() == 3 and weight_sums.is_contiguous()):
        raise KernelError(f"{name}: weight_sums must be contiguous float32 [pages, kv_heads, page_size]")
    shape, rows = weight_sums.shape, max(1, weight_sums.numel())
    pages, g, page_size = shape
    addresses, row_bytes = _Addresses(), _Sizes()
    for i, p in enumerate(pools):
        if p.dim() < 3 or p.shape[:3] != shape or not p.is_contiguous():
            raise KernelError(f"{name}: pools must be contiguous [pages, kv_heads, page_size, ...]")
        addresses[i], row_bytes[i] = at, size = p.data_ptr(), p.numel() // rows * p.element_size()
        if (at | size) % 2:
            raise KernelError(f"{name}: rows of a pool must be whole pairs of bytes")
    if not (lengths.dtype is torch.int32 and lengths.dim() == 1 and lengths.is_contiguous()):
        raise KernelError(f"{name}: lengths must be int32 [R]")
    r, flag = lengths.shape[0], _flag_address(name, error_flag)
    table_rows, columns = _check_index(name, 0, block_table)
    if table_rows < r:
        raise KernelError(f"{name}: block_table has fewer rows than requests")
    if keep < 1 or not 0 <= recent <= keep:
        raise KernelError(f"{name}: keep must be at least 1 and recent between 0 and keep")
    kept = torch.empty(r, g, keep, dtype=torch.int32, device=device)
    check(_entry("yalis_evict_tokens", "ppippp" + "iiiiiii" + "ppp")(
        ctypes.addressof(addresses), ctypes.addressof(row_bytes), len(pools), weight_sums.data_ptr(), lengths.data_ptr(), block_table.data_ptr(), columns, page_size, pages, g, r, keep,
        recent, kept.data_ptr(), flag, _raw_stream(device)), name)
    return kept


_Addresses, _Sizes = ctypes.c_void_p * 4, ctypes.c_int * 4
