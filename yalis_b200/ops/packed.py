"""A paged cache held in 4 bits: rows written and read, attention over it, and eviction by accumulated weights.

The format (``csrc/packed.cuh``): a row of one token and KV head is one 4-bit code per element and a 16-bit word with the row's
step and zero, value = (code - zero) * step; every value is a bfloat16 number.  A token takes ``head_dim / 2 + 2`` bytes for its
key and as many for its value, per KV head.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from ._lib import BF16, F32, KernelError, check, dtype_code, lib, need, stream
from .attention import (PREFILL_SPLIT_GAIN, PREFILL_SPLIT_MIN_TILES, PREFILL_SPLIT_START_UP, PREFILL_SPLIT_UNSHARED, _policy_lib,
                        sm_count)

_TYPES = {"p": ctypes.c_void_p, "i": ctypes.c_int, "l": ctypes.c_longlong, "f": ctypes.c_float}
_entries = {}


def _entry(name: str, signature: str, result=ctypes.c_int):
    """The library's function with its argument types set once: plain numbers are handed over as they are (these calls are made
    for every layer of a step, and converting thirty arguments one by one takes longer than the smaller kernels run)."""
    fn = _entries.get(name)
    if fn is None:
        fn = getattr(lib(), name)
        fn.argtypes, fn.restype = [_TYPES[c] for c in signature], result
        _entries[name] = fn
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


def _need_here(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Every tensor on the current device, whose stream the kernels are launched on."""
    here = -1
    for t in tensors:
        if t is not None:
            at = t.get_device()
            if at < 0:
                raise KernelError(f"{name}: every tensor must be on the GPU (there is no CPU path)")
            if at != here and (here >= 0 or at != torch.cuda.current_device()):
                raise KernelError(f"{name}: every tensor must be on the current device")
            here = at


def _address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _pages_arguments(name: str, pages: PackedPages):
    k, v, words = pages.k, pages.v, pages.words
    shape = k.shape
    if not (k.dtype is torch.uint8 and v.dtype is torch.uint8 and len(shape) == 4 and v.shape == shape and k.is_contiguous() and v.is_contiguous()):
        raise KernelError(f"{name}: codes must be contiguous uint8 [pages, kv_heads, page_size, head_dim / 2]")
    num_pages, g, page_size, half = shape
    if not (words.dtype is torch.int16 and words.shape == (num_pages, g, page_size, 2) and words.is_contiguous()):
        raise KernelError(f"{name}: words must be contiguous int16 [pages, kv_heads, page_size, 2]")
    if half % 4 or not 4 <= half <= 128:
        raise KernelError(f"{name}: head_dim {2 * half} must be a multiple of 8 up to 256")
    if num_pages * g * page_size >= 1 << 31:
        raise KernelError(f"{name}: {num_pages} pages of {g} x {page_size} rows are 2^31 rows or more")
    at = (k.data_ptr(), v.data_ptr(), words.data_ptr())
    if (at[0] | at[1] | at[2]) % 16:
        raise KernelError(f"{name}: pools must start on 16-byte boundaries")
    return at + (num_pages, page_size, g, 2 * half)


def _check_index(name: str, n: int, block_table: torch.Tensor, *per_token: torch.Tensor) -> None:
    for t in per_token:
        if not (t.dtype is torch.int32 and t.shape == (n,) and t.is_contiguous()):
            raise KernelError(f"{name}: positions/req_of_token: int32 [N]")
    if not (block_table.dtype is torch.int32 and block_table.dim() == 2 and block_table.is_contiguous()):
        raise KernelError(f"{name}: block_table must be contiguous int32 [R, width]")


def _check_flag(name: str, error_flag: Optional[torch.Tensor]) -> None:
    need(error_flag is None or (error_flag.dtype == torch.int32 and error_flag.numel() >= 1), name, "the error word must be int32")


_counters_of_stream = {}


def _counters(n: int, device: torch.device) -> torch.Tensor:
    """Zeroed int32 counters, which every launch leaves at zero: one buffer per stream, whose launches run one after the other; a
    recording, which may be replayed on any stream, gets its own with every launch."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(n, dtype=torch.int32, device=device)
    key = (device.index, stream().value)
    held = _counters_of_stream.get(key)
    if held is None or held.numel() < n:
        held = _counters_of_stream[key] = torch.zeros(max(n, 2048), dtype=torch.int32, device=device)
    return held


_mma_launches = {}


def _mma_launch(device: torch.device, code: int, dim: int, columns: int) -> Tuple[int, int]:
    """(blocks, floats of scratch memory) of the tensor-core kernel."""
    key = (device.index, code, dim, columns)
    found = _mma_launches.get(key)
    if found is None:
        blocks = _entry("yalis_packed_attention_mma_blocks", "iii")(code, dim, columns)
        floats = _entry("yalis_packed_attention_mma_scratch_floats", "iii", ctypes.c_longlong)(blocks, dim, columns)
        found = _mma_launches[key] = (blocks, floats)
    return found


def packed_kv_write(k: torch.Tensor, v: torch.Tensor, pages: PackedPages, positions: torch.Tensor, req_of_token: torch.Tensor,
                    block_table: torch.Tensor, error_flag: Optional[torch.Tensor] = None) -> None:
    """Store the keys and values of a step's tokens, [N, kv_heads * head_dim] in float32 or bfloat16 (column blocks of wider
    matrices are taken), in 4 bits: token n goes to place ``positions[n]`` of the request whose block-table row is
    ``req_of_token[n]`` (-1: nowhere).  No two tokens may share a place.  A token without a page is left out and raises the error
    word's bit.  Rows with a NaN, an infinity or a magnitude above 2^120 read back as NaN throughout."""
    name = "packed_kv_write"
    _need_here(name, k, v, pages.k, pages.v, pages.words, positions, req_of_token, block_table, error_flag)
    held, shape = _pages_arguments(name, pages), k.shape
    if not (k.dtype is v.dtype and len(shape) == 2 and v.shape == shape and shape[1] == held[5] * held[6] and k.stride(1) == v.stride(1) == 1):
        raise KernelError(f"{name}: k and v must be [N, kv_heads * head_dim] of one dtype with unit inner stride")
    _check_index(name, shape[0], block_table, positions, req_of_token)
    _check_flag(name, error_flag)
    code, k_at, v_at, k_step, v_step, size = dtype_code(k.dtype), k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), k.element_size()
    vector = (k_at | v_at | k_step * size | v_step * size) % 16 == 0
    check(_rows_entry()(1, k_at, v_at, k_step, v_step, code, *held, positions.data_ptr(), req_of_token.data_ptr(), block_table.data_ptr(),
                        block_table.shape[1], shape[0], vector, _address(error_flag), stream()), name)


def _rows_entry():
    return _entry("yalis_packed_rows", "ippllipppiiiipppiiipp")


def packed_kv_read(pages: PackedPages, positions: torch.Tensor, req_of_token: torch.Tensor, block_table: torch.Tensor,
                   dtype: torch.dtype = torch.bfloat16, error_flag: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values, each [N, kv_heads * head_dim] in ``dtype``, of the tokens at ``positions`` of the requests
    ``req_of_token``: what ``packed_kv_write`` left there, exactly.  Tokens of no request (-1) and tokens without a page (which
    raise the error word's bit) read as zeros."""
    name = "packed_kv_read"
    _need_here(name, pages.k, pages.v, pages.words, positions, req_of_token, block_table, error_flag)
    held, n, code = _pages_arguments(name, pages), positions.shape[0], dtype_code(dtype)
    _check_index(name, n, block_table, positions, req_of_token)
    _check_flag(name, error_flag)
    width = held[5] * held[6]
    k, v = torch.empty((n, width), dtype=dtype, device=positions.device), torch.empty((n, width), dtype=dtype, device=positions.device)
    check(_rows_entry()(0, k.data_ptr(), v.data_ptr(), width, width, code, *held, positions.data_ptr(), req_of_token.data_ptr(),
                        block_table.data_ptr(), block_table.shape[1], n, True, _address(error_flag), stream()), name)
    return k, v


UNPACK_ROWS = 64          # query rows of a pair (tokens * heads of a KV head) beyond which portions are unpacked for the prompt kernel
UNPACK_PAGE = 64          # keys of a page of the unpacked pools
UNPACK_BYTES = 2 << 30    # of unpacked keys and values at a time
SCORE_BYTES = 1 << 30     # of scores that a step of few rows may leave for its sums; beyond, the products are taken once more


@functools.lru_cache(maxsize=4096)
def _portion_splits(portions: int, q_len: int, kv_len: int, per: int, g: int, sms: int) -> Tuple[int, int]:
    """(shares of a tile's keys, tiles of keys of a share) for the prompt kernel, as the plain cache's steps choose them
    (``prefill_kv_splits``), for ``portions`` portions of ``q_len`` tokens that end at place ``kv_len``."""
    q_lens, before = (np.full(portions, v, dtype=np.int32) for v in (q_len, max(0, kv_len - q_len)))
    out = np.ones(2, dtype=np.int32)
    _policy_lib().ypol_kv_splits(q_lens.ctypes.data, before.ctypes.data, portions, 128 // per, max(1, 2 * sms // g), 0, PREFILL_SPLIT_MIN_TILES,
                                 PREFILL_SPLIT_START_UP, PREFILL_SPLIT_UNSHARED, PREFILL_SPLIT_GAIN, out.ctypes.data)
    return int(out[0]), int(out[1])


def _attend_unpacked(name, q, out, held, at, steps, n, max_q_len, max_kv_len, num_heads, scale, window, skip_single, lse2,
                     weight_sums, error_flag, raw):
    """Portions of prompts: the rows that they see are unpacked, as many requests at a time as ``UNPACK_BYTES`` hold, into pools of
    the call for the prompt kernel on the tcgen05 tensor cores (every value is a bfloat16 number, so nothing is rounded)."""
    g, dim = held[5:]
    positions, q_start, table, table_width, r = at
    width = max(1, -(-max_kv_len // UNPACK_PAGE))
    rows = width * g * UNPACK_PAGE * dim                # of a request, keys or values
    group = max(1, min(r, UNPACK_BYTES // (4 * rows)))
    per = num_heads // g
    splits, share = (1, 1) if window else _portion_splits(max(1, min(r, n // max(1, max_q_len))), max_q_len, max_kv_len, per, g, sm_count(q.device))
    need_floats = n * num_heads * splits * (dim + 2) if splits > 1 else 0
    pools = torch.empty(2 * group * rows, dtype=torch.bfloat16, device=q.device)
    items = -(-max_kv_len // 128) * group * g if weight_sums is not None else 0         # 128 keys of a KV head each
    tiles_seen = -(-max_q_len // (128 // per))          # tiles of rows that see an item, at most; about half of them on average
    each = max(16, items * tiles_seen // (8 * sm_count(q.device)))
    parts = -(-tiles_seen // each)
    work = torch.empty(group * width + 3 + 4 * items, dtype=torch.int32, device=q.device)   # counters (two of the prompt kernel's), block table
    partial = torch.empty(items * parts * 3 * 128, dtype=torch.float32, device=q.device) if items else None
    scratch = torch.empty(need_floats, dtype=torch.float32, device=q.device) if need_floats else None
    k_at, table_at = pools.data_ptr(), work.data_ptr() + 4 * (3 + 4 * items)
    v_at = k_at + 2 * group * rows
    for first in range(0, r, group):
        m = min(group, r - first)
        starts, row = q_start + 4 * first, table + 4 * first * table_width
        check(_entry("yalis_packed_unpack", "pppiiii" + "pppii" + "iii" + "ppppipp")(
            *held, positions, starts, row, table_width, m, width, window, skip_single, k_at, v_at, table_at, work.data_ptr(),
            3 + 4 * items, _address(error_flag), raw), name)
        check(_entry("yalis_prefill_attention_tcgen05_unpacked", "plplpp" + "pppiii" + "iiiiii" + "fiiiippppp")(
            q.data_ptr(), steps[0], out.data_ptr(), steps[1], k_at, v_at, positions, starts, table_at, width, UNPACK_PAGE, m * width, n, m,
            max_q_len, num_heads, g, dim, scale, window, splits, share, skip_single, _address(lse2), _address(scratch), work.data_ptr(),
            _address(error_flag), raw), name)
        if weight_sums is not None:
            check(_entry("yalis_packed_sums_tcgen05", "plpiiiii" + "pppiiiiifii" + "ppiipppp")(
                q.data_ptr(), steps[0], k_at, width, held[3], held[4], g, dim, positions, starts, row, table_width, m, n, max_kv_len, num_heads, scale,
                window, skip_single, lse2.data_ptr(), weight_sums.data_ptr(), each, parts, _address(partial), work.data_ptr() + 8, _address(error_flag), raw), name)


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
    head, is added to it (pages of different requests must differ then).  The result is [N, heads * head_dim] in q's dtype
    (``out`` may be a column block of a wider matrix); rows that see nothing are zeros, rows of no request stay as they are.
    Scores, weights and sums are float32, and with float32 queries so is every product."""
    name = "packed_attention"
    _need_here(name, q, pages.k, pages.v, pages.words, positions, q_start, block_table, weight_sums, out, error_flag)
    held = _pages_arguments(name, pages)
    page_size, g, dim = held[4:]
    code, n, r, width = dtype_code(q.dtype), q.shape[0], q_start.shape[0] - 1 if q_start.dim() == 1 else -1, num_heads * dim
    if num_heads < 1 or num_heads % g:
        raise KernelError(f"{name}: heads must be a multiple of kv_heads")
    if q.dim() != 2 or q.stride(1) != 1 or q.shape[1] < width:
        raise KernelError(f"{name}: q must be [N, >= heads*head_dim] with unit inner stride")
    _check_index(name, n, block_table, positions)
    if q_start.dtype is not torch.int32 or r < 0 or not q_start.is_contiguous():
        raise KernelError(f"{name}: q_start must be int32 [R+1]")
    need(block_table.shape[0] >= r, name, "block_table has fewer rows than requests")
    need(max_q_len >= 0 and (window is None or window > 0), name, "max_q_len and the window must be positive")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    need(math.isfinite(scale), name, "the scale must be finite")
    reach = block_table.shape[1] * page_size
    max_kv_len = reach if max_kv_len is None else min(int(max_kv_len), reach)
    if weight_sums is not None:
        need(weight_sums.dtype == torch.float32 and weight_sums.shape == pages.k.shape[:3] and weight_sums.is_contiguous(), name,
             "weight_sums must be contiguous float32 [pages, kv_heads, page_size]")
    _check_flag(name, error_flag)
    if out is None:
        out = torch.empty((n, width), dtype=q.dtype, device=q.device)
    need(out.shape == (n, width) and out.dtype is q.dtype and out.stride(1) == 1, name, "bad out tensor")
    lse2 = torch.empty((n, num_heads), dtype=torch.float32, device=q.device) if weight_sums is not None else None
    at, steps, raw = (positions.data_ptr(), q_start.data_ptr(), block_table.data_ptr(), block_table.shape[1], r), (q.stride(0), out.stride(0)), stream()
    per, aligned = num_heads // g, (q.data_ptr() | steps[0] * q.element_size()) % 16 == 0
    unpack = (code == BF16 and dim in (64, 128) and max_q_len * per > UNPACK_ROWS and per <= 128 and scale > 0 and aligned
              and (out.data_ptr() | steps[1] * 2) % 16 == 0)
    mma, scores = dim in (64, 128) and r <= 4096, None
    single = unpack and mma and n > max_q_len          # single tokens may stand beside the portions: a kernel of their own
    if unpack:
        _attend_unpacked(name, q, out, held, at, steps, n, max_q_len, max_kv_len, num_heads, scale, window or 0, single, lse2, weight_sums,
                         error_flag, raw)
    if mma and (single or not unpack):
        rows = (1 if single else max_q_len) * per
        columns = 8 if code == F32 or rows <= 8 else 16
        if weight_sums is not None and rows <= 16 and 4 * n * num_heads * max_kv_len <= SCORE_BYTES:
            scores = torch.empty(n * num_heads * max_kv_len, dtype=torch.float32, device=q.device)
        blocks, floats = _mma_launch(q.device, code, dim, columns)
        scratch = torch.empty(floats, dtype=torch.float32, device=q.device)
        check(_entry("yalis_packed_attention_mma", "plipl" + "pppiiii" + "pppii" + "iiiifipplipppp")(
            q.data_ptr(), steps[0], code, out.data_ptr(), steps[1], *held, *at, num_heads, columns, aligned, single, scale, window or 0,
            _address(lse2), _address(scores), max_kv_len, blocks, scratch.data_ptr(), _counters(blocks, q.device).data_ptr(), _address(error_flag), raw), name)
    if not mma and not unpack:
        check(_entry("yalis_packed_attention_general", "plipl" + "pppiiii" + "pppii" + "iifippp")(
            q.data_ptr(), steps[0], code, out.data_ptr(), steps[1], *held, *at, n, num_heads, scale, window or 0, _address(lse2),
            _address(error_flag), raw), name)
    if weight_sums is None or (unpack and not single):
        return out
    if scores is not None:
        check(_entry("yalis_packed_sums_of_scores", "pliiii" + "pppii" + "iiiippp")(
            scores.data_ptr(), max_kv_len, *held[3:], *at, max_kv_len, num_heads, window or 0, single, lse2.data_ptr(), weight_sums.data_ptr(), raw), name)
    elif mma:
        check(_entry("yalis_packed_weight_sums", "pli" + "pppiiii" + "pppii" + "iifiiippp")(
            q.data_ptr(), steps[0], code, *held, *at, max_kv_len, num_heads, scale, window or 0, aligned, single, lse2.data_ptr(),
            weight_sums.data_ptr(), raw), name)
    else:
        check(_entry("yalis_packed_weight_sums_general", "pli" + "pppiiii" + "pppii" + "iifippp")(
            q.data_ptr(), steps[0], code, *held, *at, max_kv_len, num_heads, scale, window or 0, lse2.data_ptr(), weight_sums.data_ptr(), raw), name)
    return out


def evict_tokens(pools: Sequence[torch.Tensor], weight_sums: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor, keep: int,
                 recent: int = 0, error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cut the caches of R requests to ``keep`` tokens, in place, for every KV head by itself.

    Of a request of ``lengths[r]`` tokens (int32 [R], row r of the block table) that holds more than ``keep``, every KV head keeps
    the last ``recent`` and, of the others, the keep - recent with the largest ``weight_sums`` (float32
    [pages, kv_heads, page_size]; of equal ones the earlier, NaN last).  They move, in their order, to the places 0 .. keep - 1 of
    the request's pages, in every tensor of ``pools`` (up to four, [pages, kv_heads, page_size, ...]: ``PackedPages.pools()``, or
    the pools of keys and values of a plain cache) and in ``weight_sums``; what lies behind them stays as it was, and the pages
    there may be given back.  Requests of at most ``keep`` tokens, and requests with a token without a page (which raise the error
    word's bit), stay as they are.  The pages of the requests must differ.  Returns int32 [R, kv_heads, keep]: the place that each
    token had, ascending, -1 where there is none."""
    name = "evict_tokens"
    pools = tuple(pools)
    _need_here(name, *pools, weight_sums, lengths, block_table, error_flag)
    need(len(pools) <= 4, name, "at most four pools")
    need(weight_sums.dtype == torch.float32 and weight_sums.dim() == 3 and weight_sums.is_contiguous(), name,
         "weight_sums must be contiguous float32 [pages, kv_heads, page_size]")
    pages, g, page_size = shape = weight_sums.shape
    addresses, row_bytes = (ctypes.c_void_p * 4)(), (ctypes.c_int * 4)()
    for i, p in enumerate(pools):
        need(p.dim() >= 3 and p.shape[:3] == shape and p.is_contiguous(), name, "pools must be contiguous [pages, kv_heads, page_size, ...]")
        addresses[i], row_bytes[i] = p.data_ptr(), p.numel() // max(1, pages * g * page_size) * p.element_size()
        need(row_bytes[i] % 2 == 0 and p.data_ptr() % 2 == 0, name, "rows of a pool must be whole pairs of bytes")
    need(lengths.dtype == torch.int32 and lengths.dim() == 1 and lengths.is_contiguous(), name, "lengths must be int32 [R]")
    r = lengths.shape[0]
    _check_index(name, 0, block_table)
    _check_flag(name, error_flag)
    need(block_table.shape[0] >= r, name, "block_table has fewer rows than requests")
    need(keep >= 1 and 0 <= recent <= keep, name, "keep must be at least 1 and recent between 0 and keep")
    kept = torch.empty((r, g, keep), dtype=torch.int32, device=lengths.device)
    check(_entry("yalis_evict_tokens", "ppippp" + "iiiiiii" + "ppp")(
        ctypes.addressof(addresses), ctypes.addressof(row_bytes), len(pools), weight_sums.data_ptr(), lengths.data_ptr(), block_table.data_ptr(),
        block_table.shape[1], page_size, pages, g, r, keep, recent, kept.data_ptr(), _address(error_flag), stream()), name)
    return kept
