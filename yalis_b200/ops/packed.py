"""A paged cache held in 4 bits: rows written and read, attention over it, and eviction by accumulated weights.

The format (``csrc/packed.cuh``): a row of one token and KV head is one 4-bit code per element and a 16-bit word with the row's
step and zero, value = (code - zero) * step; every value is a bfloat16 number.  A token takes ``head_dim / 2 + 2`` bytes for its
key and as many for its value, per KV head.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch

from ._lib import KernelError, check, dtype_code, f32, i32, i64, lib, need, need_cuda, ptr, stream


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
    need_cuda(name, *tensors)
    here = torch.cuda.current_device()
    need(all(t is None or t.device.index == here for t in tensors), name, "every tensor must be on the current device")


def _pages_arguments(name: str, pages: PackedPages):
    k, v, words = pages.pools()
    need(k.dtype == v.dtype == torch.uint8 and k.dim() == 4 and k.shape == v.shape and k.is_contiguous() and v.is_contiguous(), name,
         "codes must be contiguous uint8 [pages, kv_heads, page_size, head_dim / 2]")
    need(words.dtype == torch.int16 and words.shape == k.shape[:3] + (2,) and words.is_contiguous(), name,
         "words must be contiguous int16 [pages, kv_heads, page_size, 2]")
    need(pages.head_dim % 8 == 0 and 8 <= pages.head_dim <= 256, name, f"head_dim {pages.head_dim} must be a multiple of 8 up to 256")
    need(all(t.data_ptr() % 16 == 0 for t in (k, v, words)), name, "pools must start on 16-byte boundaries")
    return (ptr(k), ptr(v), ptr(words), i32(k.shape[0]), i32(k.shape[2]), i32(k.shape[1]), i32(pages.head_dim))


def _check_index(name: str, n: int, block_table: torch.Tensor, *per_token: torch.Tensor) -> None:
    for t in per_token:
        need(t.dtype == torch.int32 and t.shape == (n,) and t.is_contiguous(), name, "positions/req_of_token: int32 [N]")
    need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.is_contiguous(), name,
         "block_table must be contiguous int32 [R, width]")


def _check_flag(name: str, error_flag: Optional[torch.Tensor]) -> None:
    need(error_flag is None or (error_flag.dtype == torch.int32 and error_flag.numel() >= 1), name, "the error word must be int32")


def packed_kv_write(k: torch.Tensor, v: torch.Tensor, pages: PackedPages, positions: torch.Tensor, req_of_token: torch.Tensor,
                    block_table: torch.Tensor, error_flag: Optional[torch.Tensor] = None) -> None:
    """Store the keys and values of a step's tokens, [N, kv_heads * head_dim] in float32 or bfloat16 (column blocks of wider
    matrices are taken), in 4 bits: token n goes to place ``positions[n]`` of the request whose block-table row is
    ``req_of_token[n]`` (-1: nowhere).  No two tokens may share a place.  A token without a page is left out and raises the error
    word's bit.  Rows with a NaN, an infinity or a magnitude above 2^120 read back as NaN throughout."""
    name = "packed_kv_write"
    _need_here(name, k, v, pages.k, pages.v, pages.words, positions, req_of_token, block_table, error_flag)
    held, n, width = _pages_arguments(name, pages), k.shape[0], pages.num_kv_heads * pages.head_dim
    need(k.dtype == v.dtype and k.dim() == 2 and k.shape == v.shape == (n, width) and k.stride(1) == v.stride(1) == 1, name,
         "k and v must be [N, kv_heads * head_dim] of one dtype with unit inner stride")
    _check_index(name, n, block_table, positions, req_of_token)
    _check_flag(name, error_flag)
    code, size = dtype_code(k.dtype), 8 * k.element_size()
    vector = all(t.data_ptr() % min(size, 16) == 0 and (t.stride(0) * t.element_size()) % min(size, 16) == 0 for t in (k, v))
    check(lib().yalis_packed_rows(i32(1), ptr(k), ptr(v), i64(k.stride(0)), i64(v.stride(0)), i32(code), *held, ptr(positions),
                                  ptr(req_of_token), ptr(block_table), i32(block_table.shape[1]), i32(n), i32(int(vector)), ptr(error_flag),
                                  stream()), name)


def packed_kv_read(pages: PackedPages, positions: torch.Tensor, req_of_token: torch.Tensor, block_table: torch.Tensor,
                   dtype: torch.dtype = torch.bfloat16, error_flag: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values, each [N, kv_heads * head_dim] in ``dtype``, of the tokens at ``positions`` of the requests
    ``req_of_token``: what ``packed_kv_write`` left there, exactly.  Tokens of no request (-1) and tokens without a page (which
    raise the error word's bit) read as zeros."""
    name = "packed_kv_read"
    _need_here(name, pages.k, pages.v, pages.words, positions, req_of_token, block_table, error_flag)
    held, n, width, code = _pages_arguments(name, pages), positions.shape[0], pages.num_kv_heads * pages.head_dim, dtype_code(dtype)
    _check_index(name, n, block_table, positions, req_of_token)
    _check_flag(name, error_flag)
    k, v = (torch.empty((n, width), dtype=dtype, device=positions.device) for _ in range(2))
    check(lib().yalis_packed_rows(i32(0), ptr(k), ptr(v), i64(width), i64(width), i32(code), *held, ptr(positions), ptr(req_of_token),
                                  ptr(block_table), i32(block_table.shape[1]), i32(n), i32(1), ptr(error_flag), stream()), name)
    return k, v


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
    held, n, r, dim, g = _pages_arguments(name, pages), q.shape[0], q_start.numel() - 1, pages.head_dim, pages.num_kv_heads
    code = dtype_code(q.dtype)
    need(num_heads >= 1 and num_heads % g == 0, name, "heads must be a multiple of kv_heads")
    need(q.dim() == 2 and q.stride(1) == 1 and q.shape[1] >= num_heads * dim, name, "q must be [N, >= heads*head_dim] with unit inner stride")
    _check_index(name, n, block_table, positions)
    need(q_start.dtype == torch.int32 and q_start.dim() == 1 and q_start.is_contiguous() and r >= 0, name, "q_start must be int32 [R+1]")
    need(block_table.shape[0] >= r, name, "block_table has fewer rows than requests")
    need(max_q_len >= 0 and (window is None or window > 0), name, "max_q_len and the window must be positive")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    need(math.isfinite(scale), name, "the scale must be finite")
    reach = block_table.shape[1] * pages.page_size
    max_kv_len = reach if max_kv_len is None else min(int(max_kv_len), reach)
    need(weight_sums is None or (weight_sums.dtype == torch.float32 and weight_sums.shape == pages.k.shape[:3] and weight_sums.is_contiguous()),
         name, "weight_sums must be contiguous float32 [pages, kv_heads, page_size]")
    _check_flag(name, error_flag)
    if out is None:
        out = torch.empty((n, num_heads * dim), dtype=q.dtype, device=q.device)
    need(out.shape == (n, num_heads * dim) and out.dtype == q.dtype and out.stride(1) == 1, name, "bad out tensor")
    lse = torch.empty((n, num_heads), dtype=torch.float32, device=q.device) if weight_sums is not None else None
    check(lib().yalis_packed_attention_general(
        ptr(q), i64(q.stride(0)), i32(code), ptr(out), i64(out.stride(0)), *held, ptr(positions), ptr(q_start), ptr(block_table),
        i32(block_table.shape[1]), i32(r), i32(n), i32(max_kv_len), i32(num_heads), f32(scale), i32(window or 0), ptr(lse), ptr(weight_sums),
        ptr(error_flag), stream()), name)
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
    row_bytes = []
    for p in pools:
        need(p.dim() >= 3 and p.shape[:3] == weight_sums.shape and p.is_contiguous(), name, "pools must be contiguous [pages, kv_heads, page_size, ...]")
        row_bytes.append(p[0, 0, 0].numel() * p.element_size() if p.numel() else 0)
        need(row_bytes[-1] % 2 == 0 and p.data_ptr() % 2 == 0, name, "rows of a pool must be whole pairs of bytes")
    r = lengths.shape[0]
    need(lengths.dtype == torch.int32 and lengths.dim() == 1 and lengths.is_contiguous(), name, "lengths must be int32 [R]")
    _check_index(name, 0, block_table)
    _check_flag(name, error_flag)
    need(block_table.shape[0] >= r, name, "block_table has fewer rows than requests")
    need(keep >= 1 and 0 <= recent <= keep, name, "keep must be at least 1 and recent between 0 and keep")
    pages, g, page_size = weight_sums.shape
    kept = torch.empty((r, g, keep), dtype=torch.int32, device=lengths.device)
    check(lib().yalis_evict_tokens(
        (ctypes.c_void_p * 4)(*[p.data_ptr() for p in pools]), (ctypes.c_int * 4)(*row_bytes), i32(len(pools)), ptr(weight_sums), ptr(lengths),
        ptr(block_table), i32(block_table.shape[1]), i32(page_size), i32(pages), i32(g), i32(r), i32(keep), i32(recent), ptr(kept),
        ptr(error_flag), stream()), name)
    return kept
