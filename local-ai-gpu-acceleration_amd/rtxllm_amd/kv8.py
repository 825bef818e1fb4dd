"""The paged KV cache in 8 bits (include/rtxllm/kv8.h): new tokens quantised as they are
written, positions read back, attention over it.

As in rtxllm_amd.paged, torch supplies device memory and the current HIP stream of the
cache's device, every result is computed by build/librtxllm.so, int32 tensors hold
positions, starts and tables, and a call that is passed its outputs and workspace allocates
nothing and can be captured into a graph.
"""

from __future__ import annotations

import ctypes

import torch

from . import paged
from ._lib import PagedKV8Struct, lib
from .paged import PagedKV, _attn_rows, _call_rows, _type_of, _u32

FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}
CALLS = frozenset(("rtxllm_kv8_append", "rtxllm_kv8_read", "rtxllm_attn_kv8"))


class PagedKV8(PagedKV):
    """A layer's cache: codes k, v int8 or float8_e4m3fn [n_pages][n_kv_heads][page_size][head_dim], scales float32
    [n_pages][n_kv_heads][page_size / block], tails float16 [sequences][n_kv_heads][block][head_dim] and a block
    table, int32 [sequences][entries]."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 k_tail: torch.Tensor, v_tail: torch.Tensor, block_table: torch.Tensor):
        if k.dim() != 4 or k.dtype not in FORMATS or v.dtype != k.dtype or k.shape != v.shape:
            raise ValueError("k and v must be int8 or float8_e4m3fn [n_pages][n_kv_heads][page_size][head_dim] of one shape")
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or 0 in block_table.shape:
            raise ValueError("block_table must be int32 [sequences][entries]")
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        if 0 in k.shape or block_table.shape[1] * self.page_size > 1 << 24:
            raise ValueError(f"{block_table.shape[1]} entries of pages {tuple(k.shape)}: a sequence has 1..2^24 positions")
        self.sequences, self.one_sequence = block_table.shape[0], False
        if not (k.is_contiguous() and v.is_contiguous()) or block_table.stride(1) != 1:
            raise ValueError("the cache and the rows of its block table must be contiguous")
        if self.sequences > 1 and block_table.stride(0) < block_table.shape[1]:
            raise ValueError("the rows of the block table overlap")
        if not (k.is_cuda and k.device == v.device == block_table.device):
            raise ValueError("the cache and its block table must be on one GPU")
        self.device, self._index = k.device, k.get_device()
        self.block = k_tail.shape[2] if k_tail.dim() == 4 else 0
        if self.block not in (8, 16, 32, 64) or self.page_size % self.block:
            raise ValueError(f"tails {tuple(k_tail.shape)}: blocks of 8, 16, 32 or 64 positions that divide pages of {self.page_size}")
        scales = (self.n_pages, self.n_kv_heads, self.page_size // self.block)
        tails = (self.sequences, self.n_kv_heads, self.block, self.head_dim)
        parts = [self._check("k_scale", k_scale, scales), self._check("v_scale", v_scale, scales),
                 self._check("k_tail", k_tail, tails, torch.float16), self._check("v_tail", v_tail, tails, torch.float16)]
        self.capacity = block_table.shape[1] * self.page_size
        self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail = k, v, k_scale, v_scale, k_tail, v_tail
        self.block_table = block_table
        stride = max(block_table.stride(0), block_table.shape[1])
        self._struct = PagedKV8Struct(k.data_ptr(), v.data_ptr(), *parts, block_table.data_ptr(),
                                      _u32("the block table's row stride", stride), _u32("n_pages", self.n_pages),
                                      self.n_kv_heads, self.head_dim, self.page_size, self.capacity, self.block,
                                      FORMATS[k.dtype])
        self.ref = ctypes.addressof(self._struct)

    @classmethod
    def empty(cls, n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, block: int, block_table: torch.Tensor,
              dtype: torch.dtype = torch.int8) -> PagedKV8:
        """A cache with arrays of its own (all zero) for the sequences of a block table."""
        dev = block_table.device
        codes = [torch.zeros(n_pages, n_kv_heads, page_size, head_dim, dtype=dtype, device=dev) for _ in range(2)]
        scales = [torch.zeros(n_pages, n_kv_heads, page_size // block, device=dev) for _ in range(2)]
        tails = [torch.zeros(block_table.shape[0], n_kv_heads, block, head_dim, dtype=torch.float16, device=dev) for _ in range(2)]
        return cls(*codes, *scales, *tails, block_table)

    def _call(self, name: str, *args) -> None:
        if name not in CALLS:  # (of the functions of rtxllm_amd.paged, which take another struct)
            raise ValueError(f"{name}: takes fp16 pages, not a cache in 8 bits")
        super()._call(name, *args)


def _in_8_bits(cache: PagedKV) -> None:
    if not isinstance(cache, PagedKV8):
        raise ValueError(f"expected a PagedKV8, got a {type(cache).__name__}")


def _stride_of(name: str, cache: PagedKV8, x: torch.Tensor, rows: int, dtype: torch.dtype) -> int:
    """Stride in elements between the rows of x [rows][n_kv_heads][head_dim], which may lie apart."""
    shape, stride, width = x.shape, x.stride(), cache.n_kv_heads * cache.head_dim
    if (x.dtype is dtype and x.get_device() == cache._index and shape == (rows, cache.n_kv_heads, cache.head_dim) and
            stride[2] == 1 and (stride[1] == cache.head_dim or shape[1] == 1)):
        return stride[0] if rows > 1 else width
    raise ValueError(f"{name}: expected {dtype} [{rows}][{cache.n_kv_heads}][{cache.head_dim}] with contiguous rows on "
                     f"{cache.device}, got {x.dtype} {tuple(shape)} with strides {stride}")


def append(cache: PagedKV8, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, start: torch.Tensor | None = None) -> None:
    """New tokens enter the cache, k and v [rows][n_kv_heads][head_dim] of float32 or float16: sequence s has rows
    start[s] .. start[s + 1] - 1 (start None: row s), its positions pos[s], pos[s] + 1, ... Rows that are dropped again
    (drafts) are written over from within the newest block; if they had made a block whole, from its start, with the keys
    and values that the program has kept."""
    _in_8_bits(cache)
    rows, kind = k.shape[0], _type_of("k", k)
    ks, vs = _stride_of("k", cache, k, rows, k.dtype), _stride_of("v", cache, v, rows, k.dtype)
    sp, pp, sequences = _call_rows(cache, rows, pos, start)
    cache._call("rtxllm_kv8_append", k.data_ptr(), ks, v.data_ptr(), vs, kind, sp, pp, sequences, rows)


def read(cache: PagedKV8, pos: torch.Tensor, held: torch.Tensor, start: torch.Tensor | None = None, rows: int | None = None,
         dtype: torch.dtype = torch.float32, k_out: torch.Tensor | None = None,
         v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Positions pos[s], pos[s] + 1, ... of each sequence, which holds held[s], as rows of k and v
    [rows][n_kv_heads][head_dim] (rows as in append). Outputs that are not passed are of `rows` rows of dtype."""
    _in_8_bits(cache)
    given = k_out if k_out is not None else v_out
    if given is not None:
        rows, dtype = given.shape[0], given.dtype
    elif rows is None:
        if start is not None:
            raise ValueError("read: rows, or an output, says how many rows the starts are of")
        rows = pos.numel()
    if dtype not in paged.TYPES:
        raise ValueError(f"read: expected float32 or float16, got {dtype}")
    sp, pp, sequences = _call_rows(cache, rows, pos, start)
    shape = (rows, cache.n_kv_heads, cache.head_dim)
    hp = cache._check("held", held, (sequences,), torch.int32)
    k_out = cache._output("k_out", k_out, shape, dtype, fill=0.0)
    v_out = cache._output("v_out", v_out, shape, dtype, fill=0.0)
    cache._call("rtxllm_kv8_read", hp, sp, pp, sequences, rows, paged.TYPES[dtype], k_out.data_ptr(), v_out.data_ptr())
    return k_out, v_out


def attn_workspace(cache: PagedKV8, n_heads: int, sequences: int, rows: int, window: int | None = None,
                   sinks: int = 0) -> torch.Tensor:
    _in_8_bits(cache)
    near = cache.capacity if window is None else _u32("window", window)
    return cache._space(None, int(lib().rtxllm_attn_kv8_workspace(
        cache.ref, _u32("n_heads", n_heads), _u32("sequences", sequences), _u32("rows", rows), near, _u32("sinks", sinks))))


def attn(cache: PagedKV8, q: torch.Tensor, pos: torch.Tensor, start: torch.Tensor | None = None, *,
         window: int | None = None, sinks: int = 0, out: torch.Tensor | None = None,
         workspace: torch.Tensor | None = None) -> torch.Tensor:
    """rtxllm_amd.paged.attn_window over this cache, which holds the call's rows already."""
    _in_8_bits(cache)
    return _attn_rows(cache, ("rtxllm_attn_kv8_workspace", "rtxllm_attn_kv8"), q, pos, start, window, sinks, out, workspace)
