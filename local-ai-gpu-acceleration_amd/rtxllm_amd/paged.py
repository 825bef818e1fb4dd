"""Long contexts over the paged fp16 KV cache (include/rtxllm/paged_kv.h).

torch supplies device memory and the current HIP stream of the cache's device;
every result is computed by build/librtxllm.so. Shapes, types and devices are
checked on the host before any launch. Positions, slots, lengths and block
tables are int32 tensors (their bits are the C-ABI's uint32: -1 is
NO_POSITION, a padded row, which is neither read nor written). Outputs and
workspaces that are not passed are allocated; with all of them passed a call
allocates nothing and can be captured into a graph.
"""

from __future__ import annotations

import ctypes

import torch

from ._lib import PagedKVStruct, check, lib

NO_POSITION = -1
PAIRINGS = {"adjacent": 0, "halves": 1}
TYPES = {torch.float32: 0, torch.float16: 1}


def _u32(name: str, value: int) -> int:
    """The C-ABI's unsigned numbers, which ctypes would cut to their low 32 bits."""
    if 0 <= value <= 0xFFFFFFFF:
        return value
    raise ValueError(f"{name}: {value} is not in 0..2^32 - 1")


class PagedKV:
    """A layer's cache: k, v fp16 [n_pages][n_kv_heads][page_size][head_dim] and a
    block table, int32 [sequences][entries] or, for one sequence whose tokens the
    rows of a call are, [entries]."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor):
        if k.dim() != 4 or k.dtype != torch.float16 or v.dtype != torch.float16 or k.shape != v.shape:
            raise ValueError("k and v must be float16 [n_pages][n_kv_heads][page_size][head_dim] of one shape")
        if block_table.dim() not in (1, 2) or block_table.dtype != torch.int32 or block_table.shape[-1] == 0:
            raise ValueError("block_table must be int32 [sequences][entries] or [entries]")
        if 0 in k.shape or block_table.shape[-1] * k.shape[2] > 1 << 24:
            raise ValueError(f"{block_table.shape[-1]} entries of pages {tuple(k.shape)}: a sequence has 1..2^24 positions")
        if not (k.is_contiguous() and v.is_contiguous()) or block_table.stride(-1) != 1:
            raise ValueError("the cache and the rows of its block table must be contiguous")
        if not (k.is_cuda and k.device == v.device == block_table.device):
            raise ValueError("the cache and its block table must be on one GPU")
        self.k, self.v, self.block_table, self.device, self._index = k, v, block_table, k.device, k.get_device()
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.one_sequence = block_table.dim() == 1
        self.sequences = 1 if self.one_sequence else block_table.shape[0]
        self.capacity = block_table.shape[-1] * self.page_size
        stride = 0 if self.one_sequence else max(block_table.stride(0), block_table.shape[1])
        if not self.one_sequence and self.sequences > 1 and block_table.stride(0) < block_table.shape[1]:
            raise ValueError("the rows of the block table overlap")
        self._struct = PagedKVStruct(k.data_ptr(), v.data_ptr(), block_table.data_ptr(),
                                     _u32("the block table's row stride", stride), _u32("n_pages", self.n_pages),
                                     self.n_kv_heads, self.head_dim, self.page_size, self.capacity)
        self.ref = ctypes.addressof(self._struct)

    def _rows(self, count: int) -> None:
        if count < 1 or not self.one_sequence and count > self.sequences:
            raise ValueError(f"{count} rows for {self.sequences} block-table rows")

    def _group(self, heads: int) -> None:
        if heads < 1 or heads % self.n_kv_heads:
            raise ValueError(f"{heads} query heads over {self.n_kv_heads} kv heads")

    def _check(self, name: str, t: torch.Tensor, shape: tuple, dtype=torch.float32) -> int:
        if t.dtype is dtype and t.shape == shape and t.get_device() == self._index and t.is_contiguous():
            return t.data_ptr()
        raise ValueError(f"{name}: expected a contiguous {dtype} tensor of {tuple(shape)} on {self.device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")

    def _output(self, name: str, t: torch.Tensor | None, shape, dtype=torch.float32, fill=None) -> torch.Tensor:
        if t is None:
            make = torch.empty(shape, dtype=dtype, device=self.device)
            return make if fill is None else make.fill_(fill)
        self._check(name, t, shape, dtype)
        return t

    def _space(self, t: torch.Tensor | None, need: int) -> torch.Tensor:
        if need == 0:
            raise ValueError("arguments refused by the library (see include/rtxllm/paged_kv.h)")
        if t is None:
            return torch.empty(need, dtype=torch.uint8, device=self.device)
        if t.dtype != torch.uint8 or t.numel() < need or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"workspace: expected a contiguous uint8 tensor of >= {need} bytes on {self.device}")
        return t

    def _call(self, name: str, *args) -> None:
        """name(cache, *args, stream) on the cache's device and its current stream."""
        call, index = getattr(lib(), name), self._index
        # the handle torch.cuda.current_stream(index).cuda_stream gives, without the objects
        # around it (0.1 us instead of 2.7); the device alike (0.25 us)
        stream = torch._C._cuda_getCurrentRawStream(index)
        if torch._C._cuda_getDevice() == index:
            rc = call(self.ref, *args, stream)
        else:
            with torch.cuda.device(index):
                rc = call(self.ref, *args, stream)
        check(name, rc)


def _type_of(name: str, x: torch.Tensor) -> int:
    if x.dtype in TYPES:
        return TYPES[x.dtype]
    raise ValueError(f"{name}: expected float32 or float16, got {x.dtype}")


def _call_rows(cache: PagedKV, rows: int, pos: torch.Tensor, start: torch.Tensor | None) -> tuple:
    """(start, pos, sequences) of a call whose sequences have rows start[s] .. start[s + 1] - 1, or one each."""
    sequences = pos.numel()
    cache._rows(sequences)
    if start is None and rows != sequences:
        raise ValueError(f"{rows} rows for {sequences} sequences without their starts")
    at = None if start is None else cache._check("start", start, (sequences + 1,), torch.int32)
    return at, cache._check("pos", pos, (sequences,), torch.int32), sequences


def _rows_of(name: str, cache: PagedKV, x: torch.Tensor, count: int, heads: int | None) -> int:
    """Stride in floats between the rows of x [count][heads][head_dim], whose rows
    may lie apart (parts of one stacked projection)."""
    shape, stride = x.shape, x.stride()
    if (x.dtype is torch.float32 and x.get_device() == cache._index and len(shape) == 3 and shape[0] == count and
            (heads is None or shape[1] == heads) and shape[2] == cache.head_dim and stride[2] == 1 and
            (stride[1] == cache.head_dim or shape[1] == 1)):
        return stride[0] if count > 1 else shape[1] * cache.head_dim
    raise ValueError(f"{name}: expected float32 [{count}][{heads or 'heads'}][{cache.head_dim}] with contiguous rows on "
                     f"{cache.device}, got {x.dtype} {tuple(shape)} with strides {stride}")


def qk_norm_rope_append(cache: PagedKV, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, pos: torch.Tensor, *,
                        theta: float, eps: float = 1e-6, rotary_dim: int | None = None, pairing: str = "halves",
                        slot: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                        slot_pos: torch.Tensor | None = None, slot_weight: torch.Tensor | None = None) -> torch.Tensor:
    """Norm of every q and k head, rotation at pos, k and v into the cache at slot
    (default: pos); returns the rotated q [count][n_heads][head_dim]."""
    count = pos.numel()
    cache._rows(count)
    if pairing not in PAIRINGS:
        raise ValueError(f"pairing {pairing!r}: one of {sorted(PAIRINGS)}")
    qs = _rows_of("q", cache, q, count, None)
    ks = _rows_of("k", cache, k, count, cache.n_kv_heads)
    vs = _rows_of("v", cache, v, count, cache.n_kv_heads)
    width = (cache.head_dim,)
    qw = None if q_weight is None else cache._check("q_weight", q_weight, width)
    kw = None if k_weight is None else cache._check("k_weight", k_weight, width)
    rows = (count,)
    pp = cache._check("pos", pos, rows, torch.int32)
    lp = None if slot is None else cache._check("slot", slot, rows, torch.int32)
    state = (cache.sequences, cache.n_kv_heads, cache.capacity)
    sp = None if slot_pos is None else cache._check("slot_pos", slot_pos, state, torch.int32)
    sw = None if slot_weight is None else cache._check("slot_weight", slot_weight, state)
    q_out = cache._output("q_out", q_out, q.shape, fill=0.0)
    cache._call("rtxllm_qk_norm_rope_append_f16", q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, qw, kw,
                q.shape[1], cache.head_dim if rotary_dim is None else _u32("rotary_dim", rotary_dim), PAIRINGS[pairing],
                theta, eps, pp, lp, count, q_out.data_ptr(), sp, sw)
    return q_out


def page_bounds(cache: PagedKV, last: torch.Tensor, bounds: torch.Tensor, first: torch.Tensor | None = None,
                span: int = 1) -> torch.Tensor:
    """Bounds (fp16 [n_pages][n_kv_heads][2][head_dim]) of the pages that hold
    positions first..last (default: the newest page), at most span of them."""
    count = last.numel()
    cache._rows(count)
    b = cache._check("bounds", bounds, (cache.n_pages, cache.n_kv_heads, 2, cache.head_dim), torch.float16)
    f = None if first is None else cache._check("first", first, (count,), torch.int32)
    cache._call("rtxllm_kv_page_bounds_f16", f, cache._check("last", last, (count,), torch.int32), count,
                _u32("span", span), b)
    return bounds


def select_workspace(cache: PagedKV, count: int) -> torch.Tensor:
    return cache._space(None, int(lib().rtxllm_attn_select_workspace(cache.ref, _u32("count", count))))


def select_pages(cache: PagedKV, bounds: torch.Tensor, q: torch.Tensor, pos: torch.Tensor, n_select: int,
                 n_first: int = 1, n_last: int = 1, pages: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The logical pages that each query and kv head attends: int32
    [count][n_kv_heads][n_select], ascending, -1 behind the last."""
    count = pos.numel()
    cache._rows(count)
    heads = q.shape[1] if q.dim() == 3 else 0
    cache._group(heads)
    b = cache._check("bounds", bounds, (cache.n_pages, cache.n_kv_heads, 2, cache.head_dim), torch.float16)
    qp = cache._check("q", q, (count, heads, cache.head_dim))
    pp = cache._check("pos", pos, (count,), torch.int32)
    first, last, select = _u32("n_first", n_first), _u32("n_last", n_last), _u32("n_select", n_select)
    pages = cache._output("pages", pages, (count, cache.n_kv_heads, n_select), torch.int32, -1)
    ws = cache._space(workspace, int(lib().rtxllm_attn_select_workspace(cache.ref, count)))
    cache._call("rtxllm_attn_select_pages", b, qp, heads, pp, count, first, last, select, pages.data_ptr(),
                ws.data_ptr(), ws.numel())
    return pages


def attn_pages_workspace(cache: PagedKV, n_heads: int, n_select: int, count: int) -> torch.Tensor:
    return cache._space(None, int(lib().rtxllm_attn_pages_workspace(cache.ref, _u32("n_heads", n_heads), _u32("n_select", n_select),
                                                              _u32("count", count))))


def attn_pages(cache: PagedKV, q: torch.Tensor, pages: torch.Tensor, pos: torch.Tensor,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each query over the positions <= pos of its listed pages."""
    count = pos.numel()
    cache._rows(count)
    heads = q.shape[1] if q.dim() == 3 else 0
    cache._group(heads)
    n_select = pages.shape[-1]
    qp = cache._check("q", q, (count, heads, cache.head_dim))
    lp = cache._check("pages", pages, (count, cache.n_kv_heads, n_select), torch.int32)
    pp = cache._check("pos", pos, (count,), torch.int32)
    out = cache._output("out", out, q.shape, fill=0.0)
    ws = cache._space(workspace, int(lib().rtxllm_attn_pages_workspace(cache.ref, heads, n_select, count)))
    cache._call("rtxllm_attn_decode_pages_gqa_f16", qp, heads, lp, n_select, pp, count, out.data_ptr(), ws.data_ptr(),
                ws.numel())
    return out


def attn_weights_workspace(cache: PagedKV, n_heads: int, count: int) -> torch.Tensor:
    return cache._space(None, int(lib().rtxllm_attn_weights_workspace(cache.ref, _u32("n_heads", n_heads), _u32("count", count))))


def attn_weights(cache: PagedKV, q: torch.Tensor, last: torch.Tensor, weight: torch.Tensor,
                 weight_out: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each query over slots 0..last; weight_out (default: weight
    itself) = weight + each slot's softmax weight, summed over the kv head's queries.
    weight fp32 [count][n_kv_heads][capacity]."""
    count = last.numel()
    cache._rows(count)
    heads = q.shape[1] if q.dim() == 3 else 0
    cache._group(heads)
    state = (count, cache.n_kv_heads, cache.capacity)
    qp = cache._check("q", q, (count, heads, cache.head_dim))
    pp = cache._check("last", last, (count,), torch.int32)
    wp = cache._check("weight", weight, state)
    wo = wp if weight_out is None else cache._check("weight_out", weight_out, state)
    out = cache._output("out", out, q.shape, fill=0.0)
    ws = cache._space(workspace, int(lib().rtxllm_attn_weights_workspace(cache.ref, heads, count)))
    cache._call("rtxllm_attn_decode_weights_gqa_f16", qp, heads, pp, count, out.data_ptr(), wp, wo, ws.data_ptr(),
                ws.numel())
    return out


def evict_workspace(cache: PagedKV, keep: int, count: int) -> torch.Tensor:
    return cache._space(None, int(lib().rtxllm_kv_evict_workspace(cache.ref, _u32("keep", keep), _u32("count", count))))


def evict(cache: PagedKV, length: torch.Tensor, pos: torch.Tensor, keep: int, weight: torch.Tensor,
          slot_pos: torch.Tensor, n_first: int = 0, n_recent: int = 0, weight_out: torch.Tensor | None = None,
          slot_pos_out: torch.Tensor | None = None, length_out: torch.Tensor | None = None,
          workspace: torch.Tensor | None = None) -> None:
    """Sequences of more than `keep` slots keep that many for each kv head: the
    protected ones (the first n_first and the n_recent newest positions), then those
    with the largest weight. Outputs default to their inputs."""
    count = length.numel()
    cache._rows(count)
    state = (count, cache.n_kv_heads, cache.capacity)
    lp = cache._check("length", length, (count,), torch.int32)
    pp = cache._check("pos", pos, (count,), torch.int32)
    wp = cache._check("weight", weight, state)
    sp = cache._check("slot_pos", slot_pos, state, torch.int32)
    wo = wp if weight_out is None else cache._check("weight_out", weight_out, state)
    so = sp if slot_pos_out is None else cache._check("slot_pos_out", slot_pos_out, state, torch.int32)
    lo = lp if length_out is None else cache._check("length_out", length_out, (count,), torch.int32)
    first, recent = _u32("n_first", n_first), _u32("n_recent", n_recent)
    ws = cache._space(workspace, int(lib().rtxllm_kv_evict_workspace(cache.ref, _u32("keep", keep), count)))
    cache._call("rtxllm_kv_evict_f16", lp, pp, count, keep, first, recent, wp, sp, wo, so, lo, ws.data_ptr(),
                ws.numel())


def _attn_rows(cache: PagedKV, name: tuple, q: torch.Tensor, pos: torch.Tensor, start: torch.Tensor | None,
               window: int | None, sinks: int, out: torch.Tensor | None, workspace: torch.Tensor | None) -> torch.Tensor:
    if q.dim() != 3:
        raise ValueError(f"q: expected [rows][n_heads][{cache.head_dim}], got {tuple(q.shape)}")
    rows, heads = q.shape[0], q.shape[1]
    cache._group(heads)
    kind = _type_of("q", q)
    qp = cache._check("q", q, (rows, heads, cache.head_dim), q.dtype)
    sp, pp, sequences = _call_rows(cache, rows, pos, start)
    near, first = cache.capacity if window is None else _u32("window", window), _u32("sinks", sinks)
    out = cache._output("out", out, q.shape, q.dtype, fill=0.0)
    ws = cache._space(workspace, int(getattr(lib(), name[0])(cache.ref, heads, sequences, rows, near, first)))
    cache._call(name[1], qp, kind, heads, sp, pp, sequences, rows, near, first, out.data_ptr(), ws.data_ptr(), ws.numel())
    return out


def attn_window_workspace(cache: PagedKV, n_heads: int, sequences: int, rows: int, window: int | None = None,
                          sinks: int = 0) -> torch.Tensor:
    near = cache.capacity if window is None else _u32("window", window)
    return cache._space(None, int(lib().rtxllm_attn_window_workspace(
        cache.ref, _u32("n_heads", n_heads), _u32("sequences", sequences), _u32("rows", rows), near, _u32("sinks", sinks))))


def attn_window(cache: PagedKV, q: torch.Tensor, pos: torch.Tensor, start: torch.Tensor | None = None, *,
                window: int | None = None, sinks: int = 0, out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens, q [rows][n_heads][head_dim] of float32 or float16: sequence s has rows start[s] ..
    start[s + 1] - 1 (start None: row s) at positions pos[s], pos[s] + 1, ... Each sees the positions up to
    its own that are less than `window` (None: any number) behind it, and the first `sinks`."""
    return _attn_rows(cache, ("rtxllm_attn_window_workspace", "rtxllm_attn_window_f16"), q, pos, start, window, sinks, out,
                      workspace)
