"""``PagedKVCache``: a KV cache held in 4 bits, in pages that rows can share, with the attention that reads it.

Where ``KVCache`` (``cache.py``) keeps one layer's dense keys and values and returns a new cache from every call, this
cache holds all layers in one pool of 64-token pages and changes in place, so that a serving loop can

    cache = PagedKVCache.init(num_layers, num_pages, num_rows, max_seq_len, num_kv_heads, head_dim)
    cache.extend(counts)                    # room for this call's tokens of every row
    for layer in range(num_layers):
        cache.append(layer, k, v)           # [rows, S, kv heads, hd], quantised into the pages
        o = cache.attend(layer, q)          # [rows, S, heads, hd]
    cache.fork(parents)                     # best-of-n, beams: rows share pages, written pages are copied first
    cache.rollback(n)                       # drafted tokens that were not taken
    cache.free(rows); cache.compact()       # finished rows; used pages to the front of the pool

All state (page table, lengths, reference counts) is on the device and every call of the loop is a kernel launch or two
on the current stream without a host synchronisation (given ints, or tensors on the cache's device), so the loop can be
captured in a CUDA graph.  ``check`` and ``resize`` read the device, and so do the blocks and models that take this cache
(``nn.Attention``, ``apply``): those are not captured.  Page choices are
deterministic (lowest free page, rows in order).  What only the device can see (a full pool, a row past ``max_seq_len``,
a parent out of range) sets a status word that ``check`` raises; such an ``extend`` changes nothing and gives every row
zero tokens of the current call.

The format is 4.5 bits a value: 4-bit integers -7..7 with one scale of 4 significant bits for every 32 neighbouring
channels of a token (``include/jxb200.h``).  A group with a non-finite value, or one of magnitude 2^122 or more, decodes
to NaN.  Calls on one cache that change it must be ordered on the device like writes to any tensor; ``attend`` and
``read`` may run at the same time.  ``lengths`` and ``counts`` may be read, not written, and be given to ``extend``,
``rollback`` and ``read``; ``fork`` and ``free`` take no argument that lies in the cache's own tensors.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import numpy as np
import torch

from . import _native as N
from ._checks import normalize_count, normalize_float, widened

__all__ = ["PagedKVCache", "PagedKVLayer"]

PAGE_SIZE = 64
HEAD_DIMS = (64, 128, 256)
_current_device = torch.cuda.current_device
_DTYPES = {torch.float32: N.JX_F32, torch.bfloat16: N.JX_BF16}


def block_bytes(head_dim: int) -> int:
    """Bytes of one (layer, page, KV head): 64 tokens of key and value codes and their scales."""
    return PAGE_SIZE * head_dim + PAGE_SIZE * (head_dim // 32) * 4


def _positive(name: str, value) -> int:
    value = normalize_count(name, value)
    if value <= 0:
        raise ValueError(f"{name} must be positive, got {value}.")
    return value


class PagedKVCache:
    """``pages`` uint8 [layers, pages, kv heads, block], ``table`` int32 [rows, pages per row], ``lengths`` and ``counts``
    int32 [rows], ``refs`` int32 [pages], ``status`` int32 [1]: contiguous tensors on one CUDA device.  ``init`` makes an
    empty cache; the constructor takes tensors in this layout (a saved cache)."""

    def __init__(self, *, pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor,
                 refs: torch.Tensor, head_dim: int, status: Optional[torch.Tensor] = None):
        head_dim = normalize_count("head_dim", head_dim)
        if head_dim not in HEAD_DIMS:
            raise NotImplementedError(f"PagedKVCache takes a head_dim of 64, 128 or 256, got {head_dim}.")
        if status is None and isinstance(pages, torch.Tensor):
            status = torch.zeros(1, dtype=torch.int32, device=pages.device)
        for name, t, dtype, ndim in (("pages", pages, torch.uint8, 4), ("table", table, torch.int32, 2),
                                     ("lengths", lengths, torch.int32, 1), ("counts", counts, torch.int32, 1),
                                     ("refs", refs, torch.int32, 1), ("status", status, torch.int32, 1)):
            if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.ndim != ndim:
                raise TypeError(f"{name} must be a {ndim}D {dtype} tensor, got {_what(t)}.")
            if t.numel() == 0 or not t.is_contiguous():
                raise ValueError(f"{name} must be non-empty and contiguous, got shape {tuple(t.shape)}.")
            if t.device != pages.device:
                raise ValueError(f"{name} must be on {pages.device} as pages, got {t.device}.")
        if pages.shape[3] != block_bytes(head_dim):
            raise ValueError(f"pages must hold blocks of {block_bytes(head_dim)} bytes for head_dim={head_dim}, got "
                             f"{pages.shape[3]}.")
        if lengths.shape[0] != table.shape[0] or counts.shape[0] != table.shape[0]:
            raise ValueError("table, lengths and counts must have one entry per row, got "
                             f"{table.shape[0]}, {lengths.shape[0]} and {counts.shape[0]}.")
        if refs.shape[0] != pages.shape[1]:
            raise ValueError(f"refs must have one entry per page, got {refs.shape[0]} and {pages.shape[1]}.")
        if table.shape[0] > 8192 or table.shape[1] > 1 << 24 or table.numel() >= 1 << 31:
            raise ValueError(f"table must have at most 8192 rows, 2^24 pages per row and 2^31 entries, got {tuple(table.shape)}.")
        self.pages, self.table, self.lengths, self.counts = pages, table, lengths, counts
        self.refs, self.status, self.head_dim = refs, status, head_dim
        self.device = pages.device
        self.num_layers, self.num_pages, self.num_kv_heads = pages.shape[:3]
        self.num_rows, self.row_pages = table.shape
        c = N.JxKv4Cache()
        c.pages, c.table, c.lengths = pages.data_ptr(), table.data_ptr(), lengths.data_ptr()
        c.counts, c.refs, c.status = counts.data_ptr(), refs.data_ptr(), status.data_ptr()
        c.num_layers, c.num_pages, c.num_rows, c.row_pages = self.num_layers, self.num_pages, self.num_rows, self.row_pages
        c.num_kv_heads, c.head_dim = self.num_kv_heads, head_dim
        self._c = c
        self._ref = ctypes.byref(c)
        self._lib = None
        self._index = self.device.index
        self._plan_ints = 0
        self._ws_bytes: dict = {}

    @classmethod
    def init(cls, num_layers: int, num_pages: int, num_rows: int, max_seq_len: int, num_kv_heads: int, head_dim: int,
             device=None) -> "PagedKVCache":
        """An empty cache on ``device`` (the current CUDA device by default): ``num_pages`` pages of 64 tokens shared by
        ``num_rows`` rows of at most ``max_seq_len`` tokens (rounded up to whole pages)."""
        num_layers, num_pages = _positive("num_layers", num_layers), _positive("num_pages", num_pages)
        num_rows, max_seq_len = _positive("num_rows", num_rows), _positive("max_seq_len", max_seq_len)
        num_kv_heads, head_dim = _positive("num_kv_heads", num_kv_heads), _positive("head_dim", head_dim)
        if head_dim not in HEAD_DIMS:
            raise NotImplementedError(f"PagedKVCache takes a head_dim of 64, 128 or 256, got {head_dim}.")
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise RuntimeError(f"PagedKVCache lives on a CUDA device (got {dev}).")
        i32 = dict(dtype=torch.int32, device=dev)
        return cls(pages=torch.zeros(num_layers, num_pages, num_kv_heads, block_bytes(head_dim), dtype=torch.uint8, device=dev),
                   table=torch.full((num_rows, -(-max_seq_len // PAGE_SIZE)), -1, **i32),
                   lengths=torch.zeros(num_rows, **i32), counts=torch.zeros(num_rows, **i32),
                   refs=torch.zeros(num_pages, **i32), head_dim=head_dim)

    @property
    def max_seq_len(self) -> int:
        return self.row_pages * PAGE_SIZE

    def layer(self, index: int) -> "PagedKVLayer":
        """One layer of this cache, as ``nn.Attention`` and the decoder blocks take it for ``kv_cache``."""
        return PagedKVLayer(self, self._layer(index))

    # -- plumbing ----------------------------------------------------------------------------------
    def _layer(self, layer) -> int:
        if type(layer) is not int:
            layer = normalize_count("layer", layer)
        if not 0 <= layer < self.num_layers:
            raise ValueError(f"layer must be within [0, {self.num_layers}), got {layer}.")
        return layer

    def _call(self, name: str, *args):
        """One library call on the cache's device and its current stream."""
        lib = self._lib
        if lib is None:
            if self.device.type != "cuda":
                raise RuntimeError(f"{name}: PagedKVCache runs on a CUDA device (got {self.device}).")
            lib = self._lib = N.load()
        index = self._index
        if index == _current_device():
            rc = getattr(lib, name)(self._ref, *args, N.raw_stream(index))
        else:
            with torch.cuda.device(index):
                rc = getattr(lib, name)(self._ref, *args, N.raw_stream(index))
        if rc:
            N.check(rc, name)

    def _states(self, name: str, x, heads: Optional[int]) -> torch.Tensor:
        """A float32 / bfloat16 [rows, S, heads, hd] tensor on the cache's device with a dense last axis."""
        if not isinstance(x, torch.Tensor) or x.ndim != 4:
            raise ValueError(f"{name} must be a 4D tensor, got {_what(x)}.")
        if x.dtype not in _DTYPES:
            raise TypeError(f"{name} must be float32 or bfloat16, got dtype {x.dtype}.")
        shape = x.shape
        if shape[0] != self.num_rows or shape[3] != self.head_dim or (heads is not None and shape[2] != heads):
            raise ValueError(f"{name} must have shape ({self.num_rows}, S, {'heads' if heads is None else heads}, "
                             f"{self.head_dim}), got {tuple(shape)}.")
        if shape[1] <= 0 or shape[2] <= 0:
            raise ValueError(f"{name} must not contain empty axes, got shape {tuple(shape)}.")
        if x.device != self.device:
            raise ValueError(f"{name} must be on {self.device}, got {x.device}.")
        return x if x.stride(3) == 1 else x.contiguous()

    def _row_ints(self, name: str, x) -> torch.Tensor:
        """An int32 [rows] tensor on the cache's device."""
        if not isinstance(x, torch.Tensor):
            x = torch.as_tensor(x)
        if x.dtype == torch.bool or x.dtype.is_floating_point or x.dtype.is_complex:
            raise TypeError(f"{name} must contain integers, got dtype {x.dtype}.")
        if x.shape != self.lengths.shape:
            raise ValueError(f"{name} must have shape ({self.num_rows},), got {tuple(x.shape)}.")
        if x.dtype == torch.int32 and x.device == self.device and x.is_contiguous():
            return x
        x = widened(x)
        if x.dtype == torch.int64:
            x = x.clamp(-2 ** 31, 2 ** 31 - 1)
        return x.to(device=self.device, dtype=torch.int32).contiguous()

    def _plan(self) -> torch.Tensor:
        if not self._plan_ints:
            n = N.LL()
            N.check(N.load().jx_kv4_workspace_ints(self._ref, n), "jx_kv4_workspace_ints")
            self._plan_ints = n.value
        return torch.empty(self._plan_ints, dtype=torch.int32, device=self.device)

    # -- tokens ------------------------------------------------------------------------------------
    def extend(self, counts) -> None:
        """Begins a call of ``counts`` more tokens of every row (an int, or int32 [rows]; 0 leaves a row out): the rows
        grow, new pages are taken and shared pages that will be written on are copied.  Without room nothing
        changes, ``counts`` becomes zero and ``check`` raises."""
        if _is_vector(counts):
            c, n = self._row_ints("counts", counts), 0
        else:
            c, n = None, normalize_count("counts", counts)
            if n < 0:
                raise ValueError(f"counts must not be negative, got {n}.")
            n = min(n, 2 ** 31 - 1)
        ws = self._plan()
        self._call("jx_kv4_extend", None if c is None else c.data_ptr(), n, ws.data_ptr(), ws.numel())

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Quantises the call's keys and values [rows, S, kv heads, hd] into a layer's pages.  Row r has ``counts[r]``
        tokens; those behind are padding and not read."""
        layer = self._layer(layer)
        k, v = self._states("k", k, self.num_kv_heads), self._states("v", v, self.num_kv_heads)
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError(f"k and v must have the same shape and dtype, got {tuple(k.shape)} {k.dtype} and "
                             f"{tuple(v.shape)} {v.dtype}.")
        ks, vs = k.stride(), v.stride()
        self._call("jx_kv4_append", layer, k.shape[1], k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2],
                   _DTYPES[k.dtype])

    def read(self, layer: int, start=0, length: Optional[int] = None, dtype=torch.bfloat16):
        """The dequantised keys and values [rows, length, kv heads, hd] of positions ``start`` (an int, or int32 [rows])
        onwards, zeros outside a row: every value is exact in bfloat16 and float32."""
        layer = self._layer(layer)
        if dtype not in _DTYPES:
            raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}.")
        length = self.max_seq_len if length is None else _positive("length", length)
        if _is_vector(start):
            ptr, add = self._row_ints("start", start), 0
        else:
            ptr, add = None, normalize_count("start", start)
            if not 0 <= add < 1 << 31:
                raise ValueError(f"start must be within [0, 2^31), got {add}.")
        k = torch.empty((self.num_rows, length, self.num_kv_heads, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        self._call("jx_kv4_read", layer, None if ptr is None else ptr.data_ptr(), add, length, k.data_ptr(), v.data_ptr(),
                   _DTYPES[dtype])
        return k, v

    def attend(self, layer: int, q: torch.Tensor, scale: Optional[float] = None,
               sliding_window: Optional[int] = None) -> torch.Tensor:
        """Causal attention of the call's queries [rows, S, heads, hd] over a layer's pages, this call's tokens among
        them: query i of row r stands at position ``lengths[r] - counts[r] + i`` and, with a sliding window, sees that
        many positions back, its own among them.  float32 softmax of ``scale`` (``hd ** -0.5`` by default) times q.k;
        heads must be a multiple of the KV heads, and queries below 2^115 in magnitude (their products' partial sums are
        in float32).  Returns [rows, S, heads, hd] in q's dtype, zeros for the padding behind a row's ``counts[r]``
        queries."""
        layer = self._layer(layer)
        q = self._states("q", q, None)
        S, heads = q.shape[1], q.shape[2]
        if heads % self.num_kv_heads:
            raise ValueError(f"q heads must be a multiple of the {self.num_kv_heads} KV heads, got {heads}.")
        scale = self.head_dim ** -0.5 if scale is None else normalize_float("scale", scale)
        window = 0 if sliding_window is None else min(_positive("sliding_window", sliding_window), 2 ** 31 - 1)
        dtype = _DTYPES[q.dtype]
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        size = self._ws_bytes.get((S, heads, dtype))
        if size is None:
            n = N.LL()
            N.check(N.load().jx_kv4_attend_workspace(self._ref, S, heads, dtype, n), "jx_kv4_attend_workspace")
            self._ws_bytes[(S, heads, dtype)] = size = n.value
        # a workspace of its own for every call: calls on several streams, and graphs, do not share one
        ws = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        st = q.stride()
        self._call("jx_kv4_attend", layer, S, heads, q.data_ptr(), st[0], st[1], st[2], out.data_ptr(), scale, window,
                   ws.data_ptr() if size else None, size, dtype)
        return out

    def position_ids(self, length: int) -> torch.Tensor:
        """int32 [rows, length]: positions of the call's tokens; padding repeats the row's last position."""
        i = torch.arange(normalize_count("length", length), dtype=torch.int32, device=self.device)
        pos = (self.lengths - self.counts)[:, None] + i[None]
        return torch.minimum(pos, (self.lengths - 1)[:, None]).clamp(min=0)

    # -- rows and pages ------------------------------------------------------------------------------
    def fork(self, parents) -> None:
        """Row r becomes a copy of the row that ``parents[r]`` (int32 [rows]) named before the call; a negative parent
        empties it.  Pages are shared, none is copied."""
        p = self._row_ints("parents", parents)
        self._call("jx_kv4_fork", p.data_ptr())

    def rollback(self, n) -> None:
        """Every row loses its last ``n`` tokens (an int, or int32 [rows]); pages that held nothing else are given back.  A
        row of fewer tokens stays as it is and ``check`` raises."""
        if _is_vector(n):
            t, n = self._row_ints("n", n), 0
        else:
            t, n = None, normalize_count("n", n)
            if not 0 <= n < 1 << 31:
                raise ValueError(f"n must not be negative, got {n}.")
        self._call("jx_kv4_rollback", None if t is None else t.data_ptr(), n)

    def free(self, rows) -> None:
        """Empties rows: a boolean tensor [rows], or a sequence of row numbers."""
        if not isinstance(rows, torch.Tensor):
            mask = torch.zeros(self.num_rows, dtype=torch.bool)
            for r in rows:
                r = normalize_count("rows", r)
                if not 0 <= r < self.num_rows:
                    raise ValueError(f"rows must be within [0, {self.num_rows}), got {r}.")
                mask[r] = True
            rows = mask
        if rows.dtype != torch.bool or tuple(rows.shape) != (self.num_rows,):
            raise ValueError(f"rows must be a boolean tensor of shape ({self.num_rows},), got {_what(rows)}.")
        rows = rows.to(self.device).contiguous()
        self._call("jx_kv4_free", rows.data_ptr())

    def compact(self) -> torch.Tensor:
        """Moves the used pages to the front of the pool; their number as an int32 [1] tensor on the device."""
        used = torch.empty(1, dtype=torch.int32, device=self.device)
        ws = self._plan()
        self._call("jx_kv4_compact", used.data_ptr(), ws.data_ptr(), ws.numel())
        return used

    def resize(self, num_pages: int) -> "PagedKVCache":
        """A new cache of the same content with a pool of ``num_pages`` pages; used pages must lie below it (``compact``
        puts them there)."""
        num_pages = _positive("num_pages", num_pages)
        if num_pages < self.num_pages and bool((self.refs[num_pages:] != 0).any()):
            raise ValueError(f"Cannot resize the pool to {num_pages} pages below a used page; compact it first.")
        keep = min(num_pages, self.num_pages)
        pages = torch.zeros((self.num_layers, num_pages) + tuple(self.pages.shape[2:]), dtype=torch.uint8, device=self.device)
        pages[:, :keep] = self.pages[:, :keep]
        refs = torch.zeros(num_pages, dtype=torch.int32, device=self.device)
        refs[:keep] = self.refs[:keep]
        return PagedKVCache(pages=pages, refs=refs, table=self.table.clone(), lengths=self.lengths.clone(),
                            counts=self.counts.clone(), status=self.status.clone(), head_dim=self.head_dim)

    def check(self) -> None:
        """Synchronises, and raises if a call on this cache met an error on the device since the last check."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            what = ("a row or the pool had no room, or a row, page or token count was out of range"
                    if code == N.JX_ERR_RANGE else N.STATUS_NAMES.get(code, "error"))
            raise RuntimeError(f"PagedKVCache: device status {code} ({what}).")


class PagedKVLayer:
    """One layer of a ``PagedKVCache`` (``PagedKVCache.layer``): ``nn.Attention`` appends its keys and values to it and
    attends over it.  ``extend`` of the cache comes first, once for all layers."""

    def __init__(self, cache: PagedKVCache, index: int):
        self.cache, self.index = cache, index

    def update_and_attend(self, q, k, v, scale: float, sliding_window: Optional[int]) -> torch.Tensor:
        self.cache.append(self.index, k, v)
        return self.cache.attend(self.index, q, scale=scale, sliding_window=sliding_window)


def _is_vector(x) -> bool:
    """Whether an argument is one value for every row (arrays too have ``__index__``)."""
    return not hasattr(x, "__index__") or isinstance(x, (torch.Tensor, np.ndarray))


def _what(x) -> str:
    return f"{x.dtype} tensor of shape {tuple(x.shape)}" if isinstance(x, torch.Tensor) else f"{type(x)}"
