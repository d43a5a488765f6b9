"""Paged K/V caches of the caller over the CUDA C ABI: page requests on tables in device memory.

A `PagedCache` is a pool of 16-position pages with its tables as torch tensors on one GPU, for
programs that run their own layers over this library's kernels (the cache inside
`ane.stories.Engine` is the engine's own).  Sequences that start from a common prompt hold its
pages in common: `fork` shares the complete pages and copies a partly filled last one, `free`
counts references, `compact` gathers the live pages at the pool's start, `copy` moves listed pages.
Requests are enqueued on the calling thread's current CUDA stream and return without waiting;
`check` waits and raises for what the device refused.  `PrefixPlan.attend` is the attention of a
batch in groups that share their first positions, the shared pages read once per group.  The reference keeps one dense cache per
decoder (ane/stories/infer.go:113-114) and has no counterpart.

torch is used for device memory and streams only; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C

import torch

from .. import _abi
from .._abi import LLMError

PAGE = 16

_TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16}


def meta_words(n_pages: int, max_seqs: int, max_pages: int) -> int:
    """int32 words of a cache's packed tables: 4 (free pages, status, 0, 0), pages per slot,
    references per page, the free stack, the block table."""
    return 4 + max_seqs + 2 * n_pages + max_seqs * max_pages


def _need(t, what: str, dtype, device):
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or not t.is_contiguous():
        raise LLMError(_abi.LLM_ERR_INVALID, f"{what} must be a contiguous {dtype} tensor on {device}")
    return t.data_ptr()


class PagedCache:
    """A page pool and its tables.  `pool` [n_layers, n_pages, n_kv_heads, 2, 16 * head_dim] and
    `meta` (the packed tables, `meta_words`) may be the caller's; new ones are made empty, with
    page 0 handed out first."""

    def __init__(self, dtype: str, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, max_seqs: int,
                 max_pages: int, device: int = 0, pool=None, meta=None):
        if dtype not in _TORCH:
            raise LLMError(_abi.LLM_ERR_INVALID, f"cache dtype {dtype!r} (fp16 or bf16)")
        self._lib = _abi.lib()
        words = self._lib.llm_pages_work_words(n_pages, max_seqs)
        if min(n_layers, n_kv_heads, head_dim, max_pages) <= 0 or words == 0:
            raise LLMError(_abi.LLM_ERR_INVALID, "cache sizes out of range")
        self.dtype, self.torch_dtype, self.device = dtype, _TORCH[dtype], torch.device("cuda", device)
        self.n_layers, self.n_pages, self.n_kv_heads, self.head_dim = n_layers, n_pages, n_kv_heads, head_dim
        self.max_seqs, self.max_pages = max_seqs, max_pages
        shape = (n_layers, n_pages, n_kv_heads, 2, PAGE * head_dim)
        if pool is None:
            pool = torch.zeros(shape, dtype=self.torch_dtype, device=self.device)
        if tuple(pool.shape) != shape:
            raise LLMError(_abi.LLM_ERR_INVALID, f"the pool's shape is {tuple(pool.shape)}, not {shape}")
        fresh = meta is None
        if fresh:
            meta = torch.zeros(meta_words(n_pages, max_seqs, max_pages), dtype=torch.int32, device=self.device)
        if tuple(meta.shape) != (meta_words(n_pages, max_seqs, max_pages),):
            raise LLMError(_abi.LLM_ERR_INVALID, f"the packed tables have shape {tuple(meta.shape)}, "
                                                 f"not ({meta_words(n_pages, max_seqs, max_pages)},)")
        _need(pool, "the pool", self.torch_dtype, self.device)
        _need(meta, "the packed tables", torch.int32, self.device)
        self.pool, self.meta = pool, meta
        self._work = torch.zeros(words, dtype=torch.int32, device=self.device)
        a, b, c = 4 + max_seqs, 4 + max_seqs + n_pages, 4 + max_seqs + 2 * n_pages
        self.n_free, self.status, self.npages = meta[0:1], meta[1:2], meta[4:a]
        self.refs, self.free_pages, self.table = meta[a:b], meta[b:c], meta[c:].view(max_seqs, max_pages)
        if fresh:
            self.n_free.fill_(n_pages)
            self.free_pages.copy_(torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=self.device))
            self.table.fill_(-1)
        self.c_struct = _abi.llm_page_cache(
            _abi.DTYPES[dtype], n_layers, n_pages, n_kv_heads, head_dim, max_seqs, max_pages, pool.data_ptr(),
            self.n_free.data_ptr(), self.status.data_ptr(), self.npages.data_ptr(), self.refs.data_ptr(),
            self.free_pages.data_ptr(), self.table.data_ptr(), self._work.data_ptr())
        self._ref = C.addressof(self.c_struct)

    def _stream(self) -> int:
        # the current stream's handle without the Stream object around it (2 us of every call)
        return torch._C._cuda_getCurrentRawStream(self.device.index)

    def _ints(self, t, what: str, n=None):
        p = _need(t, what, torch.int32, self.device)
        if t.dim() != 1 or (n is not None and t.numel() != n):
            raise LLMError(_abi.LLM_ERR_INVALID, f"{what} has shape {tuple(t.shape)}" + ("" if n is None else f", not ({n},)"))
        return p

    def copy(self, src, dst, to: "PagedCache | None" = None) -> None:
        """Page src[i] of this cache to page dst[i] of `to` (default: this cache; on the same GPU) in
        every layer."""
        to = self if to is None else to
        if not isinstance(to, PagedCache) or to.device != self.device:
            raise LLMError(_abi.LLM_ERR_INVALID, f"`to` must be a PagedCache on {self.device}, not {getattr(to, 'device', to)}")
        at = self._ints(src, "src")
        n = src.numel()
        _abi.check(self._lib.llm_pages_copy(self.device.index, self._ref, to._ref, at, self._ints(dst, "dst", n), n,
                                            self._stream()))

    def fork(self, parents, children, lens, rooms) -> None:
        """Slot children[i] becomes the first lens[i] positions of slot parents[i] (-1: a new
        sequence; the slot itself: it grows), with pages for rooms[i] positions; all or none."""
        at = self._ints(parents, "parents")
        n = parents.numel()
        _abi.check(self._lib.llm_pages_fork(self.device.index, self._ref, at, self._ints(children, "children", n),
                                            self._ints(lens, "lens", n), self._ints(rooms, "rooms", n), n, self._stream()))

    def free(self, slots) -> None:
        """Empty the slots; pages without references go back on the free stack, ascending."""
        at = self._ints(slots, "slots")
        _abi.check(self._lib.llm_pages_free(self.device.index, self._ref, at, slots.numel(), self._stream()))

    def compact(self) -> None:
        """Move the live pages to the pool's start with the fewest moves."""
        _abi.check(self._lib.llm_pages_compact(self.device.index, self._ref, self._stream()))

    def check(self) -> None:
        """Wait for the current stream and raise for the first request the device refused."""
        _abi.check(self._lib.llm_pages_status(self.device.index, self._ref, self._stream()))

    def element_index(self):
        """[16, head_dim] int64: where (row, dim) of a K or V block lies in its 16 * head_dim values."""
        r = torch.arange(PAGE, device=self.device)[:, None]
        d = torch.arange(self.head_dim, device=self.device)[None]
        return (d // 64) * 1024 + r * 64 + (((d // 8) % 8) ^ (r % 8)) * 8 + d % 8


class PrefixPlan:
    """Attention of a batch over `cache` whose sequences share prefixes (llm_prefix_attend).

    Sequence s reads slot slots[s] and has rows[s] query rows (1 when decoding); sequences come
    group by group, group_sizes[g] of them sharing their first prefixes[g] positions, a multiple
    of 16.  max_ctx bounds the positions a sequence may have.  The plan keeps the batch's layout
    and workspace for every layer and step; calls on one plan must be ordered."""

    def __init__(self, cache: PagedCache, n_heads: int, slots, rows, group_sizes, prefixes, max_ctx: int):
        self.cache, self.n_heads, self._lib = cache, n_heads, cache._lib
        slots, rows, sizes, prefixes = (_abi.i32(list(a)) for a in (slots, rows, group_sizes, prefixes))
        if len(slots) != len(rows) or len(sizes) != len(prefixes):
            raise LLMError(_abi.LLM_ERR_INVALID, "slots and rows, group_sizes and prefixes must have one length")
        self.n_seqs, self.n_rows = len(slots), int(rows.sum())
        self._shape = torch.Size((self.n_rows, n_heads, cache.head_dim))
        h = C.c_void_p()
        self.h = None
        _abi.check(self._lib.llm_prefix_plan_create(
            cache.device.index, _abi.DTYPES[cache.dtype], n_heads, cache.n_kv_heads, cache.head_dim,
            _abi.ptr(slots, C.c_int32), _abi.ptr(rows, C.c_int32), self.n_seqs, _abi.ptr(sizes, C.c_int32),
            _abi.ptr(prefixes, C.c_int32), len(sizes), max_ctx, C.byref(h)))
        self.h = h

    def _rows(self, t, what: str):
        c = self.cache
        if not isinstance(t, torch.Tensor) or t.dtype is not c.torch_dtype or t.device != c.device or \
                t.shape != self._shape or t.stride(2) != 1:
            raise LLMError(_abi.LLM_ERR_INVALID, f"{what} must be a {c.torch_dtype} tensor [{self.n_rows}, {self.n_heads}, "
                                                 f"{c.head_dim}] on {c.device} with contiguous rows of a head")
        return t.data_ptr(), t.stride(0), t.stride(1)

    def attend(self, layer: int, q, ctx, scale: float = 0.0, out=None, lse=None):
        """Attention of query rows q [rows, n_heads, head_dim] in `layer`, sequence s having ctx[s]
        positions of which its rows are the last; returns out (new when None).  lse (optional)
        receives the log-sum-exp [rows, n_heads] in f32.  scale 0: 1 / sqrt(head_dim)."""
        c = self.cache
        qp, qr, qh = self._rows(q, "q")
        if out is None:
            out = torch.empty_like(q)
        op, orow, oh = self._rows(out, "out")
        if lse is not None:
            lp = _need(lse, "lse", torch.float32, c.device)
            if lse.shape != (self.n_rows, self.n_heads):
                raise LLMError(_abi.LLM_ERR_INVALID, f"lse has shape {tuple(lse.shape)}, not {(self.n_rows, self.n_heads)}")
        else:
            lp = None
        _abi.check(self._lib.llm_prefix_attend(self.h, c._ref, layer, c._ints(ctx, "ctx", self.n_seqs), qp, qr, qh, scale,
                                               op, orow, oh, lp, c._stream()))
        return out

    def close(self) -> None:
        if self.h is not None:
            self._lib.llm_prefix_plan_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
