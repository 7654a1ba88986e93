"""Batches of sequences over one paged KV pool, on the C ABI (gkv_batch_*).

The reference serves one sequence per cache (README.md:150: batch 1); these
operators serve many over one K and one V pool in the same page layout
(``[16 slots][Hkv][D]``, src/core/page_attention.cpp:128-129):

* :class:`BatchDecode` / :func:`batch_decode` — one new token per sequence:
  append it, attend it over the cache (or over listed pages), and optionally
  keep a running total of the attention each cached token received;
* :class:`PageBounds` / :func:`page_bounds` — the smallest and largest key of
  every page, per head and dimension;
* :class:`PageSelect` / :func:`select_pages` — the pages whose bound scores
  highest for a query, per KV head;
* :class:`CacheEvict` / :func:`evict_tokens` — keep the heaviest and the most
  recent tokens of every KV head, compacted in place.

Each class binds its tensors once (checks, workspace, outputs) and enqueues
with ``run()``, like :class:`genllm_b200.paged_attention.DecodeStep`; ``run``
reads table, lengths and tensors on the device, so it can be captured in a
CUDA graph. Its first run on another stream than the one it was bound on waits
for what that one has queued by then. A bound operator owns its workspace: runs
of one that may overlap on the GPU are the caller's to order, two operators
never share one. The functions bind and run once. Every tensor lives on the
pool's device.
"""
from __future__ import annotations

import ctypes as C
import math
import operator
from typing import Optional

import torch

from . import _lib
from ._lib import GkvError, check, lib
from .paged_attention import PAGE_BLOCK_SIZE, _TORCH_TO_GKV


def _invalid(message: str) -> GkvError:
    return GkvError(_lib.GKV_ERR_INVALID, message)


def _current_stream(device: int) -> int:
    """The current stream's handle (without a Stream object, where torch offers that)."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device) if raw is not None else torch.cuda.current_stream(device).cuda_stream


def _expect(t: torch.Tensor, what: str, device: torch.device, dtype, shape, contiguous: bool = True) -> torch.Tensor:
    """t as a tensor of this device, type and shape (None: any extent)."""
    if not isinstance(t, torch.Tensor):
        raise _invalid(f"{what} must be a tensor")
    if t.device != device:
        raise _invalid(f"{what} is on {t.device}, the pools are on {device}")
    if t.dtype != dtype:
        raise _invalid(f"{what} is {t.dtype}, expected {dtype}")
    if t.dim() != len(shape) or any(e is not None and e != s for e, s in zip(shape, t.shape)):
        raise _invalid(f"{what} has shape {tuple(t.shape)}, expected {tuple('any' if e is None else e for e in shape)}")
    if contiguous and not t.is_contiguous():
        raise _invalid(f"{what} must be contiguous")
    return t


def _count(x, what: str) -> int:
    """x as a 32-bit integer (the C structures would wrap a larger one around)."""
    try:
        n = operator.index(x)
    except TypeError:
        raise _invalid(f"{what} must be an integer, not {x!r}") from None
    if not -2 ** 31 <= n < 2 ** 31:
        raise _invalid(f"{what} {n} is out of range")
    return n


def _rows(t: torch.Tensor, what: str, device: torch.device, dtype, shape) -> torch.Tensor:
    """A [batch, heads, D] tensor of any strides whose rows are whole and 16-byte
    aligned (the stride of an extent of 1 is never used)."""
    _expect(t, what, device, dtype, shape, contiguous=False)
    if t.stride(2) != 1 or any(t.shape[i] > 1 and t.stride(i) % 8 for i in (0, 1)) or t.data_ptr() % 16:
        raise _invalid(f"{what} needs rows of contiguous elements that start on 16 bytes")
    return t


def _page_lists(pages: torch.Tensor, device: torch.device, batch: int, kv_heads: int) -> torch.Tensor:
    """A [batch, kv_heads, n] tensor of page lists, n >= 1 (a tensor without
    elements has a null address, which would mean no lists at all)."""
    _expect(pages, "pages", device, torch.int32, (batch, kv_heads, None))
    if pages.shape[2] < 1:
        raise _invalid("pages lists no page; -1 entries name none")
    return pages


def _table_stride(table: torch.Tensor) -> int:
    """Entries from one row of a [B, T, 2] page table to the next."""
    b, t, _ = table.shape
    if (table.stride(2) != 1 or (t > 1 and table.stride(1) != 2) or table.data_ptr() % 8
            or (b > 1 and (table.stride(0) % 2 or table.stride(0) < 2 * t))):
        raise _invalid("table rows must be contiguous {k_id, v_id} pairs on 8 bytes, one behind the other")
    return table.stride(0) // 2 if b > 1 else t


class PagedBatch:
    """Sequences over one pool pair: ``k_pool`` and ``v_pool`` [P, 16, Hkv, D]
    (bf16 or f16, D 64, 128 or 256), ``table`` [B, T, 2] int32 of {k_id, v_id}
    page ids per logical page (rows may be strided), ``lens`` [B] int32 cached
    tokens, negative for a sequence to skip. The tensors are the caller's: it
    writes new pages into the table and advances lens between steps."""

    def __init__(self, k_pool: torch.Tensor, v_pool: torch.Tensor, table: torch.Tensor, lens: torch.Tensor):
        if not isinstance(k_pool, torch.Tensor) or k_pool.device.type != "cuda":
            raise _invalid("the paged KV cache lives on a CUDA device")
        dev = k_pool.device
        if k_pool.dtype not in (torch.bfloat16, torch.float16):
            raise GkvError(_lib.GKV_ERR_UNSUPPORTED, f"KV dtype {k_pool.dtype}: bf16 and f16 are built")
        _expect(k_pool, "k_pool", dev, k_pool.dtype, (None, PAGE_BLOCK_SIZE, None, None))
        _expect(v_pool, "v_pool", dev, k_pool.dtype, tuple(k_pool.shape))
        _expect(lens, "lens", dev, torch.int32, (None,))
        _expect(table, "table", dev, torch.int32, (lens.shape[0], None, 2), contiguous=False)
        stride = _table_stride(table)
        self.device = dev
        self.dtype = k_pool.dtype
        self.k_pool, self.v_pool, self.table, self.lens = k_pool, v_pool, table, lens
        self.batch, self.table_pages = table.shape[0], table.shape[1]
        self.pool_pages, _, self.n_kv_heads, self.head_dim = k_pool.shape
        pool = _lib.PoolDesc(k_pool.data_ptr(), v_pool.data_ptr(), self.pool_pages, self.n_kv_heads, self.head_dim,
                             _TORCH_TO_GKV[self.dtype])
        self.desc = _lib.Batch(pool, table.data_ptr(), lens.data_ptr(), stride, self.batch, self.table_pages, dev.index)
        check(lib().gkv_batch_prepare(dev.index))

    def check_device_errors(self) -> int:
        """The device's batch error word, read and cleared (synchronises): bit
        0 = a page id outside the pool was skipped, bit 2 = a length beyond
        its table row. 0 when clean."""
        f = C.c_uint32()
        st = lib().gkv_batch_check_errors(self.device.index, C.byref(f))
        if st not in (_lib.GKV_OK, _lib.GKV_ERR_DEVICE):
            check(st)
        return f.value


class _Bound:
    """An entry point with its arguments bound; ``run`` enqueues it."""

    def __init__(self, cache: PagedBatch):
        self.cache = cache
        self._device = cache.device.index
        self._home = torch.cuda.current_stream(self._device)  # its tensors are made on this stream
        self._home_handle = self._home.cuda_stream
        self._ordered = {self._home_handle}  # streams that have waited for it
        self._keep = [cache.k_pool, cache.v_pool, cache.table, cache.lens]

    def _hold(self, *tensors):
        self._keep += [t for t in tensors if t is not None]

    def _space(self, size: int) -> torch.Tensor:
        t = torch.empty(max(16, size), dtype=torch.uint8, device=self.cache.device)
        self._hold(t)
        return t

    def _bind(self, fn, *args, result):
        self._fn, self._args, self._result = fn, args, result

    def _order(self, stream, handle: int):
        """Make the first run on `stream` follow what the bind queued: workspace
        and outputs are new there, and earlier owners of their memory may be at
        work. A captured run cannot wait for a stream outside its capture; whoever
        captures has that one finished (torch.cuda.graph synchronises first)."""
        def capturing(s):
            with torch.cuda.stream(s):
                return torch.cuda.is_current_stream_capturing()
        if capturing(stream) == capturing(self._home):
            stream.wait_stream(self._home)
            self._ordered.add(handle)

    def run(self, stream=None) -> torch.Tensor:
        """Enqueue on `stream` (default: the current one); the tensor it fills."""
        handle = _current_stream(self._device) if stream is None else stream.cuda_stream
        if stream is not None or handle != self._home_handle:
            # Memory freed while this work is pending must not be handed out again on its own stream.
            s = stream if stream is not None else torch.cuda.current_stream(self._device)
            if handle not in self._ordered:
                self._order(s, handle)
            for t in self._keep:
                t.record_stream(s)
        status = self._fn(*self._args, handle)
        if status:
            check(status)
        return self._result


class BatchDecode(_Bound):
    """One decode step of a batch (gkv_batch_decode): ``q`` [B, Hq, D] and, to
    append, ``k_new`` and ``v_new`` [B, Hkv, D] (any strides with whole rows).
    ``run()`` returns ``out`` [B, Hq, D] (f32, f16 or bf16; q's type by
    default), softmax(scale q.k) v over each sequence's tokens, the new one
    included. ``lse`` (a [B, Hq] f32 tensor, or True for a new one) receives
    the natural log of the sum of exponentials. Rows of skipped sequences stay
    as they are: 0 and -inf in tensors made here.

    ``pages`` [B, Hkv, n] int32 restricts KV head h of sequence b to the
    listed logical pages (of :class:`PageSelect`); entries that are no page in
    use are skipped, and of each list only the first min(n, pages in use)
    entries count. ``weights_out`` [B, Hkv, W] f32, W >= 16 T, receives
    ``decay * weights + attention of the step's query heads`` per attended
    token, ``weights`` (may be the same tensor) being the total so far; its
    workspace takes 4 bytes per table slot and query head."""

    def __init__(self, cache: PagedBatch, q: torch.Tensor, k_new: Optional[torch.Tensor] = None,
                 v_new: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None,
                 scale: Optional[float] = None, lse=None, pages: Optional[torch.Tensor] = None,
                 weights: Optional[torch.Tensor] = None, weights_out: Optional[torch.Tensor] = None,
                 decay: float = 1.0):
        super().__init__(cache)
        dev, b, hkv, d = cache.device, cache.batch, cache.n_kv_heads, cache.head_dim
        _rows(q, "q", dev, cache.dtype, (b, None, d))
        hq = q.shape[1]
        if (k_new is None) != (v_new is None):
            raise _invalid("k_new and v_new come together")
        if k_new is not None:
            _rows(k_new, "k_new", dev, cache.dtype, (b, hkv, d))
            _rows(v_new, "v_new", dev, cache.dtype, (b, hkv, d))
        if out is None:
            out = torch.zeros((b, hq, d), dtype=cache.dtype, device=dev)  # skipped rows stay so
        if not isinstance(out, torch.Tensor) or out.dtype not in _TORCH_TO_GKV:
            raise GkvError(_lib.GKV_ERR_UNSUPPORTED, "out must be an f32, f16 or bf16 tensor")
        _expect(out, "out", dev, out.dtype, (b, hq, d))
        if lse is True:
            lse = torch.full((b, hq), -math.inf, dtype=torch.float32, device=dev)
        elif lse is False:
            lse = None
        if lse is not None:
            _expect(lse, "lse", dev, torch.float32, (b, hq))
        if pages is not None:
            _page_lists(pages, dev, b, hkv)
        if weights is not None and weights_out is None:
            raise _invalid("weights without weights_out")
        if weights_out is not None:
            _expect(weights_out, "weights_out", dev, torch.float32, (b, hkv, None))
        if weights is not None:
            _expect(weights, "weights", dev, torch.float32, tuple(weights_out.shape))
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        size = C.c_size_t()
        check(lib().gkv_batch_decode_workspace(C.byref(cache.desc), hq, int(weights_out is not None), C.byref(size)))
        space = self._space(size.value)
        k0, k1 = (k_new.stride(0), k_new.stride(1)) if k_new is not None else (0, 0)
        v0, v1 = (v_new.stride(0), v_new.stride(1)) if v_new is not None else (0, 0)
        self.args = _lib.BatchDecodeArgs(
            q.data_ptr(), q.stride(0), q.stride(1), ptr(k_new), ptr(v_new), k0, k1, v0, v1, out.data_ptr(), ptr(lse),
            ptr(pages), ptr(weights), ptr(weights_out), weights_out.shape[2] if weights_out is not None else 0,
            pages.shape[2] if pages is not None else 0, hq, _TORCH_TO_GKV[out.dtype],
            float(scale) if scale is not None else float(d) ** -0.5, float(decay), space.data_ptr(), space.numel())
        self._hold(q, k_new, v_new, out, lse, pages, weights, weights_out)
        self.out, self.lse, self.weights_out = out, lse, weights_out
        self._bind(lib().gkv_batch_decode, C.byref(cache.desc), C.byref(self.args), result=out)


class PageBounds(_Bound):
    """Key bounds of a batch's pages (gkv_batch_page_bounds) into ``bounds``
    [P, Hkv, 2, D] (min, max; the pool's type, indexed by K page id): every
    page that holds one of the tokens [start[b], lens[b] + extra), ``start``
    an int32 [B] tensor (None: from 0). After a decode step that appended,
    ``start=lens, extra=1`` refreshes the page each token went to; after an
    eviction, which moves rows between pages, take them all again. A page that
    sequences share must hold equally many tokens of each, as full pages do."""

    def __init__(self, cache: PagedBatch, bounds: torch.Tensor, start: Optional[torch.Tensor] = None, extra: int = 0):
        super().__init__(cache)
        _expect(bounds, "bounds", cache.device, cache.dtype, (cache.pool_pages, cache.n_kv_heads, 2, cache.head_dim))
        if start is not None:
            _expect(start, "start", cache.device, torch.int32, (cache.batch,))
        self._hold(bounds, start)
        self.bounds = bounds
        self._bind(lib().gkv_batch_page_bounds, C.byref(cache.desc), start.data_ptr() if start is not None else None,
                   _count(extra, "extra"), bounds.data_ptr(), result=bounds)


class PageSelect(_Bound):
    """Each KV head's ``n_pages`` best pages for ``q`` [B, Hq, D] by their
    ``bounds`` (gkv_batch_select_pages): the largest of sum_d max(q_d min_d,
    q_d max_d) over the head's queries, in 64 bits, equal ones by the lower
    page; the ``first`` first and ``last`` last pages in any case, pages with an
    id outside the pool behind all others. ``extra``: tokens about to be appended (1 before a decode step). ``run()`` returns
    ``pages`` [B, Hkv, n_pages] int32, rising, -1 behind the last."""

    def __init__(self, cache: PagedBatch, q: torch.Tensor, bounds: torch.Tensor, n_pages: int, *, first: int = 1,
                 last: int = 1, extra: int = 1, pages: Optional[torch.Tensor] = None):
        super().__init__(cache)
        dev, b, hkv, d = cache.device, cache.batch, cache.n_kv_heads, cache.head_dim
        _rows(q, "q", dev, cache.dtype, (b, None, d))
        _expect(bounds, "bounds", dev, cache.dtype, (cache.pool_pages, hkv, 2, d))
        n_pages = _count(n_pages, "n_pages")
        first, last, extra = _count(first, "first"), _count(last, "last"), _count(extra, "extra")
        if n_pages < 1:
            raise _invalid(f"n_pages {n_pages}")
        if pages is None:
            pages = torch.full((b, hkv, n_pages), -1, dtype=torch.int32, device=dev)
        _expect(pages, "pages", dev, torch.int32, (b, hkv, n_pages))
        size = C.c_size_t()
        check(lib().gkv_batch_select_workspace(C.byref(cache.desc), C.byref(size)))
        space = self._space(size.value)
        self.args = _lib.BatchSelectArgs(q.data_ptr(), q.stride(0), q.stride(1), bounds.data_ptr(), pages.data_ptr(),
                                         n_pages, first, last, extra, q.shape[1], space.data_ptr(), space.numel())
        self._hold(q, bounds, pages)
        self.pages = pages
        self._bind(lib().gkv_batch_select_pages, C.byref(cache.desc), C.byref(self.args), result=pages)


class CacheEvict(_Bound):
    """Cut every sequence back to ``keep`` tokens per KV head
    (gkv_batch_evict): first the ``recent`` most recent, then those of the
    largest ``weights`` [B, Hkv, W] f32 (NaN first, equal ones by the lower
    slot). Kept rows behind the new length move into the slots that became
    free below it, in place, with their weight and position.

    ``seen`` [B] int32: tokens the sequence has had in all. ``tracked`` [B]
    int32 and ``positions`` [B, Hkv, W] int32: the slots kept by the eviction
    before, and the positions of the tokens they hold (None: first eviction,
    slot t holds token seen - lens + t). ``run()`` returns ``lens_out`` [B],
    which is the next eviction's ``tracked``; ``weights_out`` and
    ``positions_out`` hold the kept slots' values. Outputs may be the inputs
    (``lens_out`` may be the batch's lens). Up to 65535 sequences x KV heads."""

    def __init__(self, cache: PagedBatch, weights: torch.Tensor, seen: torch.Tensor, *, keep: int, recent: int = 0,
                 tracked: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                 weights_out: Optional[torch.Tensor] = None, positions_out: Optional[torch.Tensor] = None,
                 lens_out: Optional[torch.Tensor] = None):
        super().__init__(cache)
        dev, b, hkv = cache.device, cache.batch, cache.n_kv_heads
        _expect(weights, "weights", dev, torch.float32, (b, hkv, None))
        shape = tuple(weights.shape)
        _expect(seen, "seen", dev, torch.int32, (b,))
        if tracked is not None:
            _expect(tracked, "tracked", dev, torch.int32, (b,))
            if positions is None:
                raise _invalid("tracked without positions")
        if positions is not None:
            _expect(positions, "positions", dev, torch.int32, shape)
        weights_out = weights if weights_out is None else weights_out
        if positions_out is None:
            positions_out = positions if positions is not None else torch.zeros(shape, dtype=torch.int32, device=dev)
        lens_out = torch.zeros_like(cache.lens) if lens_out is None else lens_out
        _expect(weights_out, "weights_out", dev, torch.float32, shape)
        _expect(positions_out, "positions_out", dev, torch.int32, shape)
        _expect(lens_out, "lens_out", dev, torch.int32, (b,))
        size = C.c_size_t()
        check(lib().gkv_batch_evict_workspace(C.byref(cache.desc), C.byref(size)))
        space = self._space(size.value)
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        self.args = _lib.BatchEvictArgs(weights.data_ptr(), weights_out.data_ptr(), ptr(positions),
                                        positions_out.data_ptr(), seen.data_ptr(), ptr(tracked), lens_out.data_ptr(),
                                        shape[2], _count(keep, "keep"), _count(recent, "recent"), space.data_ptr(), space.numel())
        self._hold(weights, weights_out, positions, positions_out, seen, tracked, lens_out)
        self.lens_out, self.weights_out, self.positions_out = lens_out, weights_out, positions_out
        self._bind(lib().gkv_batch_evict, C.byref(cache.desc), C.byref(self.args), result=lens_out)


def batch_decode(cache: PagedBatch, q, k_new=None, v_new=None, *, stream=None, **options) -> torch.Tensor:
    """:class:`BatchDecode`, bound and run once on `stream` (default: the current one)."""
    with torch.cuda.stream(stream):
        return BatchDecode(cache, q, k_new, v_new, **options).run(stream)


def page_bounds(cache: PagedBatch, bounds: Optional[torch.Tensor] = None, start=None, extra: int = 0, *,
                stream=None) -> torch.Tensor:
    """:class:`PageBounds`, bound and run once; without ``bounds`` into a new
    zero-filled tensor."""
    with torch.cuda.stream(stream):
        if bounds is None:
            bounds = torch.zeros((cache.pool_pages, cache.n_kv_heads, 2, cache.head_dim), dtype=cache.dtype,
                                 device=cache.device)
        return PageBounds(cache, bounds, start, extra).run(stream)


def select_pages(cache: PagedBatch, q, bounds, n_pages: int, *, stream=None, **options) -> torch.Tensor:
    """:class:`PageSelect`, bound and run once."""
    with torch.cuda.stream(stream):
        return PageSelect(cache, q, bounds, n_pages, **options).run(stream)


def evict_tokens(cache: PagedBatch, weights, seen, *, keep: int, stream=None, **options):
    """:class:`CacheEvict`, bound and run once: (lens_out, weights_out, positions_out)."""
    with torch.cuda.stream(stream):
        op = CacheEvict(cache, weights, seen, keep=keep, **options)
        op.run(stream)
        return op.lens_out, op.weights_out, op.positions_out
