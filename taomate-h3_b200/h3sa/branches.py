"""Branches: several continuations of one stream over the pages of one clean history.

A guidance pair, candidate takes, drafted tokens or several viewers continue the same history.
Here that history is held once: a ledger of page tables, lengths and reference counts describes
which pages each sequence holds (``fork_pages``, ``free_pages``, ``compact_pages``), and
``shared_prefix_attention`` attends from all sequences at once and reads the shared pages once
for all of them. The ledger lives in device memory and no call here waits for the host:

* ``table`` int32 ``[sequences, width]``: page of each 128-row block of a sequence, -1 after the
  last page held;
* ``lengths`` int32 ``[sequences]``: rows of each sequence;
* ``refs`` int32 ``[pages]``: table entries that hold each page, 0 for a free one.

Each operation returns the new ledger and leaves the one it was given as it was. Failures that
only the device can see (too few free pages, an index out of range) are OR-ed into
``device_error`` as the ``DEVERR_*`` bits of ``h3sa._lib``; without one they go unreported. The
reference holds one history per stream and has no counterpart.

A ledger owns the pages that it describes. ``PagedLayerKV`` keeps its own lists of pages on the host
and does not learn of forks or moves: once a ledger describes its pools, such a cache must not be
written, grown or committed to, or both would hand out the same pages. e4m3 pools have one K and one
V scale per KV head, so the e4m3 history of a streaming cache, with scales per commit, is none.
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import Sequence, Union

import torch

from ._lib import LIB, Pools, check
from .kernels import HEAD_DIM, PAGE_ROWS

PoolTensors = Union[torch.Tensor, Sequence[torch.Tensor]]

# A call of a few rows takes the device about ten microseconds, so the host side counts: entry
# points are bound once, conditions are tested inline and messages built only on failure.
_FORK, _COMPACT, _FREE = LIB.h3sa_fork_pages, LIB.h3sa_compact_pages, LIB.h3sa_free_pages
_ATTEND, _ATTEND_WORK = LIB.h3sa_shared_prefix_attention, LIB.h3sa_shared_prefix_workspace
_ATTEND_TREE, _TREE_WORK = LIB.h3sa_tree_attention, LIB.h3sa_tree_workspace
_PAGES_WORK = LIB.h3sa_pages_workspace
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_I32, _F32, _BF16, _E4M3 = torch.int32, torch.float32, torch.bfloat16, torch.float8_e4m3fn
_empty_like = torch.empty_like


def _bad(t: torch.Tensor, device: torch.device, dtype: torch.dtype, shape: tuple[int, ...]) -> bool:
    return t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous()


def _refuse(what: str, name: str, device: torch.device, dtype: torch.dtype, shape: tuple[int, ...]) -> None:
    raise RuntimeError(f"{what}: {name} must be contiguous {dtype} {list(shape)} on {device}")


def _error_word(what: str, device: torch.device, word: torch.Tensor | None) -> int | None:
    if word is None:
        return None
    if word.device != device or word.dtype is not _I32 or word.numel() < 1:
        raise RuntimeError(f"{what}: device_error must be an int32 tensor on {device}")
    return word.data_ptr()


_CURRENT = contextlib.nullcontext()


def _on(stream: torch.cuda.Stream | None):
    """Results and workspaces are allocated on the stream that uses them; the current one needs no switch."""

    return _CURRENT if stream is None else torch.cuda.stream(stream)


def _handle(stream: torch.cuda.Stream | None, device: torch.device) -> int:
    """The stream to launch on, which is the current device's, as the tensors must be."""

    if device.index != _current_device() or (stream is not None and stream.device != device):
        raise RuntimeError(f"h3sa kernels run on the current device (cuda:{_current_device()}): the tensors are on "
                           f"{device}" + ("" if stream is None else f", the stream on {stream.device}"))
    return _raw_stream(device.index) if stream is None else stream.cuda_stream


def _pools(what: str, pools: PoolTensors, pages: int | None, device: torch.device) -> Pools:
    """The pool tensors of a ledger: one tensor ``[count, heads, pages*128, d]`` or a sequence of
    ``[heads, pages*128, d]``, all of one shape and dtype, of the ledger's pages where a call has them. The
    returned struct keeps its address list alive."""

    p = Pools()
    if isinstance(pools, torch.Tensor):
        if pools.ndim != 4:
            raise RuntimeError(f"{what}: stacked pools must be [count, heads, pages*128, d]")
        p.count, heads, rows, d = pools.shape
        size = pools.element_size()
        p.base, p.stride = pools.data_ptr(), pools.stride(0) * size
        if pools.device != device or not (pools.is_contiguous() or p.count == 0 or pools[0].is_contiguous()):
            raise RuntimeError(f"{what}: pool tensors must be contiguous on {device}")
    else:
        if len(pools) == 0:
            raise RuntimeError(f"{what}: no pool tensors")
        first = pools[0]
        shape, dtype, size = first.shape, first.dtype, first.element_size()
        if len(shape) != 3:
            raise RuntimeError(f"{what}: pool tensors must be [heads, pages*{PAGE_ROWS}, d]")
        heads, rows, d = shape
        for t in pools:
            if t.device != device or t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
                raise RuntimeError(f"{what}: pool tensors must be contiguous on {device}, of one "
                                   "shape and dtype")
        address = (ctypes.c_void_p * len(pools))(*[t.data_ptr() for t in pools])
        p.list, p.count = ctypes.addressof(address), len(pools)
        p._address = address
    if pages is None:
        pages = rows // PAGE_ROWS
        if heads == 0 or rows == 0 or rows % PAGE_ROWS:
            raise RuntimeError(f"{what}: pool tensors must be [heads, pages*{PAGE_ROWS}, d]")
    if heads == 0 or rows != pages * PAGE_ROWS:
        raise RuntimeError(f"{what}: pool tensors must be [heads, {pages}*{PAGE_ROWS}, d] for {pages} "
                           "reference counts")
    p.heads, p.pages, p.row_bytes = heads, pages, d * size
    return p


def _ledger(what: str, table: torch.Tensor, refs: torch.Tensor) -> tuple[torch.device, int, int, int]:
    if not table.is_cuda:
        raise RuntimeError("h3sa kernels require CUDA tensors")
    if table.ndim != 2 or refs.ndim != 1:
        raise RuntimeError(f"{what}: table must be [sequences, width] and refs [pages]")
    device, (sequences, width), (pages,) = table.device, table.shape, refs.shape
    if _bad(table, device, _I32, (sequences, width)):
        _refuse(what, "table", device, _I32, (sequences, width))
    if _bad(refs, device, _I32, (pages,)):
        _refuse(what, "refs", device, _I32, (pages,))
    return device, sequences, width, pages


def fork_pages(pools: PoolTensors, table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
               parents: torch.Tensor, *, reserve_rows: int = 0, private: bool = False,
               device_error: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None,
               ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """New branches: child c continues sequence ``parents[c]`` (int32; negative: starts empty).

    A child holds its parent's whole pages together with it and a fresh copy of the rows of the
    parent's last, partial page, so it can be written to from its own length on;
    ``private=True`` copies all of the parent's pages instead. ``reserve_rows`` more rows get
    fresh pages. Fresh pages are the lowest free ones, in child order. Rows are copied in every
    pool tensor. Returns ``(table [children, width], lengths [children], refs)`` of the children;
    the pools' and the parents' own entries stay as they are. If the device finds that it cannot
    fork all of them (``device_error``), every child comes out empty and ``refs`` unchanged.
    """

    what = "fork_pages"
    device, sequences, width, pages = _ledger(what, table, refs)
    if parents.ndim != 1:
        raise RuntimeError(f"{what}: parents must be [children]")
    children = parents.shape[0]
    if _bad(lengths, device, _I32, (sequences,)):
        _refuse(what, "lengths", device, _I32, (sequences,))
    if _bad(parents, device, _I32, (children,)):
        _refuse(what, "parents", device, _I32, (children,))
    error = _error_word(what, device, device_error)
    if not 0 <= reserve_rows < 1 << 31:
        raise ValueError(f"{what}: reserve_rows must not be negative or past 32 bits")
    p = _pools(what, pools, pages, device)
    with _on(stream):
        child_table = table.new_empty((children, width))
        child_lengths = _empty_like(parents)
        refs_out = _empty_like(refs)
        work = refs.new_empty(_PAGES_WORK(pages, children) // 4)
    code = _FORK(p, table.data_ptr(), sequences, width, lengths.data_ptr(), refs.data_ptr(),
                 parents.data_ptr(), children, int(reserve_rows), 1 if private else 0,
                 child_table.data_ptr(), child_lengths.data_ptr(), refs_out.data_ptr(),
                 work.data_ptr(), error, _handle(stream, device))
    if code:
        check("h3sa_fork_pages", code)
    return child_table, child_lengths, refs_out


def compact_pages(pools: PoolTensors, table: torch.Tensor, refs: torch.Tensor, *,
                  device_error: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None,
                  ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Move the n pages in use to the front of the pools: the i-th free page below n receives the
    i-th page in use at or past n. ``table`` must hold every reference that ``refs`` counts.
    Returns the renumbered ``(table, refs)`` and n as an int32 tensor ``[1]``."""

    what = "compact_pages"
    device, sequences, width, pages = _ledger(what, table, refs)
    error = _error_word(what, device, device_error)
    p = _pools(what, pools, pages, device)
    with _on(stream):
        table_out, refs_out = _empty_like(table), _empty_like(refs)
        live = refs.new_empty(1)
        work = refs.new_empty(_PAGES_WORK(pages, 0) // 4)
    code = _COMPACT(p, table.data_ptr(), sequences, width, refs.data_ptr(), table_out.data_ptr(),
                    refs_out.data_ptr(), live.data_ptr(), work.data_ptr(), error,
                    _handle(stream, device))
    if code:
        check("h3sa_compact_pages", code)
    return table_out, refs_out, live


def free_pages(table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
               release: torch.Tensor, *, device_error: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None,
               ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """End the sequences with ``release[s]`` (bool ``[sequences]``): their pages lose one reference
    each, their table rows become -1 and their lengths 0. Returns ``(table, lengths, refs)``."""

    what = "free_pages"
    device, sequences, width, pages = _ledger(what, table, refs)
    if _bad(lengths, device, _I32, (sequences,)):
        _refuse(what, "lengths", device, _I32, (sequences,))
    if _bad(release, device, torch.bool, (sequences,)):
        _refuse(what, "release", device, torch.bool, (sequences,))
    error = _error_word(what, device, device_error)
    with _on(stream):
        table_out, lengths_out, refs_out = _empty_like(table), _empty_like(lengths), _empty_like(refs)
    code = _FREE(table.data_ptr(), sequences, width, lengths.data_ptr(), refs.data_ptr(), pages,
                 release.data_ptr(), table_out.data_ptr(), lengths_out.data_ptr(),
                 refs_out.data_ptr(), error, _handle(stream, device))
    if code:
        check("h3sa_free_pages", code)
    return table_out, lengths_out, refs_out


def shared_prefix_attention(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor,
                            table: torch.Tensor, lengths: torch.Tensor, shared_rows: int,
                            softmax_scale: float, *, causal: bool = False,
                            k_scale: torch.Tensor | None = None,
                            v_scale: torch.Tensor | None = None,
                            out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                            device_error: torch.Tensor | None = None,
                            stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Attention of the new rows of every sequence, the shared history read once for all.

    ``query``: bf16 ``[sequences, rows, heads, 128]`` (any strides with contiguous, 16-byte
    aligned rows). Pools ``[kv_heads, pages*128, 128]`` bf16, or e4m3 with fp32 per-head
    ``k_scale`` / ``v_scale`` (not negative); query head h reads KV head ``h // (heads // kv_heads)``. Row i of
    sequence b sees its first ``lengths[b]`` keys, with ``causal`` only those up to itself, the
    query rows being the sequence's last ones (their K/V already written). The first
    ``shared_rows`` rows (a multiple of 128) are the same pages in the table rows of all
    sequences that reach that far, as ``fork_pages`` leaves them; shorter sequences are read by
    themselves. Rows that see nothing come out zero; an infinity or NaN in V of a sequence's own rows
    makes its outputs in that column infinite or NaN, ``causal`` or not. ``out``: optional contiguous bf16 result tensor; ``lse``: optional fp32
    ``[sequences, rows, heads]`` that receives the log-sum-exp (-inf for such rows). Neither may
    overlap ``query``.
    """

    return _attend("shared_prefix_attention", None, None, query, key_pool, value_pool, table, lengths, shared_rows,
                   softmax_scale, causal, k_scale, v_scale, out, lse, device_error, stream)


def _attend(what: str, masks: torch.Tensor | None, counts: int | None, query: torch.Tensor, key_pool: torch.Tensor,
            value_pool: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, shared_rows: int, softmax_scale: float,
            causal: bool, k_scale: torch.Tensor | None, v_scale: torch.Tensor | None, out: torch.Tensor | None,
            lse: torch.Tensor | None, device_error: torch.Tensor | None,
            stream: torch.cuda.Stream | None) -> torch.Tensor:
    """``shared_prefix_attention``, and with ``masks`` ``h3sa.drafts.tree_attention`` (counts: an address)."""

    if not query.is_cuda:
        raise RuntimeError("h3sa kernels require CUDA tensors")
    device, shape, pool = query.device, query.shape, key_pool.shape
    if len(shape) != 4 or shape[3] != HEAD_DIM or query.dtype is not _BF16:
        raise RuntimeError(f"{what}: query must be bf16 [sequences, rows, heads, {HEAD_DIM}]")
    batch, rows, heads, _ = shape
    strides = query.stride()
    if strides[3] != 1 or (strides[0] | strides[1] | strides[2]) % 8 or query.data_ptr() % 16:
        raise RuntimeError(f"{what}: query rows must be contiguous and 16-byte aligned")
    kind = key_pool.dtype
    if (len(pool) != 3 or pool[1] % PAGE_ROWS or pool[2] != HEAD_DIM or _bad(key_pool, device, kind, pool)
            or _bad(value_pool, device, kind, pool)):
        raise RuntimeError(f"{what}: KV pools must be contiguous [kv_heads, pages*{PAGE_ROWS}, "
                           f"{HEAD_DIM}] of one dtype on {device}")
    kv_heads, pool_rows, _ = pool
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise RuntimeError(f"{what}: {heads} query heads are no multiple of {kv_heads} KV heads")
    e4m3 = kind is _E4M3
    if e4m3:
        if k_scale is None or v_scale is None:
            raise RuntimeError(f"{what}: e4m3 pools need k_scale and v_scale")
        if _bad(k_scale, device, _F32, (kv_heads,)) or _bad(v_scale, device, _F32, (kv_heads,)):
            _refuse(what, "k_scale and v_scale", device, _F32, (kv_heads,))
    elif kind is not _BF16:
        raise RuntimeError(f"{what}: KV pools must be bf16 or e4m3")
    elif k_scale is not None or v_scale is not None:
        raise RuntimeError(f"{what}: bf16 pools take no scales")
    if table.ndim != 2:
        raise RuntimeError(f"{what}: table must be [sequences, width]")
    width = table.shape[1]
    if _bad(table, device, _I32, (batch, width)):
        _refuse(what, "table", device, _I32, (batch, width))
    if _bad(lengths, device, _I32, (batch,)):
        _refuse(what, "lengths", device, _I32, (batch,))
    if lse is not None and _bad(lse, device, _F32, (batch, rows, heads)):
        _refuse(what, "lse", device, _F32, (batch, rows, heads))
    if not 0 <= shared_rows <= width * PAGE_ROWS:
        raise RuntimeError(f"{what}: {shared_rows} shared rows are not whole pages of a table of {width} "
                           "entries")
    error = _error_word(what, device, device_error)
    need = (max(16, _ATTEND_WORK(batch, rows, heads, kv_heads, shared_rows)) if masks is None else
            _TREE_WORK(batch, rows, heads, kv_heads, shared_rows, width, 1 if e4m3 else 0))
    if out is not None and _bad(out, device, _BF16, query.shape):
        _refuse(what, "out", device, _BF16, query.shape)
    with _on(stream):
        if out is None:
            out = (_empty_like(query) if query.is_contiguous() else
                   query.new_empty(shape))
        work = lengths.new_empty(need // 4) if need else None
    args = (query.data_ptr(), strides[0], strides[1], strides[2], out.data_ptr(),
            None if lse is None else lse.data_ptr(), batch, rows, heads, kv_heads,
            key_pool.data_ptr(), value_pool.data_ptr(), pool_rows // PAGE_ROWS, 1 if e4m3 else 0,
            k_scale.data_ptr() if e4m3 else None, v_scale.data_ptr() if e4m3 else None,
            table.data_ptr(), width, lengths.data_ptr())
    if masks is None:
        code = _ATTEND(*args, shared_rows, 1 if causal else 0, softmax_scale, work.data_ptr(), need, error,
                       _handle(stream, device))
    else:
        code = _ATTEND_TREE(*args, masks.data_ptr(), counts, shared_rows, softmax_scale,
                            None if work is None else work.data_ptr(), need, error, _handle(stream, device))
    if code:
        check(f"h3sa_{what}", code)
    return out


__all__ = ["compact_pages", "fork_pages", "free_pages", "shared_prefix_attention"]
