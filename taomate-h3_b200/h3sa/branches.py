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
``device_error`` as the ``DEVERR_*`` bits of ``h3sa._lib``. The reference holds one history per
stream and has no counterpart.
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import Sequence, Union

import torch

from ._lib import LIB, Pools, call, ptr, stream_handle
from .kernels import HEAD_DIM, PAGE_ROWS

PoolTensors = Union[torch.Tensor, Sequence[torch.Tensor]]


def _on(stream: torch.cuda.Stream | None):
    """Results and workspaces are allocated on the stream that uses them."""

    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _check(what: str, device: torch.device, dtype: torch.dtype,
           tensors: Sequence[tuple[str, torch.Tensor, tuple[int, ...]]]) -> None:
    for name, t, shape in tensors:
        if t.device != device or t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
            raise RuntimeError(f"{what}: {name} must be contiguous {dtype} {list(shape)} on {device}")


def _check_error_word(what: str, device: torch.device, word: torch.Tensor | None) -> None:
    if word is not None and (word.device != device or word.dtype != torch.int32 or word.numel() < 1):
        raise RuntimeError(f"{what}: device_error must be an int32 tensor on {device}")


def _pools(what: str, pools: PoolTensors, pages: int, device: torch.device) -> Pools:
    """The pool tensors of a ledger: one tensor ``[count, heads, pages*128, d]`` or a sequence of
    ``[heads, pages*128, d]``, all of one shape and dtype. The returned struct keeps its address
    list alive."""

    p = Pools()
    if isinstance(pools, torch.Tensor):
        if pools.ndim != 4:
            raise RuntimeError(f"{what}: stacked pools must be [count, heads, pages*128, d]")
        first = pools
        shape = tuple(pools.shape[1:])
        p.base, p.count = pools.data_ptr(), pools.shape[0]
        p.stride = pools.stride(0) * pools.element_size()
        if pools.device != device or not (pools.is_contiguous() or pools[0].is_contiguous()):
            raise RuntimeError(f"{what}: pool tensors must be contiguous on {device}")
    else:
        if len(pools) == 0:
            raise RuntimeError(f"{what}: no pool tensors")
        first = pools[0]
        shape = tuple(first.shape)
        dtype = first.dtype
        for t in pools:
            if t.device != device or t.dtype != dtype or t.shape != first.shape or not t.is_contiguous():
                raise RuntimeError(f"{what}: pool tensors must be contiguous on {device}, of one "
                                   "shape and dtype")
        address = (ctypes.c_void_p * len(pools))(*[t.data_ptr() for t in pools])
        p.list, p.count = ctypes.addressof(address), len(pools)
        p._address = address
    if len(shape) != 3 or shape[0] == 0 or shape[1] != pages * PAGE_ROWS:
        raise RuntimeError(f"{what}: pool tensors must be [heads, {pages}*{PAGE_ROWS}, d] for {pages} "
                           "reference counts")
    p.heads, p.pages = shape[0], pages
    p.row_bytes = shape[2] * first.element_size()
    return p


def _ledger(what: str, table: torch.Tensor, refs: torch.Tensor) -> tuple[torch.device, int, int, int]:
    if not table.is_cuda:
        raise RuntimeError("h3sa kernels require CUDA tensors")
    if table.ndim != 2 or refs.ndim != 1:
        raise RuntimeError(f"{what}: table must be [sequences, width] and refs [pages]")
    sequences, width = table.shape
    _check(what, table.device, torch.int32, (("table", table, (sequences, width)),
                                             ("refs", refs, (refs.shape[0],))))
    return table.device, sequences, width, refs.shape[0]


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

    device, sequences, width, pages = _ledger("fork_pages", table, refs)
    if parents.ndim != 1:
        raise RuntimeError("fork_pages: parents must be [children]")
    children = parents.shape[0]
    _check("fork_pages", device, torch.int32, (("lengths", lengths, (sequences,)),
                                               ("parents", parents, (children,))))
    _check_error_word("fork_pages", device, device_error)
    if reserve_rows < 0:
        raise ValueError("fork_pages: reserve_rows must not be negative")
    p = _pools("fork_pages", pools, pages, device)
    with _on(stream):
        child_table = torch.empty((children, width), dtype=torch.int32, device=device)
        child_lengths = torch.empty(children, dtype=torch.int32, device=device)
        refs_out = torch.empty_like(refs)
        work = torch.empty(LIB.h3sa_pages_workspace(pages, children), dtype=torch.uint8, device=device)
    call("h3sa_fork_pages", p, ptr(table), sequences, width, ptr(lengths), ptr(refs), ptr(parents),
         children, int(reserve_rows), 1 if private else 0, ptr(child_table), ptr(child_lengths),
         ptr(refs_out), ptr(work), ptr(device_error), stream_handle(stream))
    return child_table, child_lengths, refs_out


def compact_pages(pools: PoolTensors, table: torch.Tensor, refs: torch.Tensor, *,
                  device_error: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None,
                  ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Move the n pages in use to the front of the pools: the i-th free page below n receives the
    i-th page in use at or past n. ``table`` must hold every reference that ``refs`` counts.
    Returns the renumbered ``(table, refs)`` and n as an int32 tensor ``[1]``."""

    device, sequences, width, pages = _ledger("compact_pages", table, refs)
    _check_error_word("compact_pages", device, device_error)
    p = _pools("compact_pages", pools, pages, device)
    with _on(stream):
        table_out, refs_out = torch.empty_like(table), torch.empty_like(refs)
        live = torch.empty(1, dtype=torch.int32, device=device)
        work = torch.empty(LIB.h3sa_pages_workspace(pages, 0), dtype=torch.uint8, device=device)
    call("h3sa_compact_pages", p, ptr(table), sequences, width, ptr(refs), ptr(table_out),
         ptr(refs_out), ptr(live), ptr(work), ptr(device_error), stream_handle(stream))
    return table_out, refs_out, live


def free_pages(table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
               release: torch.Tensor, *, device_error: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None,
               ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """End the sequences with ``release[s]`` (bool ``[sequences]``): their pages lose one reference
    each, their table rows become -1 and their lengths 0. Returns ``(table, lengths, refs)``."""

    device, sequences, width, pages = _ledger("free_pages", table, refs)
    _check("free_pages", device, torch.int32, (("lengths", lengths, (sequences,)),))
    _check("free_pages", device, torch.bool, (("release", release, (sequences,)),))
    _check_error_word("free_pages", device, device_error)
    with _on(stream):
        table_out, lengths_out = torch.empty_like(table), torch.empty_like(lengths)
        refs_out = torch.empty_like(refs)
    call("h3sa_free_pages", ptr(table), sequences, width, ptr(lengths), ptr(refs), pages,
         ptr(release), ptr(table_out), ptr(lengths_out), ptr(refs_out), ptr(device_error),
         stream_handle(stream))
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
    ``k_scale`` / ``v_scale``; query head h reads KV head ``h // (heads // kv_heads)``. Row i of
    sequence b sees its first ``lengths[b]`` keys, with ``causal`` only those up to itself, the
    query rows being the sequence's last ones (their K/V already written). The first
    ``shared_rows`` rows (a multiple of 128) are the same pages in the table rows of all
    sequences that reach that far, as ``fork_pages`` leaves them. Rows that see nothing come out
    zero. ``out``: optional contiguous bf16 result tensor; ``lse``: optional fp32
    ``[sequences, rows, heads]`` that receives the log-sum-exp (-inf for such rows).
    """

    what = "shared_prefix_attention"
    if not query.is_cuda:
        raise RuntimeError("h3sa kernels require CUDA tensors")
    device = query.device
    if query.ndim != 4 or query.dtype != torch.bfloat16 or query.shape[3] != HEAD_DIM:
        raise RuntimeError(f"{what}: query must be bf16 [sequences, rows, heads, {HEAD_DIM}]")
    batch, rows, heads, _ = query.shape
    strides = query.stride()
    if strides[3] != 1 or strides[0] % 8 or strides[1] % 8 or strides[2] % 8 or query.data_ptr() % 16:
        raise RuntimeError(f"{what}: query rows must be contiguous and 16-byte aligned")
    if (key_pool.ndim != 3 or key_pool.shape != value_pool.shape or key_pool.shape[2] != HEAD_DIM
            or key_pool.shape[1] % PAGE_ROWS or key_pool.dtype != value_pool.dtype
            or not key_pool.is_contiguous() or not value_pool.is_contiguous()
            or key_pool.device != device or value_pool.device != device):
        raise RuntimeError(f"{what}: KV pools must be contiguous [kv_heads, pages*{PAGE_ROWS}, "
                           f"{HEAD_DIM}] of one dtype on {device}")
    kv_heads, pool_rows, _ = key_pool.shape
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise RuntimeError(f"{what}: {heads} query heads are no multiple of {kv_heads} KV heads")
    e4m3 = key_pool.dtype == torch.float8_e4m3fn
    if e4m3:
        if k_scale is None or v_scale is None:
            raise RuntimeError(f"{what}: e4m3 pools need k_scale and v_scale")
        _check(what, device, torch.float32, (("k_scale", k_scale, (kv_heads,)),
                                             ("v_scale", v_scale, (kv_heads,))))
    elif key_pool.dtype != torch.bfloat16:
        raise RuntimeError(f"{what}: KV pools must be bf16 or e4m3")
    elif k_scale is not None or v_scale is not None:
        raise RuntimeError(f"{what}: bf16 pools take no scales")
    if table.ndim != 2:
        raise RuntimeError(f"{what}: table must be [sequences, width]")
    width = table.shape[1]
    _check(what, device, torch.int32, (("table", table, (batch, width)),
                                       ("lengths", lengths, (batch,))))
    if out is not None:
        _check(what, device, torch.bfloat16, (("out", out, (batch, rows, heads, HEAD_DIM)),))
    if lse is not None:
        _check(what, device, torch.float32, (("lse", lse, (batch, rows, heads)),))
    _check_error_word(what, device, device_error)
    need = LIB.h3sa_shared_prefix_workspace(batch, rows, heads, kv_heads, shared_rows)
    with _on(stream):
        if out is None:
            out = torch.empty((batch, rows, heads, HEAD_DIM), dtype=torch.bfloat16, device=device)
        work = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
    call("h3sa_shared_prefix_attention", ptr(query), (ctypes.c_int64 * 3)(*strides[:3]), ptr(out),
         ptr(lse), batch, rows, heads, kv_heads, ptr(key_pool), ptr(value_pool),
         pool_rows // PAGE_ROWS, 1 if e4m3 else 0, ptr(k_scale), ptr(v_scale), ptr(table), width,
         ptr(lengths), int(shared_rows), 1 if causal else 0, float(softmax_scale), ptr(work),
         work.numel(), ptr(device_error), stream_handle(stream))
    return out


__all__ = ["compact_pages", "fork_pages", "free_pages", "shared_prefix_attention"]
