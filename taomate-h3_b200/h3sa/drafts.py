"""Drafted trees: rows proposed behind the sequences of a ledger, verified together, one path of them kept.

A step, over the pages that ``h3sa.branches`` keeps books of:

* ``draft_tree``: the ancestors and positions of every drafted row, once for all layers;
* ``append_rows``: the rows' keys and values to the pages behind ``lengths``, keys (and queries) rotated on
  the way; prompts and single tokens alike;
* ``tree_attention``: each drafted row attends to the history and its own ancestors;
* ``keep_rows``: the rows of one accepted path become history, in every layer.

Row i of a sequence's tree is row ``lengths + i`` of its pages, which the sequence must hold to itself
(``fork_pages(..., reserve_rows=...)``), and is no part of ``lengths`` until it is kept. ``counts`` (int32
``[sequences]``) says how many rows of a sequence are nodes, all without it. No call waits for the host;
failures that only the device can see are OR-ed into ``device_error``, as in ``h3sa.branches``.
"""

from __future__ import annotations

import torch

from ._lib import LIB, Heads, check
from .branches import _BF16, _E4M3, _F32, _I32, PoolTensors, _attend, _bad, _error_word, _handle, _on, _pools, _refuse
from .kernels import HEAD_DIM, PAGE_ROWS
from .rotary import _rotary

_TREE, _APPEND, _KEEP = LIB.h3sa_draft_tree, LIB.h3sa_append_rows, LIB.h3sa_keep_rows
_empty_like = torch.empty_like


def _counts(what: str, counts: torch.Tensor | None, device: torch.device, batch: int) -> int | None:
    if counts is None:
        return None
    if _bad(counts, device, _I32, (batch,)):
        _refuse(what, "counts", device, _I32, (batch,))
    return counts.data_ptr()


def draft_tree(parents: torch.Tensor, lengths: torch.Tensor, *, counts: torch.Tensor | None = None,
               device_error: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None,
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """Ancestor bits and positions of trees: ``parents`` int32 ``[sequences, nodes]`` (up to 65535 and 1024), each a
    row in front of its own, or -1 for a root. Returns ``masks`` int32 ``[sequences, nodes, ceil(nodes / 32)]``, whose
    bit n % 32 of word n // 32 says whether node n is the row itself or above it, and ``positions`` int32
    ``[sequences, nodes]``, ``lengths`` plus the row's depth. Rows behind ``counts`` get zeros. A parent that is
    neither makes its row a root (``device_error``)."""

    what = "draft_tree"
    if not parents.is_cuda:
        raise RuntimeError("h3sa kernels require CUDA tensors")
    if parents.ndim != 2:
        raise RuntimeError(f"{what}: parents must be [sequences, nodes]")
    device, (batch, nodes) = parents.device, parents.shape
    if _bad(parents, device, _I32, (batch, nodes)):
        _refuse(what, "parents", device, _I32, (batch, nodes))
    if _bad(lengths, device, _I32, (batch,)):
        _refuse(what, "lengths", device, _I32, (batch,))
    live = _counts(what, counts, device, batch)
    error = _error_word(what, device, device_error)
    handle = _handle(stream, device)
    with _on(stream):
        masks, positions = parents.new_empty((batch, nodes, (nodes + 31) // 32)), _empty_like(parents)
    code = _TREE(parents.data_ptr(), batch, nodes, lengths.data_ptr(), live, masks.data_ptr(), positions.data_ptr(), error,
                 handle)
    if code:
        check("h3sa_draft_tree", code)
    return masks, positions


def append_rows(key: torch.Tensor, value: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor,
                table: torch.Tensor, lengths: torch.Tensor, *, counts: torch.Tensor | None = None,
                positions: torch.Tensor | None = None, frequencies: torch.Tensor | None = None,
                interleaved: bool = False, factor: float = 1.0, query: torch.Tensor | None = None,
                query_out: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                v_scale: torch.Tensor | None = None, device_error: torch.Tensor | None = None,
                stream: torch.cuda.Stream | None = None) -> torch.Tensor | None:
    """New rows to the pages of their sequences: row i < ``counts[b]`` of ``key`` and ``value`` (bf16 ``[sequences, rows,
    kv_heads, 128]``, any strides with contiguous rows) becomes row ``lengths[b] + i``; ``lengths`` stay.

    With ``frequencies`` (``h3sa.rotary``) keys are rotated on the way, and so is ``query`` (bf16 ``[sequences, rows,
    heads, 128]``), which is returned in ``query_out`` (a new tensor by default, ``query`` itself for in place) with
    zeros behind ``counts``. ``positions``: int32, int64 or float64 ``[sequences, rows]`` (``[..., axes]``), or
    the rows' own places. e4m3 pools: rows are divided by the positive ``k_scale`` / ``v_scale`` of their KV head and
    rounded once, at most 448. Rows past the table, or whose page is none of the pool, are not written
    (``device_error``). No two sequences may write the same page.
    """

    what = "append_rows"
    if not key.is_cuda:
        raise RuntimeError("h3sa kernels require CUDA tensors")
    device, shape, pool, kind = key.device, key.shape, key_pool.shape, key_pool.dtype
    if len(shape) != 4 or shape[3] != HEAD_DIM or key.dtype is not _BF16:
        raise RuntimeError(f"{what}: key must be bf16 [sequences, rows, kv_heads, {HEAD_DIM}]")
    batch, rows, kv_heads, _ = shape
    if value.shape != shape or value.dtype is not _BF16 or value.device != device:
        raise RuntimeError(f"{what}: value must be bf16 {list(shape)} on {device}")
    if (len(pool) != 3 or pool[0] != kv_heads or pool[1] % PAGE_ROWS or pool[2] != HEAD_DIM
            or _bad(key_pool, device, kind, pool) or _bad(value_pool, device, kind, pool)):
        raise RuntimeError(f"{what}: KV pools must be contiguous [{kv_heads}, pages*{PAGE_ROWS}, {HEAD_DIM}] of one "
                           f"dtype on {device}")
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
    live = _counts(what, counts, device, batch)
    error = _error_word(what, device, device_error)
    (kb, kn, kh, k1), (vb, vn, vh, v1) = key.stride(), value.stride()
    if k1 != 1 or v1 != 1:
        raise RuntimeError(f"{what}: rows of key and value must be contiguous")
    rotary = None
    if frequencies is not None:
        rotary = _rotary(what, frequencies, positions, shape[:2], HEAD_DIM, interleaved, factor, device)
    handle = _handle(stream, device)
    to_rotate = rotated = None
    if query is not None:
        wide = query.shape
        if (len(wide) != 4 or wide[0] != batch or wide[1] != rows or wide[3] != HEAD_DIM or query.dtype is not _BF16
                or query.device != device):
            raise RuntimeError(f"{what}: query must be bf16 [{batch}, {rows}, heads, {HEAD_DIM}] on {device}")
        if query_out is None:
            with _on(stream):
                query_out = _empty_like(query) if query.is_contiguous() else query.new_empty(wide)
        elif query_out.shape != wide or query_out.dtype is not _BF16 or query_out.device != device:
            raise RuntimeError(f"{what}: query_out must be bf16 {list(wide)} on {device}")
        (qb, qn, qh, q1), (ob, on, oh, o1) = query.stride(), query_out.stride()
        if q1 != 1 or o1 != 1:
            raise RuntimeError(f"{what}: rows of query and query_out must be contiguous")
        to_rotate = Heads(query.data_ptr(), qb, qn, qh, wide[2], 0)
        rotated = Heads(query_out.data_ptr(), ob, on, oh, wide[2], 0)
    elif query_out is not None:
        raise RuntimeError(f"{what}: query_out without a query")
    code = _APPEND(Heads(key.data_ptr(), kb, kn, kh, kv_heads, 0), Heads(value.data_ptr(), vb, vn, vh, kv_heads, 0),
                   to_rotate, rotated, batch, rows, key_pool.data_ptr(), value_pool.data_ptr(), pool[1] // PAGE_ROWS,
                   1 if e4m3 else 0, k_scale.data_ptr() if e4m3 else None, v_scale.data_ptr() if e4m3 else None,
                   table.data_ptr(), width, lengths.data_ptr(), live, rotary, error, handle)
    if code:
        check("h3sa_append_rows", code)
    return query_out


def tree_attention(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, table: torch.Tensor,
                   lengths: torch.Tensor, masks: torch.Tensor, softmax_scale: float, *,
                   counts: torch.Tensor | None = None, shared_rows: int = 0, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   lse: torch.Tensor | None = None, device_error: torch.Tensor | None = None,
                   stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Attention of the drafted rows of every sequence: row i < ``counts[b]`` of sequence b sees the keys j <
    ``lengths[b]``, and key ``lengths[b] + n`` of each node n < ``counts[b]`` whose bit is set in ``masks`` (int32
    ``[sequences, rows, ceil(rows / 32)]``, ``draft_tree``'s or any others).

    All other arguments are those of ``shared_prefix_attention``; the first ``shared_rows`` rows are the same pages
    in the table rows of all sequences whose ``lengths`` reach that far. Rows behind ``counts``, and rows that see
    nothing, come out zero with a log-sum-exp of -inf. An infinity or NaN in K or V of a drafted row reaches only the rows that
    see it; one in V of a sequence's history makes all its outputs in that column infinite or NaN. The lengths stay on the
    device, so the kernels are chosen by the width of ``table``: one no wider than the longest sequence needs is the fastest.
    """

    what = "tree_attention"
    if query.ndim != 4:
        raise RuntimeError(f"{what}: query must be bf16 [sequences, rows, heads, {HEAD_DIM}]")
    device, (batch, rows, _, _) = query.device, query.shape
    words = (batch, rows, (rows + 31) // 32)
    if _bad(masks, device, _I32, words):
        _refuse(what, "masks", device, _I32, words)
    return _attend(what, masks, _counts(what, counts, device, batch), query, key_pool, value_pool, table, lengths,
                   shared_rows, softmax_scale, False, k_scale, v_scale, out, lse, device_error, stream)


def keep_rows(pools: PoolTensors, table: torch.Tensor, lengths: torch.Tensor, path: torch.Tensor, *,
              device_error: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """The accepted rows become history: row ``lengths[b] + path[b, k]`` moves to row ``lengths[b] + k`` in every pool
    tensor, and the new lengths are returned. ``path`` int32 ``[sequences, steps]``: drafted rows in ascending
    order, negative after the last one. A path that does not ascend or leaves the table, or a page that is none of
    the pool, leaves its sequence as it was (``device_error``). Pool tensors may not overlap."""

    what = "keep_rows"
    if not table.is_cuda:
        raise RuntimeError("h3sa kernels require CUDA tensors")
    if table.ndim != 2 or path.ndim != 2:
        raise RuntimeError(f"{what}: table must be [sequences, width] and path [sequences, steps]")
    device, (sequences, width), steps = table.device, table.shape, path.shape[1]
    if _bad(table, device, _I32, (sequences, width)):
        _refuse(what, "table", device, _I32, (sequences, width))
    if _bad(lengths, device, _I32, (sequences,)):
        _refuse(what, "lengths", device, _I32, (sequences,))
    if _bad(path, device, _I32, (sequences, steps)):
        _refuse(what, "path", device, _I32, (sequences, steps))
    p = _pools(what, pools, None, device)
    error = _error_word(what, device, device_error)
    handle = _handle(stream, device)
    with _on(stream):
        kept = _empty_like(lengths)
    code = _KEEP(p, table.data_ptr(), sequences, width, lengths.data_ptr(), path.data_ptr(), steps, kept.data_ptr(), error,
                 handle)
    if code:
        check("h3sa_keep_rows", code)
    return kept


__all__ = ["append_rows", "draft_tree", "keep_rows", "tree_attention"]
