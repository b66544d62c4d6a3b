"""Attention over the pages that matter: bounds of every page's keys, and the pages that they rank highest for a query.

A long sequence's newest token attends to few of its pages in earnest.  ``page_bounds`` keeps, for every page and head of
a pool, the least and the largest value of each key channel in 8 bits; ``page_select`` finds from them, without reading a
key, the pages that may hold a query's highest scores; ``paged_attention(..., pages=...)`` reads these pages only.
``PagedKVPool(..., bounds=True)`` keeps the bounds by itself.

Bounds are int8 ``[num_pages, heads, 2, D]`` (lows, then highs) and float32 steps ``[num_pages, heads]``: the values of a
page's tokens lie between ``lows * step`` and ``highs * step``.  The step is the least power of two of which 127 reach the
page's largest magnitude (1 where all keys are zero; +inf, with bounds of zero, where a key is not finite), and the bounds are
rounded outwards, so they are the same however a page came to hold its tokens.
"""

from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from .. import _lib
from .._device import compute_device, device_ctx
from .paged_pool import _POOL, _ROWS, _flag, _index, _pool_fields, _raise_flag, _workspace
from .rotary import _launch, _rows

_BOUNDS = struct.Struct("<" + _POOL + "QQQQQ")
_SELECT = struct.Struct("<" + _ROWS + "QQQQQQQQqqiiiiiiiiiiii")
assert (_BOUNDS.size, _SELECT.size) == (120, 168)


def _bounds_checked(bounds: torch.Tensor, steps: torch.Tensor, shape: Tuple[int, ...], dev: torch.device) -> None:
    if (bounds.shape != shape or bounds.dtype is not torch.int8 or bounds.get_device() != dev.index
            or not bounds.is_contiguous()):
        raise ValueError(f"bounds must be a contiguous int8 tensor {list(shape)} on {dev}, got {tuple(bounds.shape)} {bounds.dtype}")
    if (steps.shape != shape[:2] or steps.dtype is not torch.float32 or steps.get_device() != dev.index
            or not steps.is_contiguous()):
        raise ValueError(f"steps must be a contiguous float32 tensor {list(shape[:2])} on {dev}, got {tuple(steps.shape)} {steps.dtype}")


def page_bounds(
    k_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    scale_k: Optional[torch.Tensor] = None,
    start: Optional[torch.Tensor] = None,
    bounds: Optional[torch.Tensor] = None,
    steps: Optional[torch.Tensor] = None,
    head_dim: Optional[int] = None,
    check: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Bounds of the keys of every page that holds tokens ``start[b] .. lengths[b] - 1``; returns ``(bounds, steps)``.

    After an append, ``start`` is the lengths before it (default: 0, all pages) and ``lengths`` those after it: a page is read
    whole, up to its last token, whichever of them are new.  ``bounds`` / ``steps``, where given, are updated in place, the other
    pages' left as they are; else they are made (bounds of 0 and steps of 1 for pages that are not read).  A page that
    sequences share is read for each of them, so it is to hold the same tokens for all, as full pages do.  The pages, table, lengths and
    ``check`` are those of ``paged_attention``; ``head_dim`` is only needed for int4 pages of an odd one.  One launch.
    """
    B = lengths.shape[0] if lengths.dim() == 1 else -1
    pool, dev, table = _pool_fields(k_pages, k_pages, block_table, scale_k, scale_k, B, head_dim)
    lens = _index(lengths, (B,), dev, "lengths")
    first = None if start is None else _index(start, (B,), dev, "start")
    shape = (pool[7], pool[9], 2, pool[10])
    if (bounds is None) != (steps is None):
        raise ValueError("bounds and steps must be given together")
    if bounds is None:
        bounds, steps = torch.zeros(shape, dtype=torch.int8, device=dev), torch.ones(shape[:2], device=dev)
    else:
        _bounds_checked(bounds, steps, shape, dev)
    flag = _flag(check, dev)
    args = _BOUNDS.pack(*pool, 0 if first is None else first.data_ptr(), lens.data_ptr(), bounds.data_ptr(), steps.data_ptr(),
                        0 if flag is None else flag.data_ptr())
    st = _launch(_lib.load().skv_pool_bounds, args, dev)
    if st:
        _lib.check(st, "page_bounds")
    del table
    if flag is not None:
        _raise_flag(flag, "page_bounds")
    return bounds, steps


def page_select(
    q: torch.Tensor,
    bounds: torch.Tensor,
    steps: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    page_size: int,
    keep: int,
    first: int = 1,
    recent: int = 1,
    causal: bool = False,
    new_lengths: Optional[torch.Tensor] = None,
    check: bool = False,
) -> torch.Tensor:
    """The ``keep`` pages of its sequence that each new token's queries read, for each key head: int32
    ``[B, heads, S_q, keep]``, page numbers within the sequence in ascending order, then -1.

    ``q``, ``lengths``, ``causal``, ``new_lengths`` and what a query sees are those of ``paged_attention``, which takes the result as
    ``pages``.  A query that sees no more than ``keep`` pages gets them all; else it gets the ``first`` ones, the ``recent`` ones up to
    its newest token (at least one), and of the others those whose keys may score highest, ties to the lowest page.

    The score of a page is the largest, over the query heads that share a key head, of ``sum_d max(q_d low_d, q_d high_d)``
    with the query in 8 bits: ``n = rint(q / t)``, ``t`` the least power of two of which 127 reach the row's largest
    magnitude.  The products and sums are whole numbers and exact, so equal inputs give equal pages on any device.  A page whose step is
    not finite goes before all others, one that the table does not name behind them; a query row that is not finite scores 0.
    Rows that require a gradient are read as constants.  The scores are kept meanwhile, 4 bytes for each of the table's pages, key heads and new
    tokens (4 GB for 8192 tokens, 32 heads and 4096 pages): a long prompt chooses in parts.  One launch.
    """
    shape = q.shape
    if len(shape) != 4:
        raise ValueError(f"q must be 4-D [batch, heads, seq, head_dim], got shape {tuple(q.shape)}")
    B, Hq, S_q, D = shape
    shape = bounds.shape
    if len(shape) != 4:
        raise ValueError(f"bounds must be [num_pages, heads, 2, head_dim], got {tuple(bounds.shape)}")
    if not bounds.is_cuda:
        compute_device()   # raises where there is no CUDA device at all
        raise ValueError("the bounds must be CUDA tensors")
    dev = bounds.device
    N, H = shape[0], shape[1]
    _bounds_checked(bounds, steps, (N, H, 2, D), dev)
    if H < 1 or Hq < 1 or Hq % H:
        raise ValueError(f"{Hq} query heads do not share {H} key heads evenly")
    if page_size < 1:
        raise ValueError(f"page_size must be >= 1, got {page_size}")
    if first < 0 or recent < 1 or first + recent > keep:
        raise ValueError(f"keep {keep} pages with the first {first} (>= 0) and the last {recent} (>= 1) of them")
    shape = block_table.shape
    if len(shape) != 2 or shape[0] != B:
        raise ValueError(f"block_table must be [batch={B}, width], got {tuple(block_table.shape)}")
    width = shape[1]
    table = _index(block_table, shape, dev, "block_table")
    lens = _index(lengths, (B,), dev, "lengths")
    new = None if new_lengths is None else _index(new_lengths, (B,), dev, "new_lengths")
    qd, q_rows = _rows(q, dev)
    pages = torch.empty(B, H, S_q, keep, dtype=torch.int32, device=dev)
    flag = _flag(check, dev)
    lib = _lib.load()
    with device_ctx(dev):
        stream = _lib.stream_of(dev)
        scratch = _workspace("select", dev, stream, max(16, lib.skv_pool_select_scratch_bytes(B, H, S_q, width)))
        st = lib.skv_pool_select(_SELECT.pack(
            *q_rows, bounds.data_ptr(), steps.data_ptr(), table.data_ptr(), lens.data_ptr(), 0 if new is None else new.data_ptr(),
            pages.data_ptr(), scratch.data_ptr(), 0 if flag is None else flag.data_ptr(), table.stride(0), scratch.numel(), width, N,
            page_size, H, D, B, S_q, keep, first, recent, bool(causal), 0), stream)
    if st:
        _lib.check(st, "page_select")
    del table, qd
    if flag is not None:
        _raise_flag(flag, "page_select")
    return pages
