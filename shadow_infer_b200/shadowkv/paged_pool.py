"""Serving from a page pool: append new tokens, attend from them, read tokens back.

``PagedKVStore`` keeps the pages of sequences of one length and hands attention a dense gather.
These operators serve sequences of different lengths from one pool of pages and never
build the dense cache.  A pool is plain tensors, so a program may own them (one set per layer, one
table for all layers) or let ``PagedKVPool`` do it:

* ``k_pages`` / ``v_pages`` ``[num_pages, heads, page_size, row]``: float32 (fp32), float16 (fp16), int8
  (int8) rows of ``head_dim``, or uint8 (int4) rows of ``head_dim / 2`` bytes, and ``scale_k`` / ``scale_v``
  ``[num_pages, heads, page_size, 1]`` (int8) or ``[num_pages, heads, page_size, groups, 1]`` (int4): the
  rows and scales of ``PagedKVStore``'s pages (shadowinfer/shadowkv/paged_kv_store.py:24-58), bit for bit;
* ``block_table`` int32 ``[batch, width]``: token t of sequence b is row ``t % page_size`` of page
  ``block_table[b, t // page_size]``;
* ``lengths`` int32 ``[batch]``.

Tables and lengths stay on the device: no call waits for the GPU (unless ``check`` asks for it), and
every call can be captured in a CUDA graph.  Entries of the table past a sequence's length are not
read, and neither are rows past it.  A page number outside the pool is never followed: its tokens are not written,
not attended to, zero when read.  A token whose position lies outside the rotary tables is not written either, key or value;
its rows keep what they held, so a program does not count it.  ``check=True`` waits for the call and raises
``ValueError`` if either happened.

Like the other caches' operators these serve: rows that require a gradient are read as constants
(``apply_rotary`` by itself has a gradient).
"""

from __future__ import annotations

import math
import struct
from typing import Any, List, Optional, Sequence, Tuple

import torch

from .. import _lib
from .._device import as_device, compute_device, device_ctx
from .rotary import _DTYPE_CODE, _NO_ROWS, _back, _common, _launch, _like, _rope_fields, _rows

_PRECISION_CODE = {torch.float32: 0, torch.float16: 1, torch.int8: 2, torch.uint8: 3}
_POOL, _ROWS, _ROPE = "QQQQQqiiiiiiii", "Qqqqii", "QQQqqiiiiii"
_APPEND = struct.Struct("<" + _POOL + _ROWS * 4 + _ROPE + "QQQii")
_READ = struct.Struct("<" + _POOL + _ROWS * 2 + "QQQii")
_ATTENTION = struct.Struct("<" + _POOL + _ROWS * 2 + "QQQqQiifi")
_SPARSE = struct.Struct("<" + _POOL + _ROWS * 2 + "QQQqQiifi" + "QqqqQqii")
assert (_APPEND.size, _READ.size, _ATTENTION.size, _SPARSE.size) == (336, 192, 216, 272)
_NO_ROPE = (0,) * 11
_SCRATCH = {}         # (device, stream) -> attention scratch
_SCRATCH_BYTES = {}   # (device, head_dim) -> its size


_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)


def _scratch(dev: torch.device, stream: int, head_dim: int) -> torch.Tensor:
    """The attention's scratch on a stream: partial results and arrival counters that every call leaves zero.  Calls
    of one stream follow each other, so they share one; a graph being captured gets its own.  (Found by the stream's handle,
    like the blocks of torch's own allocator: an external stream outlives its calls.)"""
    need = _SCRATCH_BYTES.get((dev.index, head_dim))
    if need is None:   # by the SMs of dev, which is the current device
        need = _SCRATCH_BYTES[dev.index, head_dim] = _lib.load().skv_pool_attention_scratch_bytes(head_dim)
    t = _SCRATCH.get((dev.index, stream))
    capturing = _capturing()
    if t is None or capturing or t.numel() < need:
        t = torch.empty(need, dtype=torch.uint8, device=dev)
        t[:_lib.load().skv_pool_attention_scratch_zeros()].zero_()
        if not capturing:
            _SCRATCH[dev.index, stream] = t
    return t


_WORK = {}            # (operator, device, stream) -> its workspace
_WORK_KEPT = 1 << 26  # larger workspaces are a call's own


def _workspace(what: str, dev: torch.device, stream: int, need: int) -> torch.Tensor:
    """``need`` bytes for an operator's calls on a stream: shared and kept like the attention's scratch."""
    t = _WORK.get((what, dev.index, stream))
    capturing = _capturing()
    if t is None or capturing or t.numel() < need:
        t = torch.empty(need if capturing or need > _WORK_KEPT else 1 << (need - 1).bit_length(), dtype=torch.uint8, device=dev)
        if not capturing and need <= _WORK_KEPT:
            _WORK[what, dev.index, stream] = t
    return t


def _index(t: torch.Tensor, shape: Tuple[int, ...], dev: torch.device, name: str) -> torch.Tensor:
    """An int32 table on ``dev`` whose last dimension is contiguous."""
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if t.dtype is not torch.int32 or not t.is_cuda or t.get_device() != dev.index:
        if t.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
        if t.dtype is torch.int64:   # numbers that 32 bits do not hold stay outside of every pool
            t = t.clamp(-2 ** 31, 2 ** 31 - 1)
        t = t.to(device=dev, dtype=torch.int32)
    return t if t.is_contiguous() or t.stride(-1) == 1 else t.contiguous()


def _pool_fields(k_pages, v_pages, block_table, scale_k, scale_v, batch: int, head_dim: Optional[int]):
    """The ``skv_pool`` fields, the pool's device and the table that was used (kept until the launch)."""
    shape = k_pages.shape
    dtype = k_pages.dtype
    same = v_pages is k_pages
    if len(shape) != 4 or not (same or (v_pages.shape == shape and v_pages.dtype is dtype)):
        raise ValueError("k_pages/v_pages must be alike [num_pages, heads, page_size, row], got "
                         f"{tuple(k_pages.shape)} {k_pages.dtype} and {tuple(v_pages.shape)} {v_pages.dtype}")
    code = _PRECISION_CODE.get(dtype)
    if code is None:
        raise ValueError(f"Unsupported page precision: {k_pages.dtype}")
    if not k_pages.is_cuda:
        compute_device()   # raises where there is no CUDA device at all
        raise ValueError("the pages must be CUDA tensors")
    dev = k_pages.device
    if not k_pages.is_contiguous() or not (same or (v_pages.get_device() == dev.index and v_pages.is_contiguous())):
        raise ValueError("the pages must be contiguous tensors on one device")
    N, H, P, row = shape
    D = (2 * row if code == 3 else row) if head_dim is None else head_dim
    if row != ((D + 1) // 2 if code == 3 else D):
        raise ValueError(f"page rows of {row} do not hold a head_dim of {D}")
    group = sk = sv = 0
    if code >= 2:
        if scale_k is None or scale_v is None:
            raise ValueError("int8/int4 pages need scale_k and scale_v")
        groups = scale_k.shape[3] if code == 3 and scale_k.dim() == 5 else 1
        want = (N, H, P, 1) if code == 2 else (N, H, P, groups, 1)
        for s in (scale_k,) if scale_v is scale_k else (scale_k, scale_v):
            if s.shape != want or s.dtype is not torch.float32 or s.get_device() != dev.index or not s.is_contiguous():
                if code == 3 and s.dim() == 5 and s.shape != want and s.shape[:3] + s.shape[4:] == (N, H, P, 1):
                    raise ValueError(f"{groups} int4 groups do not divide a head_dim of {D}, or scale_v has others: {s.shape[3]}")
                raise ValueError(f"scales must be contiguous float32 [{N}, {H}, {P}, {'1' if code == 2 else 'groups, 1'}] "
                                 f"on {dev}, got {tuple(s.shape)} {s.dtype}")
        if code == 3:
            if groups < 1 or D % groups:
                raise ValueError(f"{groups} int4 groups do not divide a head_dim of {D}")
            group = D // groups
        sk, sv = scale_k.data_ptr(), scale_v.data_ptr()
    table_shape = block_table.shape
    if len(table_shape) != 2 or table_shape[0] != batch:
        raise ValueError(f"block_table must be [batch={batch}, width], got {tuple(block_table.shape)}")
    table = _index(block_table, table_shape, dev, "block_table")
    return ((k_pages.data_ptr(), v_pages.data_ptr(), sk, sv, table.data_ptr(), table.stride(0), table_shape[1], N, P, H,
             D, group, code, batch), dev, table)


def _staged(host: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """``host`` on ``dev`` without waiting for the GPU: through pinned memory, which torch keeps until the copy is done."""
    return host.pin_memory().to(dev, non_blocking=True)


def _flag(check: bool, dev: torch.device) -> Optional[torch.Tensor]:
    return torch.zeros(1, dtype=torch.int32, device=dev) if check else None


def _raise_flag(flag: torch.Tensor, what: str) -> None:
    if int(flag.item()):
        raise ValueError(f"{what}: a page number, length or position lies outside the pool or the tables")


def paged_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    scale_k: Optional[torch.Tensor] = None,
    scale_v: Optional[torch.Tensor] = None,
    new_lengths: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    cos: Optional[torch.Tensor] = None,
    sin: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    check: bool = False,
) -> Optional[torch.Tensor]:
    """Write new tokens' keys and values into their pages, rotated and quantised on the way; returns the rotated ``q``.

    ``k`` / ``v`` ``[B, heads, S, D]`` (fp32, fp16 or bf16, any strides over the first three dimensions): row s of
    sequence b becomes token ``lengths[b] + s`` where ``s < new_lengths[b]`` (default: all S).  ``lengths`` counts the
    tokens held BEFORE the call and is not changed.  With ``cos`` / ``sin`` (``rotary_tables``) keys are turned to
    their positions first, as ``apply_rotary`` does (in fp32, not rounded in between), and
    ``q`` ``[B, H_q, S, D]``, where given, is returned turned, all S rows of it.  ``positions`` as for
    ``apply_rotary``; default: the token's index.

    The pages' precision is their type.  Rows and scales are those of ``PagedKVStore.append``
    (paged_kv_store.py:189-224): int8 ``amax / 127`` a row, int4 ``amax / 7`` a group; one that holds a NaN has
    the scale NaN and is read as NaN.  One launch.
    """
    shape = k.shape
    if len(shape) != 4 or v.shape != shape:
        if k.dim() != 4 or v.dim() != 4:
            raise ValueError(f"k/v must be 4-D [batch, heads, tokens, head_dim], got k.dim={k.dim()}, v.dim={v.dim()}")
        raise ValueError(f"k/v shapes disagree: {tuple(k.shape)} vs {tuple(v.shape)}")
    B, H, S, D = shape
    pool, dev, table = _pool_fields(k_pages, v_pages, block_table, scale_k, scale_v, B, D)
    if H != pool[9]:
        raise ValueError(f"k/v have {H} heads, the pool has {pool[9]}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin must be given together")
    lens = _index(lengths, (B,), dev, "lengths")
    new = None if new_lengths is None else _index(new_lengths, (B,), dev, "new_lengths")
    kd, k_rows = _rows(k, dev, _common(k, v, q))
    vd, v_rows = _rows(v, dev, kd.dtype)
    q_rows = q_out_rows = _NO_ROWS
    qd = q_out = None
    if q is not None:
        shape = q.shape
        if len(shape) != 4 or shape != (B, shape[1], S, D):
            raise ValueError(f"q must be [batch, heads, {S}, {D}], got {tuple(q.shape)}")
        if cos is None:
            raise ValueError("q without cos and sin has nothing to be rotated by")
        qd, q_rows = _rows(q, dev, kd.dtype)
        q_out, q_out_rows = _like(qd)
    rope, keep = _NO_ROPE, None
    if cos is not None:
        rope, keep = _rope_fields(cos, sin, positions, B, S, D, bool(interleaved), False, dev)
    flag = _flag(check, dev)
    args = _APPEND.pack(*pool, *k_rows, *v_rows, *q_rows, *q_out_rows, *rope, lens.data_ptr(),
                        0 if new is None else new.data_ptr(), 0 if flag is None else flag.data_ptr(), S, 0)
    st = _launch(_lib.load().skv_pool_append, args, dev)
    if st:
        _lib.check(st, "paged_append")
    del table, keep, vd, qd
    if flag is not None:
        _raise_flag(flag, "paged_append")
    return None if q_out is None else _back(q_out, q, dev)


def paged_read(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    tokens: int,
    scale_k: Optional[torch.Tensor] = None,
    scale_v: Optional[torch.Tensor] = None,
    start: Optional[torch.Tensor] = None,
    head_dim: Optional[int] = None,
    dtype: torch.dtype = torch.float32,
    check: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Dense ``(k, v)`` ``[B, heads, tokens, D]``: the values that tokens ``start[b] .. start[b] + tokens - 1`` stand for.

    Tokens at or past ``lengths[b]`` are zero.  ``start`` int32 ``[B]`` (default: 0).  ``head_dim`` is only needed for
    int4 pages of an odd one.  ``dtype``: float32, float16 or bfloat16, rounded once.
    """
    if tokens < 0:
        raise ValueError(f"tokens must be >= 0, got {tokens}")
    if dtype not in _DTYPE_CODE:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    B = lengths.shape[0] if lengths.dim() == 1 else -1
    pool, dev, table = _pool_fields(k_pages, v_pages, block_table, scale_k, scale_v, B, head_dim)
    lens = _index(lengths, (B,), dev, "lengths")
    first = None if start is None else _index(start, (B,), dev, "start")
    k = torch.empty((B, pool[9], tokens, pool[10]), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    st = k.stride()
    rows = (st[0], st[1], st[2], _DTYPE_CODE[dtype], pool[9])
    flag = _flag(check, dev)
    args = _READ.pack(*pool, k.data_ptr(), *rows, v.data_ptr(), *rows, 0 if first is None else first.data_ptr(),
                      lens.data_ptr(), 0 if flag is None else flag.data_ptr(), tokens, 0)
    st = _launch(_lib.load().skv_pool_read, args, dev)
    if st:
        _lib.check(st, "paged_read")
    del table
    if flag is not None:
        _raise_flag(flag, "paged_read")
    return k, v


def _listed_pages(pages: torch.Tensor, shape: Tuple[int, int, int], dev: torch.device) -> torch.Tensor:
    """``pages`` as int32 ``[*shape, keep]`` on ``dev`` whose last dimension is contiguous."""
    have = pages.shape
    if len(have) != 4 or have[3] < 1:
        raise ValueError(f"pages must be [batch, heads, seq, keep], got {tuple(pages.shape)}")
    want = (*shape, have[3])
    if have != want:
        try:
            pages = pages.expand(want)
        except RuntimeError:
            raise ValueError(f"pages must broadcast to {[*shape, 'keep']}, got {tuple(pages.shape)}") from None
    return _index(pages, want, dev, "pages")


def _evenly_spaced(rows: Tuple[int, ...], B: int, S: int, heads: int) -> bool:
    """Whether the rows (their ``skv_rows`` fields) of (sequence, token, head), in this order, are evenly spaced."""
    _, sb, sh, ss, _, _ = rows
    return (S == 1 or heads == 1 or ss == heads * sh) and (B == 1 or (heads == 1 and S == 1) or sb == (S * ss if S > 1 else heads * sh))


def paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    scale_k: Optional[torch.Tensor] = None,
    scale_v: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    causal: bool = False,
    new_lengths: Optional[torch.Tensor] = None,
    check: bool = False,
    pages: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of each sequence's newest tokens over its pages; returns ``[B, H_q, S_q, D]`` in ``q``'s type.

    ``q`` ``[B, H_q, S_q, D]`` (fp32, fp16 or bf16, any strides over the first three dimensions): the S_q newest tokens,
    one while decoding.  ``lengths`` counts the tokens to attend to, the new ones included (append first).  Query
    head h reads key head ``h // (H_q / heads)``.  A query sees every token of its sequence, or with ``causal``
    those up to itself: query i tokens ``<= lengths[b] - S_q + i``.  ``new_lengths`` int32 ``[B]``: only the first
    ``new_lengths[b]`` queries are tokens, the rest padding of a ragged prompt (``S_q`` above is then
    ``new_lengths[b]``).  A query that sees nothing (padding, an empty sequence) gives zeros.
    ``scale`` defaults to ``1/sqrt(D)``.

    ``pages`` (int32 or int64, broadcast to ``[B, heads, S_q, keep]``; ``page_select`` finds them) leaves each query, of those
    tokens, the ones in the listed pages, which are all that is read: an entry counts if it is one of the pages
    that the query sees and larger than every entry before it, so lists are ascending and anything else in them, -1 among it, stands
    for no page.  One launch, or two.

    The result has ``q``'s dimension order in memory (as torch's own operators keep it), so that the output of a
    ``[B, S, H, D]`` projection goes back to one without a copy.  (With ``pages``, several new tokens of another order are
    copied to that one, and the result has it.)

    Scores, softmax and sums are fp32.  What the tensor cores multiply is rounded less than the result is: a weight (times the
    exponent of its token's V scale) is one fp16 operand of 11 bits for bf16 results and two (22 bits) else, and below 2^-36 of
    its query's largest it is rounded to that step; an int4 scale of V has 14 bits for 16-bit results of a few queries, 18 for
    many, 21 for fp32 ones; for 16-bit results the sums over a sequence's tiles are cut off, not rounded, at 2^-24 a step.  Queries of
    2^98 and more in magnitude leave that range (NaN).  What is
    not finite reaches the queries that see it and no others: a key all of their values, a value its own ones.  Every page is read once for all the query rows that share its key
    head.  The sequences are split over the whole GPU by their lengths on the device, long ones into
    parts that are joined in token order, so equal calls give equal bits.
    """
    shape = q.shape
    if len(shape) != 4:
        raise ValueError(f"q must be 4-D [batch, heads, seq, head_dim], got shape {tuple(q.shape)}")
    B, Hq, S_q, D = shape
    pool, dev, table = _pool_fields(k_pages, v_pages, block_table, scale_k, scale_v, B, D)
    if Hq % pool[9]:
        raise ValueError(f"{Hq} query heads do not share {pool[9]} key heads evenly")
    lens = _index(lengths, (B,), dev, "lengths")
    new = None if new_lengths is None else _index(new_lengths, (B,), dev, "new_lengths")
    if pages is not None:
        listed = _listed_pages(pages, (B, pool[9], S_q), dev)
    qd, q_rows = _rows(q, dev)
    if pages is not None and not _evenly_spaced(q_rows, B, S_q, Hq):
        qd, q_rows = _rows(qd.transpose(1, 2).contiguous().transpose(1, 2), dev)
    out, out_rows = _like(qd)
    if pages is not None and not _evenly_spaced(out_rows, B, S_q, Hq):
        out, out_rows = _like(torch.empty((B, S_q, Hq, D), dtype=qd.dtype, device=dev).transpose(1, 2))
    flag = _flag(check, dev)
    lib = _lib.load()
    with device_ctx(dev):
        stream = _lib.stream_of(dev)
        scratch = _scratch(dev, stream, D)
        fields = (*pool, *q_rows, *out_rows, lens.data_ptr(), 0 if new is None else new.data_ptr(), scratch.data_ptr(), scratch.numel(),
                  0 if flag is None else flag.data_ptr(), S_q, bool(causal), 1.0 / math.sqrt(D) if scale is None else scale, 0)
        if pages is None:
            st = lib.skv_pool_attention(_ATTENTION.pack(*fields), stream)
        else:
            sb, sh, ss, _ = listed.stride()
            keep = listed.shape[3]
            tables = _workspace("tables", dev, stream, B * S_q * pool[9] * (keep + 32) * 4)
            st = lib.skv_pool_sparse_attention(_SPARSE.pack(*fields, listed.data_ptr(), sb, sh, ss, tables.data_ptr(), tables.numel(),
                                                            keep, 0), stream)
    if st:
        _lib.check(st, "paged_attention")
    del table, qd
    if flag is not None:
        _raise_flag(flag, "paged_attention")
    return _back(out, q, dev)


class _Family:
    """Sequences that reordered beams' pages are among (which of them holds which, the device alone knows), and the pages named by those
    of them that have ended."""

    def __init__(self) -> None:
        self.rows = set()
        self.pages: List[int] = []


class PagedKVPool:
    """The pages of one layer for ``batch_size`` sequences of different lengths, and their bookkeeping.

    ``append`` takes pages from the free list, writes the new tokens and advances the lengths; ``attention`` and
    ``read`` use what is held; ``release`` ends a sequence and returns its pages.  ``block_table`` and ``lengths``
    are device tensors (for graphs and for the functions above); ``token_counts`` are the lengths on the host.

    ``fork`` lets empty sequences go on from a sequence, and ``reorder`` lets the beams of a search go on from one another.  A page is free
    again when the last sequence that it is shared by is released; sequences that were reordered return theirs together, when
    the last of them (and of those that were forked from them since) is.  With ``bounds``, ``append`` keeps the
    pages' bounds (``page_bounds``) and ``attention`` can be told to read the pages that they rank highest only.
    """

    def __init__(
        self,
        num_pages: int,
        batch_size: int,
        num_heads: int,
        head_dim: int,
        max_tokens: int,
        page_size: int = 32,
        precision: str = "fp16",
        int4_group_size: int = 16,
        device: Any = "cuda",
        bounds: bool = False,
    ) -> None:
        if min(num_pages, batch_size, num_heads, head_dim, max_tokens, page_size) < 1:
            raise ValueError("PagedKVPool sizes must be >= 1")
        if precision not in ("fp32", "fp16", "int8", "int4"):
            raise ValueError(f"Unsupported page precision: {precision}")
        if int4_group_size < 1:
            raise ValueError(f"int4_group_size must be >= 1, got {int4_group_size}")
        dev = as_device(device)
        if dev.type != "cuda":
            raise ValueError(f"PagedKVPool lives on a CUDA device, got {dev}")
        if dev.index is None:
            dev = compute_device()
        self.precision, self.page_size = precision, int(page_size)
        self.batch_size, self.num_heads, self.head_dim = int(batch_size), int(num_heads), int(head_dim)
        shape = (num_pages, num_heads, page_size)
        group = int4_group_size if head_dim % int4_group_size == 0 else head_dim
        row = (head_dim + 1) // 2 if precision == "int4" else head_dim
        dtype = {"fp32": torch.float32, "fp16": torch.float16, "int8": torch.int8, "int4": torch.uint8}[precision]
        tail = {"int8": (1,), "int4": (head_dim // group, 1)}.get(precision)
        self.k_pages, self.v_pages = (torch.zeros(*shape, row, dtype=dtype, device=dev) for _ in range(2))
        self.scale_k, self.scale_v = (None if tail is None else torch.ones(*shape, *tail, device=dev) for _ in range(2))
        self.bounds = self.steps = None
        if bounds:
            self.bounds = torch.zeros(num_pages, num_heads, 2, head_dim, dtype=torch.int8, device=dev)
            self.steps = torch.ones(num_pages, num_heads, device=dev)
        # each sequence's pages; of reordered sequences those that were taken for it, wherever they are now
        self._table = torch.full((batch_size, -(-max_tokens // page_size)), -1, dtype=torch.int32)
        self.block_table = self._table.to(dev)
        self.lengths = torch.zeros(batch_size, dtype=torch.int32, device=dev)
        self.token_counts: List[int] = [0] * batch_size
        self._free = list(range(num_pages - 1, -1, -1))
        self._names = [0] * num_pages       # how many sequences (or families, for those that have ended) name a page
        self._family: List[Optional[_Family]] = [None] * batch_size

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _pages_held(self, b: int) -> int:
        return -(-self.token_counts[b] // self.page_size)

    def append(
        self,
        k: torch.Tensor,
        v: torch.Tensor,
        q: Optional[torch.Tensor] = None,
        cos: Optional[torch.Tensor] = None,
        sin: Optional[torch.Tensor] = None,
        new_lengths: Optional[Sequence[int]] = None,
        positions: Optional[torch.Tensor] = None,
        interleaved: bool = False,
        check: bool = False,
    ) -> Optional[torch.Tensor]:
        """``paged_append`` behind each sequence's tokens (``new_lengths``: host numbers, default all rows).  A call
        that the free pages or the table cannot hold raises ``RuntimeError``, and one whose tokens the rotary tables do not
        reach ``ValueError``; neither changes anything.  ``positions`` are on the device: only ``check=True``, which
        waits for the call, refuses those outside the tables (without it their tokens count as held, but are not
        written)."""
        S = int(k.shape[2]) if k.dim() == 4 else 0
        new = [S] * self.batch_size if new_lengths is None else [int(n) for n in new_lengths]
        if len(new) != self.batch_size or min(new) < 0 or max(new) > S:
            raise ValueError(f"new_lengths must be {self.batch_size} numbers in [0, {S}], got {new}")
        P = self.page_size
        grown = [-(-(c + n) // P) for c, n in zip(self.token_counts, new)]
        wanted = [g - self._pages_held(b) for b, g in enumerate(grown)]
        if max(grown) > self.block_table.shape[1]:
            raise RuntimeError(f"a sequence of {max(c + n for c, n in zip(self.token_counts, new))} tokens does not fit "
                               f"the table of {self.block_table.shape[1]} pages of {P}")
        if sum(wanted) > len(self._free):
            raise RuntimeError(f"{sum(wanted)} pages wanted, {len(self._free)} free")
        last = max((c + n for c, n in zip(self.token_counts, new) if n), default=0)
        if cos is not None and positions is None and last > cos.shape[0]:
            raise ValueError(f"position {last - 1} lies outside rotary tables of {cos.shape[0]} positions")
        block_table = self.block_table
        taken = self._free[len(self._free) - sum(wanted):][::-1]
        places = [(b, g - n + i) for b, (g, n) in enumerate(zip(grown, wanted)) for i in range(n)]
        if taken:
            host, block_table = self._with_pages(places, taken)
        fresh = None if new_lengths is None else _staged(torch.tensor(new, dtype=torch.int32), self.lengths.device)
        out = paged_append(k, v, self.k_pages, self.v_pages, block_table, self.lengths, self.scale_k, self.scale_v, fresh,
                           q, cos, sin, positions, interleaved, check)
        if taken:
            self._take(host, taken)
            self.block_table.copy_(block_table)
        start = None if self.bounds is None else self.lengths.clone()
        self.lengths += S if fresh is None else fresh
        self.token_counts = [c + n for c, n in zip(self.token_counts, new)]
        if start is not None:
            from .page_selection import page_bounds

            page_bounds(self.k_pages, self.block_table, self.lengths, self.scale_k, start, self.bounds, self.steps, self.head_dim)
        return out

    def _with_pages(self, places: List[Tuple[int, int]], pages: List[int]) -> Tuple[torch.Tensor, torch.Tensor]:
        """The host's and the device's table with ``pages`` at ``places`` (sequence, number), without waiting for the GPU: one copy of
        the host's, unless a sequence has been reordered."""
        rows, columns = zip(*places)
        host = self._table.clone()
        host.numpy()[rows, columns] = pages
        if not any(self._family):
            return host, _staged(host, self.lengths.device)
        at = _staged(torch.tensor([rows, columns, pages], dtype=torch.int64), self.lengths.device)
        table = self.block_table.clone()
        table[at[0], at[1]] = at[2].to(torch.int32)
        return host, table

    def _take(self, host: torch.Tensor, pages: List[int]) -> None:
        """``pages``, the last of the free ones, are taken as the table ``host`` has them."""
        self._table = host
        del self._free[len(self._free) - len(pages):]
        for p in pages:
            self._names[p] = 1

    def attention(self, q: torch.Tensor, scale: Optional[float] = None, causal: bool = False,
                  new_lengths: Optional[torch.Tensor] = None, keep: Optional[int] = None, first: int = 1,
                  recent: int = 1) -> torch.Tensor:
        """``paged_attention`` over everything held, or with ``keep`` over the pages that ``page_select`` chooses."""
        pages = None
        if keep is not None:
            if self.bounds is None:
                raise ValueError("a choice of pages needs PagedKVPool(..., bounds=True)")
            from .page_selection import page_select

            pages = page_select(q, self.bounds, self.steps, self.block_table, self.lengths, self.page_size, keep, first, recent, causal,
                                new_lengths)
        return paged_attention(q, self.k_pages, self.v_pages, self.block_table, self.lengths, self.scale_k, self.scale_v,
                               scale, causal, new_lengths, pages=pages)

    def read(self, tokens: Optional[int] = None, start: Optional[torch.Tensor] = None,
             dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """``paged_read`` of ``tokens`` tokens (default: the longest sequence's)."""
        return paged_read(self.k_pages, self.v_pages, self.block_table, self.lengths,
                          max(self.token_counts) if tokens is None else tokens, self.scale_k, self.scale_v, start,
                          self.head_dim, dtype)

    def fork(self, b: int, others: Sequence[int]) -> None:
        """The empty sequences ``others`` go on from sequence ``b``: its full pages are shared, a last page that is partly filled is
        copied to a page of their own.  Raises ``ValueError`` for sequences that are not empty and ``RuntimeError`` where too few pages are free;
        nothing has changed then."""
        rows = [range(self.batch_size)[i] for i in (b, *others)]
        if len(set(rows)) != len(rows) or any(self.token_counts[r] for r in rows[1:]):
            raise ValueError(f"sequences {rows[1:]} are to be different, empty, and not {rows[0]}")
        if len(rows) == 1 or self.token_counts[rows[0]] == 0:
            return
        j, partly = divmod(self.token_counts[rows[0]], self.page_size)
        taken = self._free[len(self._free) - len(rows) + 1:][::-1] if partly else []
        if partly and len(taken) < len(rows) - 1:
            raise RuntimeError(f"{len(rows) - 1} pages wanted, {len(self._free)} free")
        if len(rows) > 1024:
            raise ValueError(f"{len(rows) - 1} sequences go on from one, 1023 at most")
        from .beam import paged_reorder

        host, table = self._with_pages([(r, j) for r in rows[1:]], taken) if taken else (self._table, self.block_table)
        at = _staged(torch.tensor(rows, dtype=torch.int64), self.lengths.device)
        parents = torch.zeros(1, len(rows), dtype=torch.int64, device=self.lengths.device)
        lengths = self.lengths[at[:1]].expand(len(rows)).contiguous()
        new_table, new_lengths = paged_reorder(self.k_pages, self.v_pages, table[at], lengths, parents, self.scale_k, self.scale_v,
                                               self.bounds, self.steps, self.head_dim)
        self.block_table.index_copy_(0, at, new_table)
        self.lengths.index_copy_(0, at, new_lengths)
        if taken:
            self._take(host, taken)
        if self._family[rows[0]] is None:
            shared = self._table[rows[0], :j]
            self._table[rows[1:], :j] = shared
            for p in shared.tolist():
                self._names[p] += len(rows) - 1
        else:
            self._join(rows)
        for r in rows[1:]:
            self.token_counts[r] = self.token_counts[rows[0]]

    def reorder(self, parents: torch.Tensor, check: bool = False) -> None:
        """``paged_reorder`` of all sequences: ``parents`` ``[groups, beams]``, ``groups * beams`` the batch size.  The sequences of a group
        must be equally long (``ValueError``).  The parents stay on the device; one outside its group leaves an empty sequence
        there that the host counts as long as the others, unless ``check=True``, which waits, refuses it by ``ValueError``."""
        if parents.dim() != 2 or parents.numel() != self.batch_size:
            raise ValueError(f"parents must be [groups, beams] of {self.batch_size} sequences, got {tuple(parents.shape)}")
        groups, beams = parents.shape
        for g in range(groups):
            counts = self.token_counts[g * beams:(g + 1) * beams]
            if min(counts) != max(counts):
                raise ValueError(f"the sequences of group {g} are not equally long: {counts}")
        if check and not bool(((parents >= 0) & (parents < beams)).all()):
            raise ValueError(f"a parent lies outside its group of {beams}")
        from .beam import paged_reorder

        table, lengths = paged_reorder(self.k_pages, self.v_pages, self.block_table, self.lengths, parents, self.scale_k, self.scale_v,
                                       self.bounds, self.steps, self.head_dim)
        self.block_table.copy_(table)
        self.lengths.copy_(lengths)
        for g in range(groups):
            if beams > 1 and self.token_counts[g * beams]:
                self._join(range(g * beams, (g + 1) * beams))

    def _join(self, rows: Sequence[int]) -> None:
        """Sequences ``rows``, and those that their pages are among already, return their pages together from now on."""
        family = self._family[rows[0]] or _Family()
        for r in rows:
            other = self._family[r]
            if other is family and r in family.rows:
                continue
            mine = {r} if other is None else other.rows
            if other is not None and other is not family:
                family.pages.extend(other.pages)
            family.rows |= mine
            for o in mine:
                self._family[o] = family

    def release(self, b: int) -> int:
        """End sequence ``b``: its pages are free again, but for those that other sequences share and, if it was reordered, until the
        others of its family have ended.  Returns how many became free."""
        b = range(self.batch_size)[b]
        pages = [p for p in self._table[b].tolist() if p >= 0]
        self._table[b] = -1
        family, self._family[b] = self._family[b], None
        if family is not None:
            family.rows.discard(b)
            family.pages.extend(pages)
            pages = [] if family.rows else family.pages
        free = []
        for p in pages:
            self._names[p] -= 1
            if self._names[p] == 0:
                free.append(p)
        self._free.extend(reversed(free))
        self.block_table[b].fill_(-1)
        self.lengths[b:b + 1].zero_()   # (an assignment to one element waits for the GPU)
        self.token_counts[b] = 0
        return len(free)

    def __repr__(self) -> str:
        return (f"PagedKVPool(precision={self.precision}, heads={self.num_heads}, head_dim={self.head_dim}, "
                f"page_size={self.page_size}, pages={self.k_pages.shape[0]}, free={len(self._free)}, "
                f"tokens={self.token_counts})")


def paged_block_forward(block, hidden: torch.Tensor, pool: PagedKVPool, cos: Optional[torch.Tensor] = None,
                        sin: Optional[torch.Tensor] = None, causal: bool = False,
                        new_lengths: Optional[Sequence[int]] = None, keep: Optional[int] = None, first: int = 1,
                        recent: int = 1) -> torch.Tensor:
    """One transformer block over a page pool, for prompts and for single tokens: the block's own modules (the layout
    of ``packed_block_forward``; ``num_kv_heads`` where the keys are shared) around ``pool.append`` (queries and keys
    rotated, keys and values quantised into their pages) and ``pool.attention``.

    ``hidden`` [B, S, hidden_dim] are the S newest tokens; returns their new hidden states.  Rows s >=
    ``new_lengths[b]`` (host numbers, default all S) are the padding of a ragged prompt: nothing is stored for
    them and their outputs mean nothing.  ``keep`` / ``first`` / ``recent`` as for ``pool.attention``: each query reads ``keep`` pages only.
    """
    import torch.nn.functional as F

    B, S, _ = hidden.shape
    nh, hd = int(block.num_heads), int(block.head_dim)
    nkv = int(getattr(block, "num_kv_heads", nh))
    normed = block.ln1(hidden)
    q = block.q_proj(normed).view(B, S, nh, hd).transpose(1, 2)
    k = block.k_proj(normed).view(B, S, nkv, hd).transpose(1, 2)
    v = block.v_proj(normed).view(B, S, nkv, hd).transpose(1, 2)
    if cos is None:
        pool.append(k, v, new_lengths=new_lengths)
    else:
        q = pool.append(k, v, q=q, cos=cos, sin=sin, new_lengths=new_lengths)
    fresh = None if new_lengths is None else _staged(torch.tensor(list(new_lengths), dtype=torch.int32), pool.lengths.device)
    attn = pool.attention(q, causal=causal, new_lengths=fresh, keep=keep, first=first, recent=recent).transpose(1, 2).reshape(B, S, nh * hd)
    hidden = hidden + block.o_proj(attn)
    return hidden + block.down_proj(F.gelu(block.up_proj(block.ln2(hidden))))
