"""Rotary positions: the tables and the turn of queries and keys by their positions.

The reference's models leave positions to the checkpoint's own attention module
(shadowinfer/models/diffusion_llama.py:357-375 calls it before the cache); a serving step
needs them next to the paged cache, which stores keys after the turn.
"""

from __future__ import annotations

import math
import struct
from typing import Any, Optional, Tuple

import torch

from .. import _lib
from .._device import _get_device, as_device, back, compute_device, device_ctx

_DTYPE_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ARGS = struct.Struct("<" + "Qqqqii" * 4 + "QQQqqiiiiii" + "iiii")   # skv_rotary_args
assert _ARGS.size == 240
_NO_ROWS = (0, 0, 0, 0, 0, 0)


def rotary_tables(
    rotary_dim: int,
    max_positions: int,
    base: float = 10000.0,
    scaling: Optional[str] = None,
    factor: float = 1.0,
    original_positions: Optional[int] = None,
    device: Any = "cuda",
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(cos, sin)`` float32 ``[max_positions, rotary_dim / 2]``: pair i turns by ``p * base**(-2 i / rotary_dim)``.

    ``scaling`` stretches the positions a model was trained on by ``factor``:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: the base raised to ``base * factor ** (rotary_dim / (rotary_dim - 2))``, which leaves the
      fastest pair as it is and divides the slowest one's frequency by ``factor``;
    * ``"ntk_parts"``: pairs that turn over 32 times within ``original_positions`` keep their frequency, those
      that turn less than once are divided by ``factor``, a linear ramp in between, and the
      tables are multiplied by ``0.1 ln(factor) + 1``.

    Angles are computed in 64 bits (a 32-bit angle is off by 4e-3 at position 65536).
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if max_positions < 1:
        raise ValueError(f"max_positions must be >= 1, got {max_positions}")
    if scaling not in (None, "linear", "ntk", "ntk_parts"):
        raise ValueError(f"unknown rotary scaling: {scaling}")
    if factor <= 0 or (scaling == "ntk_parts" and (original_positions is None or original_positions < 1)):
        raise ValueError("rotary scaling needs a positive factor (and original_positions for 'ntk_parts')")
    gain = 1.0
    if scaling == "ntk":
        base = base * factor ** (rotary_dim / max(1, rotary_dim - 2))
    inv = base ** (-torch.arange(rotary_dim // 2, dtype=torch.float64) * 2 / rotary_dim)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "ntk_parts":
        keep = ((original_positions * inv / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        inv = inv / factor * (1 - keep) + inv * keep
        gain = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    dev = as_device(device)
    angle = torch.arange(max_positions, dtype=torch.float64, device=dev)[:, None] * inv.to(dev)
    return (angle.cos() * gain).float(), (angle.sin() * gain).float()


def _rows(t: torch.Tensor, dev: torch.device, dtype: Optional[torch.dtype] = None):
    """``t`` [B, H, S, D] as the kernels read it (on ``dev``, fp32 / fp16 / bf16, the last dimension contiguous), and its
    ``skv_rows`` fields."""
    have = t.dtype
    code = _DTYPE_CODE.get(have)
    if t.requires_grad or code is None or (dtype is not None and have is not dtype) or not t.is_cuda or t.get_device() != dev.index:
        if dtype is None:
            dtype = have if code is not None else torch.float32
        t = t.detach().to(device=dev, dtype=dtype)
        code = _DTYPE_CODE[dtype]
    st = t.stride()
    if st[3] != 1 and t.shape[3] != 1:
        t = t.contiguous()
        st = t.stride()
    return t, (t.data_ptr(), st[0], st[1], st[2], code, t.shape[1])


def _common(t: torch.Tensor, *others: Optional[torch.Tensor]) -> Optional[torch.dtype]:
    """The type of rows that share a launch: their own (None), or fp32, which holds fp16 and bf16, where they differ."""
    have = t.dtype
    for o in others:
        if o is not None and o.dtype is not have:
            return torch.float32
    return None


def _like(t: torch.Tensor):
    """An output laid out like ``t`` (dense, dimensions in the order of ``t``'s strides), and its ``skv_rows`` fields."""
    out = torch.empty_like(t)
    st = out.stride()
    if st[3] != 1 and t.shape[3] != 1:
        out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        st = out.stride()
    return out, (out.data_ptr(), st[0], st[1], st[2], _DTYPE_CODE[out.dtype], t.shape[1])


def _launch(entry, args: bytes, dev: torch.device) -> int:
    """``entry(args, stream)`` on ``dev`` and its current stream."""
    if _get_device is not None and _get_device() == dev.index:
        return entry(args, _lib.stream_of(dev))
    with device_ctx(dev):
        return entry(args, _lib.stream_of(dev))


def _back(out: torch.Tensor, given: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """``out``, which lies on ``dev``, in ``given``'s type where that is one of floating numbers, and where ``given`` lies."""
    if out.dtype is not given.dtype and given.dtype.is_floating_point:
        out = out.to(given.dtype)
    return out if given.is_cuda and given.get_device() == dev.index else back(out, given.device)


def _table_checked(t: torch.Tensor, dev: torch.device, name: str) -> torch.Tensor:
    if t.dim() != 2:
        raise ValueError(f"{name} must be [max_positions, rotary_dim / 2], got {tuple(t.shape)}")
    if t.dtype is not torch.float32 or not t.is_cuda or t.get_device() != dev.index or not t.is_contiguous():
        t = t.detach().to(device=dev, dtype=torch.float32).contiguous()
    return t


def _rope_fields(cos, sin, positions, B: int, S: int, D: int, interleaved: bool, inverse: bool, dev: torch.device):
    """The ``skv_rope`` fields, and the tensors they point into (to be kept until the launch)."""
    cos, sin = _table_checked(cos, dev, "cos"), _table_checked(sin, dev, "sin")
    count, half = cos.shape
    if sin.shape != (count, half):
        raise ValueError(f"cos/sin shapes disagree: {tuple(cos.shape)} vs {tuple(sin.shape)}")
    if half < 1 or 2 * half > D:
        raise ValueError(f"the tables rotate {2 * half} values of a head of {D}")
    if positions is None:
        return (cos.data_ptr(), sin.data_ptr(), 0, 0, 0, 0, 2 * half, count, interleaved, inverse, 0), (cos, sin)
    if positions.dtype is torch.int64:
        size = 8
    elif positions.dtype is torch.int32:
        size = 4
    else:
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    if not positions.is_cuda or positions.get_device() != dev.index:
        positions = positions.to(dev)
    if positions.shape != (B, S):
        try:
            positions = positions.expand(B, S)
        except RuntimeError:
            raise ValueError(f"positions must broadcast to [{B}, {S}], got {tuple(positions.shape)}") from None
    st = positions.stride()
    return ((cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), st[0], st[1], size, 2 * half, count, interleaved, inverse, 0),
            (cos, sin, positions))


class _Turn(torch.autograd.Function):
    """``apply_rotary`` of rows that a gradient is wanted of: it is the gradient of the result, turned the other way."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(cos, sin, *(() if positions is None else (positions,)))
        ctx.how = dict(interleaved=interleaved, inverse=not inverse)
        return apply_rotary(q, cos, sin, k, positions, interleaved, inverse)

    @staticmethod
    def backward(ctx, gq, gk=None):
        cos, sin, *positions = ctx.saved_tensors
        how = dict(ctx.how, positions=positions[0] if positions else None)
        if gq is not None and gk is not None:
            gq, gk = apply_rotary(gq, cos, sin, gk, **how)
        elif gq is not None:
            gq = apply_rotary(gq, cos, sin, **how)
        elif gk is not None:
            gk = apply_rotary(gk, cos, sin, **how)
        return gq, gk, None, None, None, None, None


def apply_rotary(
    q: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    k: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    inverse: bool = False,
):
    """``q`` (and ``k``) ``[B, heads, S, D]`` turned by their positions; returns ``q'``, or ``(q', k')`` with ``k``.

    A pair ``(a, b)`` at position p becomes ``(a c - b s, b c + a s)`` with ``c, s = cos[p][i], sin[p][i]``.  Pairs
    are ``(x[i], x[i + rot/2])``, or ``(x[2i], x[2i+1])`` with ``interleaved``, over the first
    ``rot = 2 * cos.shape[1]`` values of a head; the others are copied.  ``positions``: int32 or int64, broadcast to
    ``[B, S]`` (default: 0 .. S-1); rows whose position the tables do not hold become NaN.
    ``inverse`` turns by minus the angle: the gradient with respect to the rows, and, where the tables have no gain (that of
    ``"ntk_parts"`` comes in a second time), back.  Rows that require a gradient get theirs; the tables get none.

    fp32, fp16 and bf16 rows are read in place with any strides over the first three dimensions
    (slices of one projection's output, transposed views); products and sums are fp32, rounded once to the
    rows' type.  One launch for both tensors.
    """
    shape = q.shape
    if len(shape) != 4:
        raise ValueError(f"q must be 4-D [batch, heads, seq, head_dim], got shape {tuple(q.shape)}")
    B, _, S, D = shape
    if k is not None and (k.dim() != 4 or k.shape != (B, k.shape[1], S, D)):
        raise ValueError(f"q/k shapes disagree: {tuple(q.shape)} vs {tuple(k.shape)}")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Turn.apply(q, k, cos, sin, positions, interleaved, inverse)
    dev = q.device if q.is_cuda else compute_device(k, cos)
    qd, q_rows = _rows(q, dev, _common(q, k))
    q_out, q_out_rows = _like(qd)
    kd = k_out = None
    k_rows = k_out_rows = _NO_ROWS
    if k is not None:
        kd, k_rows = _rows(k, dev, qd.dtype)
        k_out, k_out_rows = _like(kd)
    rope, keep = _rope_fields(cos, sin, positions, B, S, D, bool(interleaved), bool(inverse), dev)
    args = _ARGS.pack(*q_rows, *k_rows, *q_out_rows, *k_out_rows, *rope, B, S, D, 0)
    st = _launch(_lib.load().skv_rotary, args, dev)
    if st:
        _lib.check(st, "apply_rotary")
    del keep, kd
    if k is None:
        return _back(q_out, q, dev)
    return _back(q_out, q, dev), _back(k_out, k, dev)
