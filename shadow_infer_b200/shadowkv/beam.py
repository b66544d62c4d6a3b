"""Beam search over a page pool: the best continuations of every search, and sequences that go on from others.

The reference generates by denoising and has no search (shadowinfer/execution/blockwise_generate.py); a pool's sequences are the
states of one.  A step selects (``beam_select``), lets every beam's pages follow its parent (``paged_reorder``), appends the
chosen tokens' keys and values and attends.  Nothing waits for the GPU and all of it can be captured in a CUDA graph;
``PagedKVPool.fork`` and ``PagedKVPool.reorder`` do the bookkeeping.
"""

from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from .. import _lib
from .._device import back, compute_device, device_ctx
from .paged_pool import _POOL, _flag, _index, _pool_fields, _raise_flag, _workspace
from .page_selection import _bounds_checked
from .rotary import _DTYPE_CODE, _launch

_BEAM = struct.Struct("<QqqQQQQQQqiiiiii")
_REORDER = struct.Struct("<" + _POOL + "QQQQQQQii")
assert (_BEAM.size, _REORDER.size) == (104, 144)
_SCRATCH_BYTES = {}   # (device, B, beams, V, keep) -> the selection's scratch


def beam_select(
    logits: torch.Tensor,
    scores: torch.Tensor,
    keep: Optional[int] = None,
    finished: Optional[torch.Tensor] = None,
    pad_token: int = 0,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``keep`` best continuations of each search: ``(scores, parents, tokens)``, each ``[B, keep]``, best first.

    ``logits`` ``[B, beams, V]`` (fp32, fp16 or bf16, other types as fp32; any strides over the first two dimensions) are those of each beam's next
    token, ``scores`` ``[B, beams]`` the beams' log-probabilities so far.  A continuation scores
    ``scores[b, r] + log_softmax(logits[b, r])[token]``; scores are compared in 64 bits, a beam's own continuations by their logits, and
    ties go to the lowest beam, then to the lowest token.  A row's exponentials are 32-bit numbers, so the logarithm of their sum is up to 2^-19 off,
    by the same for equal rows of a call: their continuations tie, others of different beams that are nearer than that may change places.
    ``parents`` and ``tokens`` are int64, the new scores float32.  ``keep`` (at most 128)
    defaults to the number of beams; a search that sets beams aside as they end wants twice as many.

    A ``finished`` beam (bool ``[B, beams]``) has a single continuation: ``pad_token``, at the score that it has.
    Tokens that are not allowed have logits of -inf; a NaN counts as one, and logits of +inf share their beam's whole probability.
    A beam whose score is not finite (a search that starts from one beam gives the others -inf), or to which no token is allowed,
    has continuations of -inf only.  Where fewer than ``keep`` are better, the first of those fill up the result.  One launch, or two.
    """
    if logits.dim() != 3:
        raise ValueError(f"logits must be [batch, beams, vocabulary], got {tuple(logits.shape)}")
    B, beams, V = logits.shape
    if scores.shape != (B, beams):
        raise ValueError(f"scores must be {[B, beams]}, got {tuple(scores.shape)}")
    keep = beams if keep is None else int(keep)
    if beams < 1 or V < 1 or not 1 <= keep <= min(128, beams * V):
        raise ValueError(f"keep must be in [1, min(128, {beams} beams x {V} tokens)], got {keep}")
    if finished is not None and (finished.shape != (B, beams) or finished.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f"finished must be bool {[B, beams]}, got {tuple(finished.shape)} {finished.dtype}")
    if finished is not None and not 0 <= pad_token < V:
        raise ValueError(f"pad_token {pad_token} is not in a vocabulary of {V}")
    dev = logits.device if logits.is_cuda else compute_device(scores)
    x, code = logits, _DTYPE_CODE.get(logits.dtype)
    if code is None or not x.is_cuda or x.requires_grad:
        x = x.detach().to(device=dev, dtype=x.dtype if code is not None else torch.float32)
        code = _DTYPE_CODE[x.dtype]
    sb, sr, sv = x.stride()
    if sv != 1 and V != 1:
        x = x.contiguous()
        sb, sr, sv = x.stride()
    cum = scores
    if cum.dtype is not torch.float32 or not cum.is_contiguous() or cum.get_device() != dev.index or cum.requires_grad:
        cum = cum.detach().to(device=dev, dtype=torch.float32).contiguous()
    done = finished
    if done is not None and (done.get_device() != dev.index or not done.is_contiguous()):
        done = done.to(dev).contiguous()
    values = torch.empty(B, keep, dtype=torch.float32, device=dev)
    parents = torch.empty(B, keep, dtype=torch.int64, device=dev)
    tokens = torch.empty(B, keep, dtype=torch.int64, device=dev)
    lib = _lib.load()
    with device_ctx(dev):   # (the size depends on the device's SMs)
        stream = _lib.stream_of(dev)
        need = _SCRATCH_BYTES.get((dev.index, B, beams, V, keep))
        if need is None:
            if len(_SCRATCH_BYTES) > 4096:   # (sizes that a server has met: not more than some)
                _SCRATCH_BYTES.clear()
            need = _SCRATCH_BYTES[dev.index, B, beams, V, keep] = max(16, lib.skv_beam_scratch_bytes(B, beams, V, keep))
        scratch = _workspace("beam", dev, stream, need)
        st = lib.skv_beam_select(_BEAM.pack(
            x.data_ptr(), sb, sr, cum.data_ptr(), 0 if done is None else done.data_ptr(), values.data_ptr(), parents.data_ptr(),
            tokens.data_ptr(), scratch.data_ptr(), scratch.numel(), code, B, beams, V, keep, pad_token if finished is not None else 0),
            stream)
    if st:
        _lib.check(st, "beam_select")
    del x, cum, done
    if logits.is_cuda:
        return values, parents, tokens
    return back(values, logits.device), back(parents, logits.device), back(tokens, logits.device)


def paged_reorder(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    parents: torch.Tensor,
    scale_k: Optional[torch.Tensor] = None,
    scale_v: Optional[torch.Tensor] = None,
    bounds: Optional[torch.Tensor] = None,
    steps: Optional[torch.Tensor] = None,
    head_dim: Optional[int] = None,
    check: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Sequences go on from others of their group; returns the new ``(block_table, lengths)``, int32.

    ``parents`` ``[groups, beams]`` (int32 or int64, as from ``beam_select``; ``groups * beams`` is the pool's batch, sequence
    ``g * beams + c`` is beam c of group g): beam c goes on from beam ``parents[g, c]`` and gets its pages and length (table
    entries behind the tokens, pages taken ahead, stay each beam's own).  Pages that are full are shared from then on.  A last page that
    is partly filled must be its sequence's own, and the beams of a group equally long: of a parent's children, the parent itself keeps
    the page, else the first child does, and the n-th beam of the group that keeps none is given the page that the n-th beam without
    children has there, with the tokens (and the page's ``bounds`` / ``steps``, where given) copied.  So no page is allocated, every
    sequence's last page is its own again, and nothing waits for the host; the pages of ended beams belong to their group until all of
    it ends.

    Pages are changed in place, the tables are new tensors.  A parent outside its group leaves an empty sequence, a last page
    that cannot be had a table entry of -1 (beams that are not equally long: a full page may be shared and is never given away, and entries
    that held a longer beam's own tokens are -1); ``check=True`` waits and raises ``ValueError`` for them.  One launch.
    """
    if parents.dim() != 2:
        raise ValueError(f"parents must be [groups, beams], got {tuple(parents.shape)}")
    groups, beams = parents.shape
    B = groups * beams
    if parents.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"parents must be int32 or int64, got {parents.dtype}")
    pool, dev, table = _pool_fields(k_pages, v_pages, block_table, scale_k, scale_v, B, head_dim)
    lens = _index(lengths, (B,), dev, "lengths")
    if (bounds is None) != (steps is None):
        raise ValueError("bounds and steps must be given together")
    if bounds is not None:
        _bounds_checked(bounds, steps, (pool[7], pool[9], 2, pool[10]), dev)
    new_table = torch.empty_like(table, memory_format=torch.contiguous_format)
    new_lengths = torch.empty_like(lens)
    if B == 0:
        return new_table, new_lengths
    from_ = parents
    if from_.get_device() != dev.index or not from_.is_contiguous():
        from_ = from_.to(dev).contiguous()
    flag = _flag(check, dev)
    args = _REORDER.pack(*pool, lens.data_ptr(), from_.data_ptr(), new_table.data_ptr(), new_lengths.data_ptr(),
                         0 if bounds is None else bounds.data_ptr(), 0 if steps is None else steps.data_ptr(),
                         0 if flag is None else flag.data_ptr(), 8 if from_.dtype is torch.int64 else 4, beams)
    st = _launch(_lib.load().skv_pool_reorder, args, dev)
    if st:
        _lib.check(st, "paged_reorder")
    del table, lens, from_
    if flag is not None:
        _raise_flag(flag, "paged_reorder")
    return new_table, new_lengths
