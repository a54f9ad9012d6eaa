"""Beam selection and the reordering of per-sequence state rows (device side).

The reference samples one token per request (studio_compute/inference.py:176-218);
several beams over one cache also need, after each step,

  beam_select    the best continuations over a group's beams and the vocabulary
  reorder_rows   state rows (GDN state, conv taps) that follow their beams

Both run on the device without a synchronisation: parents and new slots go from one
call to the next as tensors. plan_reorder is the same slot rule on the host, for the
page tables (engine.HybridCacheEngine.reorder).
"""

from __future__ import annotations

import ctypes
import functools
import operator

import numpy as np
import torch

from . import _capi
from ._torch import fast, on_device, ptr, require_cuda, stream_of

MAX_BEAMS = 64   # beams of one group
MAX_SELECT = 64  # continuations asked for at once

_select = _capi.bind("sc_beam_select")
_reorder = _capi.bind("sc_reorder_rows")
_Pointers, _Sizes, _Layers = ctypes.c_void_p * 4, ctypes.c_int64 * 4, ctypes.c_int * 4


@functools.lru_cache(maxsize=256)
def _workspace(groups: int, beams: int, vocab: int, n: int, fp32: int) -> int:
    return _capi.lib().sc_beam_select_workspace(groups, beams, vocab, n, fp32)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: int, *,
                finished: torch.Tensor | None = None, pad_token: int = 0) -> tuple:
    """The n best continuations of each group's beams.

    logits [G, K, V] bf16 or fp32 (contiguous along V, rows evenly spaced), scores
    [G, K] fp32 the beams' summed log-probabilities (-inf: the beam is dead). The score
    of token v after beam k is scores[k] + log_softmax(logits[k])[v] in fp32; the result
    is ordered by score, equal ones by the lower beam, then the lower token. finished
    [G, K] bool: such a beam's only continuation is pad_token, its score unchanged.
    Returns (scores fp32, parents int32, tokens int32), each [G, n]. Where fewer than n
    continuations have a score above -inf, those of lowest index follow with -inf (a NaN
    score counts as -inf).
    """
    if fast is not None:
        done = fast.beam_select(logits, scores, n, finished, pad_token)
        if done is not None:
            return done
    if not isinstance(logits, torch.Tensor) or logits.dim() != 3:
        raise ValueError("beam_select: logits must be a [groups, beams, vocab] tensor")
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor (the product path has no CPU fallback)")
    fp32 = logits.dtype is torch.float32
    if not fp32 and logits.dtype is not torch.bfloat16:
        raise TypeError(f"logits must be bfloat16 or float32, got {logits.dtype}")
    for name, value in (("n", n), ("pad_token", pad_token)):
        if not -1 << 31 <= operator.index(value) < 1 << 31:  # it would wrap on its way
            raise ValueError(f"beam_select: {name}={value} does not fit 32 bits")
    if n < 0:
        raise ValueError(f"beam_select: n={n}")
    groups, beams, vocab = logits.shape
    if beams < 1 or vocab < 1:
        raise ValueError("beam_select: at least one beam and one token")
    stride = vocab
    if not logits.is_contiguous() and groups:
        across, stride, step = logits.stride()
        if beams == 1:
            stride = across if groups > 1 else vocab
        if (step != 1 and vocab > 1) or stride < vocab or (groups > 1 and across != beams * stride):
            raise ValueError(
                "beam_select: logits need a contiguous vocabulary and evenly spaced rows")
    require_cuda("scores", scores, torch.float32, 2, align=4)
    if scores.shape != (groups, beams):
        raise ValueError(f"scores must be [{groups}, {beams}], got {tuple(scores.shape)}")
    if finished is not None:
        require_cuda("finished", finished, torch.bool, 2, align=1)
        if finished.shape != (groups, beams):
            raise ValueError(f"finished must be [{groups}, {beams}], got {tuple(finished.shape)}")
    on_device(logits.get_device(), scores=scores, finished=finished)
    need = _workspace(groups, beams, vocab, n, int(fp32))
    work = scores.new_empty(need // 4)
    best, parents, tokens = scores.new_empty((3, groups, n)).unbind(0)
    parents, tokens = parents.view(torch.int32), tokens.view(torch.int32)
    _select(logits.data_ptr(), fp32, stride, scores.data_ptr(), ptr(finished), pad_token,
            best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), work.data_ptr(), need, groups,
            beams, vocab, n, stream_of(logits))
    return best, parents, tokens


def reorder_rows(pools, slots: torch.Tensor, parents: torch.Tensor) -> torch.Tensor:
    """Let each group's state rows follow their beams, in place; returns the new slots.

    pools: up to four contiguous tensors [layers, rows, ...] (any type, rows of a
    multiple of 16 bytes); beam k of group g holds row slots[g, k] of every layer (all
    slots distinct). Child j continues beam parents[g, j]: the first child of a beam
    keeps the beam's row, each later child gets a copy in the row of a beam without
    children (ascending), so nothing else moves. slots, parents, result: int32 [G, K].
    """
    if fast is not None:
        done = fast.reorder_rows(pools, slots, parents)
        if done is not None:
            return done
    require_cuda("slots", slots, torch.int32, 2, align=4)
    require_cuda("parents", parents, torch.int32, 2, align=4)
    groups, beams = shape = slots.shape
    if parents.shape != shape:
        raise ValueError("reorder_rows: slots and parents must have the same shape")
    pools = list(pools)
    count = len(pools)
    if count > 4:
        raise ValueError(f"reorder_rows: at most 4 pools, got {count}")
    rows, bases, sizes, layers = None, _Pointers(), _Sizes(), _Layers()
    for i, pool in enumerate(pools):
        if not isinstance(pool, torch.Tensor) or not pool.is_cuda or pool.dim() < 2:
            raise ValueError(f"reorder_rows: pool {i} must be a CUDA tensor [layers, rows, ...]")
        if not pool.is_contiguous():
            raise ValueError(f"reorder_rows: pool {i} must be contiguous")
        size = pool.shape
        if rows is not None and rows != size[1]:
            raise ValueError("reorder_rows: every pool must have the same rows")
        rows = size[1]
        bases[i], layers[i] = pool.data_ptr(), size[0]
        sizes[i] = pool.stride(1) * pool.element_size()
    on_device(slots.get_device(), parents=parents, **{f"pool {i}": p for i, p in enumerate(pools)})
    out = torch.empty_like(slots)
    if rows is None:  # the new slots alone: any slot is in range
        rows = (1 << 31) - 1
    _reorder(bases, sizes, layers, count, rows, slots.data_ptr(), parents.data_ptr(),
             out.data_ptr(), groups, beams or 1, stream_of(slots))
    return out


def plan_reorder(slots, parents) -> tuple:
    """reorder_rows' slot rule for one group on the host: (new slots, [(source, destination)])."""
    slots, parents = [int(s) for s in slots], [int(p) for p in parents]
    free = [slots[b] for b in range(len(slots)) if b not in set(parents)]
    new, copies, seen = [], [], set()
    for p in parents:
        if p in seen:
            copies.append((slots[p], free.pop(0)))
            new.append(copies[-1][1])
        else:
            new.append(slots[p])
        seen.add(p)
    return np.asarray(new, np.int64), copies
