"""Rotary positions with several axes, the q/k norm and the KV append (device side).

The reference hands each attention layer's projections to mlx-vlm's
`_prepare_projected_qkv` (studio_compute/mlx_decode.py:94-100): per-head RMS norm
of q and k, rotary positions (time, height, width for images and video) and the
cache write. Here that is one launch over any number of tokens, decode rows and
packed prompts alike:

  RotaryPlan      the frequencies of a model's rotary positions, laid out once
  rotary_append   norm, turn, write k/v through a slot mapping; returns q
  rotary          norm and turn only; returns (q, k)
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _capi, paged
from ._torch import ptr, require_cuda, stream_of


class RotaryPlan:
    """Which axis and frequency turn each pair (i, i + rotary_dim / 2) of a head.

    sections: frequency pairs of each position axis, summing to rotary_dim / 2
    (None: one axis). Without `interleaved` they follow one another; with it pair i
    takes axis i mod A while that axis has pairs left, and axis 0 otherwise.
    inv_freq: the rotary_dim / 2 frequencies (default base^(-2i / rotary_dim)).
    """

    def __init__(self, head_dim: int, rotary_dim: int | None = None, base: float = 10000.0,
                 sections=None, interleaved: bool = False, inv_freq=None,
                 device: str | torch.device = "cuda"):
        rot = head_dim if rotary_dim is None else rotary_dim
        if head_dim not in (64, 128, 256):
            raise ValueError(f"RotaryPlan: head_dim must be 64, 128 or 256, got {head_dim}")
        if rot < 16 or rot % 16 or rot > head_dim:
            raise ValueError("RotaryPlan: rotary_dim must be a multiple of 16 in [16, head_dim], "
                             f"got {rot}")
        half = rot // 2
        sections = [half] if sections is None else [int(s) for s in sections]
        if not sections or min(sections) < 0 or sum(sections) != half:
            raise ValueError(f"RotaryPlan: sections must sum to {half}, got {sections}")
        if inv_freq is None:
            inv_freq = [float(base) ** (-i / half) for i in range(half)]
        else:
            inv_freq = [float(f) for f in inv_freq]
            if len(inv_freq) != half:
                raise ValueError(f"RotaryPlan: {half} frequencies are needed, got {len(inv_freq)}")
        self.head_dim, self.rotary_dim, self.axes = head_dim, rot, len(sections)
        self.sections, self.interleaved = tuple(sections), bool(interleaved)
        self.axis = torch.tensor(axis_of_pairs(sections, interleaved), dtype=torch.int32,
                                 device=device)
        self.inv_freq = torch.tensor(inv_freq, dtype=torch.float64)
        self.turns = (self.inv_freq / (2 * math.pi)).to(device)  # whole turns per position


def axis_of_pairs(sections, interleaved: bool) -> list:
    """The position axis of each frequency pair."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    half, count = sum(sections), len(sections)
    return [i % count if i < count * sections[i % count] else 0 for i in range(half)]


def _operand(name: str, t: torch.Tensor, plan: RotaryPlan) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the product path has no CPU fallback)")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be torch.bfloat16, got {t.dtype}")
    if t.dim() != 3 or t.shape[2] != plan.head_dim:
        raise ValueError(f"{name} must be [ntok, heads, {plan.head_dim}], got {tuple(t.shape)}")
    if t.stride(2) != 1 and t.numel():
        raise ValueError(f"{name} must be contiguous along the head dimension")


def _run(q, k, v, positions, plan, q_weight, k_weight, eps, q_out, k_out, pool, slots) -> None:
    _operand("q", q, plan)
    _operand("k", k, plan)
    ntok, hq, dim = q.shape
    hkv = k.shape[1]
    if k.shape[0] != ntok:
        raise ValueError("rotary: q and k must have the same tokens")
    if positions.dim() == 1:
        positions = positions[None]
    if (positions.dtype != torch.int32 or not positions.is_cuda
            or tuple(positions.shape) != (plan.axes, ntok)
            or (ntok > 1 and positions.stride(1) != 1)):
        raise ValueError(f"positions must be CUDA int32 [{plan.axes}, {ntok}] (one row per axis), "
                         f"got {positions.dtype} {tuple(positions.shape)}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            require_cuda(name, w, torch.bfloat16, 1)
            if w.shape[0] != dim:
                raise ValueError(f"{name} must have {dim} entries")
    if plan.turns.device != q.device:
        raise ValueError(f"the plan is on {plan.turns.device}, q on {q.device}")
    pages, page = (0, 0) if pool is None else (pool.shape[0], pool.shape[3])
    vs = (0, 0) if v is None else v.stride()
    strides = (ctypes.c_int64 * 6)(q.stride(0), q.stride(1), k.stride(0), k.stride(1), vs[0], vs[1])
    _capi.call("sc_rotary_append", ptr(q), ptr(k), ptr(v), strides, ptr(positions),
               positions.stride(0), plan.axes, ptr(plan.turns), ptr(plan.axis), ptr(q_weight),
               ptr(k_weight), float(eps), ptr(q_out), ptr(k_out), ptr(pool), ptr(slots), ntok, hq,
               hkv, dim, plan.rotary_dim, page, pages, stream_of(q))


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, plan: RotaryPlan, *,
           q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
           eps: float = 1e-6) -> tuple:
    """Norm (where a weight is given) and turn q [ntok, Hq, D] and k [ntok, Hkv, D].

    positions: int32 [axes, ntok] (or [ntok] for one axis). q and k may be strided
    views with a contiguous last dimension. Returns new contiguous (q, k).
    """
    _operand("q", q, plan)
    _operand("k", k, plan)
    q_out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    k_out = torch.empty(k.shape, dtype=torch.bfloat16, device=k.device)
    _run(q, k, None, positions, plan, q_weight, k_weight, eps, q_out, k_out, None, None)
    return q_out, k_out


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                  plan: RotaryPlan, kv_pool: torch.Tensor, slot_mapping: torch.Tensor, *,
                  q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                  eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """rotary() and paged.kv_append of the turned k and of v, in one launch; returns q.

    slot_mapping [ntok] int64 as in kv_append (< 0: nothing is written for that token;
    its q is still turned). An 8-bit pool takes the turned k from a scratch tensor
    through its own append kernel (two launches).
    """
    _operand("v", v, plan)
    if v.shape != k.shape:
        raise ValueError("rotary_append: k and v must have the same shape")
    num_pages, hkv, page, dim = paged._pool_dims(kv_pool)
    require_cuda("slot_mapping", slot_mapping, torch.int64, 1, align=8)
    if k.shape[1:] != (hkv, dim) or slot_mapping.shape[0] != k.shape[0]:
        raise ValueError("rotary_append: k/v must be [ntok, Hkv, D] with one slot per token")
    if kv_pool.dtype == torch.uint8:
        q_out, k_out = rotary(q, k, positions, plan, q_weight=q_weight, k_weight=k_weight, eps=eps)
        paged.kv_append(k_out, v.contiguous(), kv_pool, slot_mapping)
        return q_out if out is None else out.copy_(q_out)
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    else:
        require_cuda("out", out, torch.bfloat16, 3)
        if out.shape != q.shape:
            raise ValueError("rotary_append: out must have q's shape")
    _run(q, k, v, positions, plan, q_weight, k_weight, eps, out, None, kv_pool, slot_mapping)
    return out
