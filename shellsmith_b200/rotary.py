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
import functools
import math

import torch

from . import _capi, paged
from ._torch import fast, on_device, require_cuda, stream_of


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
        self.device_index = self.turns.get_device()
        self._home = stream_of(self.turns) if self.turns.is_cuda else 0
        self.turns_ptr, self.axis_ptr = self.turns.data_ptr(), self.axis.data_ptr()
        self.packed = (head_dim, rot, self.axes, self.turns_ptr, self.axis_ptr, self.device_index,
                       self._home, self.turns, self.axis)

    def used(self) -> None:
        """A call on the current stream reads the tables: if they came from another stream, the
        allocator does not hand their memory out before the call is done."""
        if stream_of(self.turns) != self._home:
            stream = torch.cuda.current_stream(self.device_index)
            self.turns.record_stream(stream)
            self.axis.record_stream(stream)


def axis_of_pairs(sections, interleaved: bool) -> list:
    """The position axis of each frequency pair."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    half, count = sum(sections), len(sections)
    return [i % count if i < count * sections[i % count] else 0 for i in range(half)]


_append = _capi.bind("sc_rotary_append")


@functools.lru_cache(maxsize=256)
def _strides(*values) -> ctypes.Array:
    return (ctypes.c_int64 * 6)(*values)


def _operand(name: str, t: torch.Tensor, dim: int) -> tuple:
    """Shape and strides of a [ntok, heads, D] bf16 operand."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the product path has no CPU fallback)")
    if t.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be torch.bfloat16, got {t.dtype}")
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != dim:
        raise ValueError(f"{name} must be [ntok, heads, {dim}], got {tuple(shape)}")
    if stride[2] != 1 and t.numel():
        raise ValueError(f"{name} must be contiguous along the head dimension")
    return shape, stride


def _weight(name: str, w: torch.Tensor | None, dim: int) -> int | None:
    if w is None:
        return None
    require_cuda(name, w, torch.bfloat16, 1)
    if w.shape[0] != dim:
        raise ValueError(f"{name} must have {dim} entries")
    return w.data_ptr()


def _run(q, k, v, k_shape, strides, positions, plan, q_weight, k_weight, eps, q_out, k_out, pool,
         slots, page, pages) -> None:
    dim, ntok = plan.head_dim, q.shape[0]
    if k_shape[0] != ntok:
        raise ValueError("rotary: q and k must have the same tokens")
    shape, pos_stride = positions.shape, positions.stride()
    if len(shape) == 1:
        shape, pos_stride = (1, *shape), (0, *pos_stride)
    if (positions.dtype is not torch.int32 or not positions.is_cuda or len(shape) != 2
            or shape[0] != plan.axes or shape[1] != ntok or (ntok > 1 and pos_stride[1] != 1)):
        raise ValueError(f"positions must be CUDA int32 [{plan.axes}, {ntok}] (one row per axis), "
                         f"got {positions.dtype} {tuple(positions.shape)}")
    if plan.device_index != q.get_device():
        raise ValueError(f"the plan is on {plan.turns.device}, q on {q.device}")
    on_device(plan.device_index, k=k, positions=positions, q_weight=q_weight, k_weight=k_weight)
    plan.used()
    _append(q.data_ptr(), k.data_ptr(), v, _strides(*strides), positions.data_ptr(), pos_stride[0],
            plan.axes, plan.turns_ptr, plan.axis_ptr, _weight("q_weight", q_weight, dim),
            _weight("k_weight", k_weight, dim), eps, q_out.data_ptr(), k_out, pool, slots, ntok,
            q.shape[1], k_shape[1], dim, plan.rotary_dim, page, pages, stream_of(q))


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, plan: RotaryPlan, *,
           q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
           eps: float = 1e-6) -> tuple:
    """Norm (where a weight is given) and turn q [ntok, Hq, D] and k [ntok, Hkv, D].

    positions: int32 [axes, ntok] (or [ntok] for one axis). q and k may be strided
    views with a contiguous last dimension. Returns new contiguous (q, k).
    """
    q_shape, qs = _operand("q", q, plan.head_dim)
    k_shape, ks = _operand("k", k, plan.head_dim)
    q_out, k_out = q.new_empty(q_shape), k.new_empty(k_shape)
    _run(q, k, None, k_shape, (qs[0], qs[1], ks[0], ks[1], 0, 0), positions, plan, q_weight,
         k_weight, eps, q_out, k_out.data_ptr(), None, None, 0, 0)
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
    if fast is not None:
        done = fast.rotary_append(q, k, v, positions, kv_pool, slot_mapping, q_weight, k_weight,
                                  eps, out, plan.packed)
        if done is not None:
            return done
    q_shape, qs = _operand("q", q, plan.head_dim)
    k_shape, ks = _operand("k", k, plan.head_dim)
    v_shape, vs = _operand("v", v, plan.head_dim)
    if v_shape != k_shape:
        raise ValueError("rotary_append: k and v must have the same shape")
    pages, hkv, page, dim = paged._pool_dims(kv_pool)
    require_cuda("slot_mapping", slot_mapping, torch.int64, 1, align=8)
    if k_shape[1] != hkv or k_shape[2] != dim or slot_mapping.shape[0] != k_shape[0]:
        raise ValueError("rotary_append: k/v must be [ntok, Hkv, D] with one slot per token")
    on_device(plan.device_index, v=v, kv_pool=kv_pool, slot_mapping=slot_mapping, out=out)
    if out is not None:
        require_cuda("out", out, torch.bfloat16, 3)
        if out.shape != q_shape:
            raise ValueError("rotary_append: out must have q's shape")
    if kv_pool.dtype is torch.uint8:
        q_out, k_out = rotary(q, k, positions, plan, q_weight=q_weight, k_weight=k_weight, eps=eps)
        if not v.is_contiguous() or v.data_ptr() % 16:  # one token's view may be off a boundary
            v = v.clone(memory_format=torch.contiguous_format)
        paged.kv_append(k_out, v, kv_pool, slot_mapping)
        return q_out if out is None else out.copy_(q_out)
    if out is None:
        out = q.new_empty(q_shape)
    _run(q, k, v.data_ptr(), k_shape, (qs[0], qs[1], ks[0], ks[1], vs[0], vs[1]), positions, plan,
         q_weight, k_weight, eps, out, None, kv_pool.data_ptr(), slot_mapping.data_ptr(), page,
         pages)
    return out
