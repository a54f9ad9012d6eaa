"""The cache path's C ABI registered as PyTorch operators: torch.ops.shellcache.*.

Each operator calls the same libshellcache.so entry point as the Python shims
(numerics, paged) and has a fake (meta) kernel, so shapes and dtypes propagate
under FakeTensorMode and torch.compile tracing without running a kernel. State
and page pools are mutated in place, as the C ABI does; an operator never
returns an alias of its inputs, so the ones the reference names with a
(output, next_state) result return the output and advance `state`.

  shellcache::gdn_decode                 sc_gdn_decode / _bf16 (numerics.gdn_decode)
  shellcache::gated_delta_token          gdn_token.py:18-42 call site, state in place
  shellcache::gated_delta_chunked        ops.py:151 call site, fp32 state in place
  shellcache::gated_delta_chunks         gdn_fused.py:86-122 call site, fp32 state in place
  shellcache::kv_append                  sc_kv_append / _q8
  shellcache::paged_decode_attention     sc_paged_decode_attention / _q8
  shellcache::paged_decode_attention_fused  append + split-K + merge in one launch
  shellcache::rotary_append              sc_rotary (rotary.rotary_append)
  shellcache::shared_prefix_attention    sc_shared_prefix_attention
  shellcache::beam_select                sc_beam_select
  shellcache::reorder_rows               sc_reorder_rows

Importing this module registers the operators (once per process).
"""

from __future__ import annotations

import functools
from typing import List, Optional, Tuple

import torch

from . import beam, numerics, paged, rotary

_LIB = "shellcache"


@torch.library.custom_op(f"{_LIB}::gdn_decode", mutates_args=("state",))
def gdn_decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
               beta: torch.Tensor, state: torch.Tensor,
               state_slot: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One-token GDN update of rows b (state row state_slot[b]); returns out [B, Hv, dv]."""
    return numerics.gdn_decode(q, k, v, g, beta, state, state_slot)


@gdn_decode.register_fake
def _(q, k, v, g, beta, state, state_slot=None):
    return q.new_empty((q.shape[0], v.shape[1], v.shape[2]), dtype=torch.bfloat16)


@torch.library.custom_op(f"{_LIB}::gated_delta_token", mutates_args=("state_BHVK",))
def gated_delta_token(q_BLJK: torch.Tensor, k_BLJK: torch.Tensor, v_BLHV: torch.Tensor,
                      g_BLH: torch.Tensor, beta_BLH: torch.Tensor,
                      state_BHVK: torch.Tensor) -> torch.Tensor:
    """The reference's token step; returns out [B, 1, Hv, dv] and advances the state."""
    out, _ = numerics.gated_delta_token(q_BLJK, k_BLJK, v_BLHV, g_BLH, beta_BLH, state_BHVK)
    return out


@gated_delta_token.register_fake
def _(q_BLJK, k_BLJK, v_BLHV, g_BLH, beta_BLH, state_BHVK):
    return v_BLHV.new_empty(v_BLHV.shape, dtype=torch.bfloat16)


def _require_fp32_state(state: torch.Tensor, name: str) -> None:
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"shellcache::{name} advances a contiguous fp32 state in place")


@torch.library.custom_op(f"{_LIB}::gated_delta_chunked", mutates_args=("state",))
def gated_delta_chunked(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                        beta: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
    """The reference's chunked recurrence; returns y [B, T, Hv, dv], state in place."""
    _require_fp32_state(state, "gated_delta_chunked")
    y, _ = numerics.gated_delta_chunked(q, k, v, g, beta, state)
    return y


@gated_delta_chunked.register_fake
def _(q, k, v, g, beta, state):
    return v.new_empty(v.shape)


@torch.library.custom_op(f"{_LIB}::gated_delta_chunks", mutates_args=("state",))
def gated_delta_chunks(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, a: torch.Tensor,
                       b: torch.Tensor, a_log: torch.Tensor, dt_bias: torch.Tensor,
                       state: torch.Tensor) -> torch.Tensor:
    """The reference's chunked prefill from gate logits; returns y, state in place."""
    _require_fp32_state(state, "gated_delta_chunks")
    y, _ = numerics.gated_delta_chunks(q, k, v, a, b, a_log, dt_bias, state)
    return y


@gated_delta_chunks.register_fake
def _(q, k, v, a, b, a_log, dt_bias, state):
    return v.new_empty(v.shape, dtype=torch.bfloat16)


@torch.library.custom_op(f"{_LIB}::kv_append", mutates_args=("kv_pool",))
def kv_append(k: torch.Tensor, v: torch.Tensor, kv_pool: torch.Tensor,
              slot_mapping: torch.Tensor) -> None:
    """Write k/v [ntok, Hkv, D] into the pool at slot_mapping (int64, < 0 skips)."""
    paged.kv_append(k, v, kv_pool, slot_mapping)


@kv_append.register_fake
def _(k, v, kv_pool, slot_mapping):
    return None


@torch.library.custom_op(f"{_LIB}::paged_decode_attention", mutates_args=())
def paged_decode_attention(q: torch.Tensor, kv_pool: torch.Tensor, block_table: torch.Tensor,
                           ctx_len: torch.Tensor, scale: float,
                           pages_per_split: Optional[int] = None,
                           max_pages_in_batch: Optional[int] = None,
                           total_pages: Optional[int] = None) -> torch.Tensor:
    """Split-K decode attention of q [B, Hq, D] over each row's pages; returns out."""
    return paged.paged_decode_attention(q, kv_pool, block_table, ctx_len, scale,
                                        pages_per_split=pages_per_split,
                                        max_pages_in_batch=max_pages_in_batch,
                                        total_pages=total_pages)


@paged_decode_attention.register_fake
def _(q, kv_pool, block_table, ctx_len, scale, pages_per_split=None, max_pages_in_batch=None,
      total_pages=None):
    return torch.empty_like(q)


@torch.library.custom_op(f"{_LIB}::paged_decode_attention_fused", mutates_args=("kv_pool",))
def paged_decode_attention_fused(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                                 slot_mapping: torch.Tensor, kv_pool: torch.Tensor,
                                 block_table: torch.Tensor, ctx_len: torch.Tensor,
                                 scale: float, pages_per_split: Optional[int] = None,
                                 max_pages_in_batch: Optional[int] = None,
                                 total_pages: Optional[int] = None) -> torch.Tensor:
    """The new tokens' KV append and split-K attention in one launch; returns out."""
    return paged.paged_decode_attention_fused(q, k_new, v_new, slot_mapping, kv_pool,
                                              block_table, ctx_len, scale,
                                              pages_per_split=pages_per_split,
                                              max_pages_in_batch=max_pages_in_batch,
                                              total_pages=total_pages)


@paged_decode_attention_fused.register_fake
def _(q, k_new, v_new, slot_mapping, kv_pool, block_table, ctx_len, scale,
      pages_per_split=None, max_pages_in_batch=None, total_pages=None):
    return torch.empty_like(q)


OPERATORS = ("gdn_decode", "gated_delta_token", "gated_delta_chunked", "gated_delta_chunks",
             "kv_append", "paged_decode_attention", "paged_decode_attention_fused")


# ---- group decode: several continuations of shared prompts in one step
@torch.library.custom_op(f"{_LIB}::rotary_append", mutates_args=("kv_pool",))
def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                  kv_pool: torch.Tensor, slot_mapping: torch.Tensor, rotary_dim: int,
                  base: float = 10000.0, sections: Optional[List[int]] = None,
                  interleaved: bool = False, q_weight: Optional[torch.Tensor] = None,
                  k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """Norm and turn q, k by positions [axes, ntok] and append k, v; returns q."""
    plan = _plan(q.shape[-1], rotary_dim, base, tuple(sections) if sections else None,
                 interleaved, q.device)
    return rotary.rotary_append(q, k, v, positions, plan, kv_pool, slot_mapping,
                                q_weight=q_weight, k_weight=k_weight, eps=eps)


@functools.lru_cache(maxsize=32)
def _plan(head_dim, rotary_dim, base, sections, interleaved, device) -> rotary.RotaryPlan:
    """A plan is a function of these values alone: made once for each."""
    return rotary.RotaryPlan(head_dim, rotary_dim, base=base, sections=sections,
                             interleaved=interleaved, device=device)


@rotary_append.register_fake
def _(q, k, v, positions, kv_pool, slot_mapping, rotary_dim, base=10000.0, sections=None,
      interleaved=False, q_weight=None, k_weight=None, eps=1e-6):
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{_LIB}::shared_prefix_attention", mutates_args=())
def shared_prefix_attention(q: torch.Tensor, kv_pool: torch.Tensor, block_table: torch.Tensor,
                            ctx_len: torch.Tensor, scale: float, group_rows: List[int],
                            group_sizes: List[int], prefix_tokens: List[int],
                            max_suffix_pages: Optional[int] = None,
                            total_suffix_pages: Optional[int] = None) -> torch.Tensor:
    """Decode attention of q [B, Hq, D] with shared prefixes read once; returns out. Group i
    is the next group_sizes[i] of group_rows, sharing prefix_tokens[i] tokens (the plan is
    laid out in every call: a program that decodes on keeps a paged.PrefixGroups)."""
    if len(group_sizes) != len(prefix_tokens) or sum(group_sizes) != len(group_rows):
        raise ValueError("shared_prefix_attention: group_rows, group_sizes and prefix_tokens "
                         "do not describe the same groups")
    groups, at = [], 0
    for size, tokens in zip(group_sizes, prefix_tokens):
        groups.append((group_rows[at:at + size], tokens))
        at += size
    plan = paged.PrefixGroups(groups, q.shape[0], q.shape[1], kv_pool.shape[1], q.shape[2],
                              device=q.device)
    return paged.shared_prefix_attention(q, kv_pool, block_table, ctx_len, scale, plan,
                                         max_suffix_pages=max_suffix_pages,
                                         total_suffix_pages=total_suffix_pages)


@shared_prefix_attention.register_fake
def _(q, kv_pool, block_table, ctx_len, scale, group_rows, group_sizes, prefix_tokens,
      max_suffix_pages=None, total_suffix_pages=None):
    return torch.empty_like(q)


@torch.library.custom_op(f"{_LIB}::beam_select", mutates_args=())
def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: int,
                finished: Optional[torch.Tensor] = None, pad_token: int = 0
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The n best continuations of each group's beams: (scores, parents, tokens) [G, n]."""
    best, parents, tokens = beam.beam_select(logits, scores, n, finished=finished,
                                             pad_token=pad_token)
    return best, parents.clone(), tokens.clone()  # an operator's results share no storage


@beam_select.register_fake
def _(logits, scores, n, finished=None, pad_token=0):
    shape = (logits.shape[0], n)
    return (scores.new_empty(shape, dtype=torch.float32),
            scores.new_empty(shape, dtype=torch.int32), scores.new_empty(shape, dtype=torch.int32))


@torch.library.custom_op(f"{_LIB}::reorder_rows", mutates_args=("pools",))
def reorder_rows(pools: List[torch.Tensor], slots: torch.Tensor, parents: torch.Tensor
                 ) -> torch.Tensor:
    """Rows of every pool follow their beams, in place; returns the new slots."""
    return beam.reorder_rows(pools, slots, parents)


@reorder_rows.register_fake
def _(pools, slots, parents):
    return torch.empty_like(slots)


GROUP_OPERATORS = ("rotary_append", "shared_prefix_attention", "beam_select", "reorder_rows")
