"""Beam search over the paged engine: several continuations of one prompt decoded together.

One step of a prompt's beams is what this module's operators are for: q/k norm, rotary
positions and the KV append in one launch (rotary), attention that reads the prompt's
shared pages once for all beams (paged.shared_prefix_attention), the choice of the next
beams from their logits (beam.beam_select), and the move of GDN state, conv taps and
pages to the beams that go on (HybridCacheEngine.reorder). The GDN layers run as in
resident.PagedResident; the projections are resident.ToyHybridModel's.

The reference samples each request by itself (studio_compute/inference.py:176-218) and
has no beams; its per-layer decode order is mlx_decode.py:18-106.
"""

from __future__ import annotations

from dataclasses import dataclass, field

import torch

from . import beam, gdn_layer, paged, rotary
from .engine import HybridCacheEngine


@dataclass
class Beam:
    tokens: list = field(default_factory=list)   # generated, without padding
    score: float = 0.0                           # summed log-probability
    finished: bool = False


class BeamSearch:
    """Beams over one prompt on a HybridCacheEngine (with tap rings) and a model."""

    def __init__(self, cache: HybridCacheEngine, model, plan: rotary.RotaryPlan, *,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                 stop_token: int | None = None):
        if cache.taps is None:
            raise ValueError("BeamSearch runs GDN layers from projections: gdn_taps=True")
        self.cache, self.model, self.plan = cache, model, plan
        self.q_weight, self.k_weight, self.stop = q_weight, k_weight, stop_token
        c = cache.cfg
        self._glue_ws = gdn_layer.SplitWorkspace(c.max_seqs, model.layers[c.gdn_layers[0]].glue,
                                                 cache.device)
        self.slots: list = []
        self.beams: list = []

    # ---------------------------------------------------------------- prompt
    def start(self, prompt: list, beams: int) -> None:
        """Prefill the prompt once and open `beams` sequences over its cache."""
        if not prompt or not 1 <= beams <= beam.MAX_BEAMS:
            raise ValueError(f"start: a prompt and 1 to {beam.MAX_BEAMS} beams")
        if self.slots:
            raise ValueError("start: close() the open beams first")
        eng = self.cache
        # The prompt's pages, and its partial last page for a snapshot and each fork.
        forks = beams if beams > 1 and len(prompt) % eng.cfg.page_size else 0
        pages = eng.blocks.pages_for(len(prompt)) + forks
        if eng.blocks.free_slots < beams or eng.blocks.free_pages < pages:
            raise MemoryError(f"{beams} slots and {pages} pages needed, "
                              f"{eng.blocks.free_slots} and {eng.blocks.free_pages} free")
        if beams > 1 and not eng.free_snapshot_rows:
            raise MemoryError("a snapshot row is needed to fork the beams, none is free")
        self.slots = [eng.admit("beam", len(prompt))]
        try:
            self._logits = self._prefill(self.slots[0], prompt)
            if beams > 1:
                snap = eng.snapshot(self.slots[0])
                try:
                    for _ in range(beams - 1):
                        self.slots.append(eng.fork(snap, owner="beam"))
                finally:
                    eng.drop_snapshot(snap)
            self.beams = [Beam() for _ in range(beams)]
            # Until the beams differ only the first one counts.
            self._scores = torch.full((1, beams), -float("inf"), device=eng.device)
            self._scores[0, 0] = 0.0
            self._logits = self._logits.expand(beams, -1)
            self._choose()
        except BaseException:
            self.close()
            raise

    def _prefill(self, slot: int, ids: list) -> torch.Tensor:
        eng, model, c, dev = self.cache, self.model, self.cache.cfg, self.cache.device
        n = len(ids)
        span = torch.tensor([0, n], dtype=torch.int32, device=dev)
        slot_t = torch.tensor([slot], dtype=torch.int32, device=dev)
        zero = torch.zeros(1, dtype=torch.int32, device=dev)
        slots = torch.from_numpy(eng.blocks.prompt_slots(slot, 0, n)).to(dev)
        pos = torch.arange(n, dtype=torch.int32, device=dev).expand(self.plan.axes, n)
        h = model.hidden(ids)
        for layer in range(c.layers):
            if c.is_attention(layer):
                q, k, v = model.attention_inputs(layer, h)
                pool = eng.kv[eng.attn_index[layer]]
                q = rotary.rotary_append(q, k, v, pos, self.plan, pool, slots,
                                         q_weight=self.q_weight, k_weight=self.k_weight)
                kk, vv = paged.kv_gather(pool, slots)
                group = c.q_heads // c.kv_heads
                kk, vv = (t.float().repeat_interleave(group, 1).transpose(0, 1) for t in (kk, vv))
                o = torch.nn.functional.scaled_dot_product_attention(
                    q.float().transpose(0, 1), kk, vv, is_causal=True, scale=eng.scale)
                h = model.residual(layer, h, o.transpose(0, 1).to(torch.bfloat16))
            else:
                qkv, z, a, b = model.gdn_inputs(layer, h)
                i = eng.gdn_index[layer]
                h = model.residual(layer, h, gdn_layer.gdn_prefill(
                    qkv, z, a, b, model.layers[layer].glue, eng.taps[i], eng.state[i], span,
                    slot_t, zero))
        return model.logits(h[-1:])

    # ---------------------------------------------------------------- steps
    def step(self) -> bool:
        """One token for every beam, then the best beams go on; False when all are done.

        Raises OutOfPages, with nothing changed, where the pool cannot hold the token: the
        step may be taken again when there is room.
        """
        if all(b.finished for b in self.beams):
            return False
        eng, model, c = self.cache, self.model, self.cache.cfg
        eng.begin_step(self.slots)
        n = eng.rows
        rows = torch.tensor(self.slots, dtype=torch.long, device=eng.device)

        def spread(t):
            full = torch.zeros((n,) + t.shape[1:], dtype=t.dtype, device=t.device)
            full[rows] = t
            return full

        h = model.hidden([b.tokens[-1] for b in self.beams])
        for layer in range(c.layers):
            if c.is_attention(layer):
                q, k, v = (spread(t) for t in model.attention_inputs(layer, h))
                q = eng.append_rotary(layer, q, k, v, self.plan, q_weight=self.q_weight,
                                      k_weight=self.k_weight)
                out = torch.empty_like(q)
                eng.group_attention_layer(layer, q, out)
            else:
                qkv, z, a, b = (spread(t) for t in model.gdn_inputs(layer, h))
                out = torch.empty((n, c.gdn_value_heads * 128), dtype=torch.bfloat16,
                                  device=eng.device)
                i = eng.gdn_index[layer]
                gdn_layer.gdn_decode_split(qkv, z, a, b, model.layers[layer].glue, eng.taps[i],
                                           eng.position[:n], eng.state[i], eng.state_slot[:n],
                                           out=out, workspace=self._glue_ws)
            h = model.residual(layer, h, out[rows])
        self._logits = model.logits(h)
        self._choose()
        return not all(b.finished for b in self.beams)

    def _choose(self) -> None:
        """The best continuations of the beams become the beams."""
        count = len(self.beams)
        done = torch.tensor([[b.finished for b in self.beams]], device=self.cache.device)
        pad = 0 if self.stop is None else self.stop
        best, parents, tokens = beam.beam_select(self._logits[None].contiguous(), self._scores,
                                                 count, finished=done, pad_token=pad)
        parents, tokens = parents[0].tolist(), tokens[0].tolist()
        scores = best[0].tolist()
        chosen = []
        for p, t, s in zip(parents, tokens, scores):
            old = self.beams[p]
            chosen.append(Beam(old.tokens if old.finished else old.tokens + [t], s,
                               old.finished or t == self.stop))
        self.slots = self.cache.reorder(self.slots, parents, reuse_pages=True)
        self.beams, self._scores = chosen, best

    def search(self, prompt: list, beams: int, max_tokens: int) -> list:
        """The best continuations of the prompt, up to max_tokens long, best first."""
        if max_tokens < 1:
            raise ValueError(f"search: max_tokens={max_tokens}, the prompt gives one at least")
        self.start(prompt, beams)
        while len(max(self.beams, key=lambda b: len(b.tokens)).tokens) < max_tokens and self.step():
            pass
        return list(self.beams)

    def close(self) -> None:
        """Release the beams' slots and pages."""
        for slot in self.slots:
            self.cache.release(slot)
        self.slots, self.beams = [], []
