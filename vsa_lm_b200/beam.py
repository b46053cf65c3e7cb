"""Beam search over the decode state of a hybrid model: the state of B prompts repeated for B x K beams,
moved between beams after every selection, and the token history read back through the parents.

The reference samples only (vsa_lm/config/bolt3.py:321-333, 459-526) and has no counterpart. The
selection and the moves are kernels (kernels.beam_select, kernels.BeamReorder); the state is
rearranged in place, so steps replayed from CUDA graphs go on pointing at it.
"""
from __future__ import annotations

import torch

from . import kernels as K

_RING = ("ring_kr", "ring_kp", "ring_v", "ring_b")
_SINKS = ("sink_k", "sink_v")


def _layer_tensors(st) -> list[torch.Tensor]:
    """The device tensors a Bolt3LayerState holds now, one row per (sequence, KV head) first."""
    out = [getattr(st, k) for k in _RING]
    if st.sinks_set:
        out += [getattr(st, k) for k in _SINKS]
    if st.has_bank:
        out += [t for t in st.bank.values() if t is not None]
    if st.big_prev is not None:
        out += [t for t in st.big_prev.values() if isinstance(t, torch.Tensor)]
    return out


def _repeat(t: torch.Tensor, dim: int, rows: int, beams: int) -> torch.Tensor:
    """Every group of `rows` entries of dimension `dim` repeated `beams` times."""
    return t.unflatten(dim, (-1, rows)).repeat_interleave(beams, dim=dim).flatten(dim, dim + 1).contiguous()


def expand_beams(model, states, kv_caches, beams: int):
    """(states, kv_caches) of B sequences copied for B x beams: beam j of sequence b is sequence
    b * beams + j of the new state."""
    from .bolt3 import Bolt3LayerState

    out_s, out_c = [], []
    for li, blk in enumerate(model.blocks):
        c = kv_caches[li]
        if not hasattr(blk, "vsa"):
            out_s.append(None)
            out_c.append(c.repeated(beams))
            continue
        new = Bolt3LayerState(blk.vsa, c.B * beams, c.ring_kp.device)
        for k in _RING + _SINKS:
            getattr(new, k).copy_(_repeat(getattr(c, k), 0, c.HKV, beams))
        for k, t in c.bank.items():
            if t is not None:
                new.bank[k].copy_(_repeat(t, 0, c.HKV, beams))
        new.slot_pos, new.cur_slot, new.cur_len = list(c.slot_pos), c.cur_slot, c.cur_len
        new.prev_slot, new.sinks_set, new.n_filled = c.prev_slot, c.sinks_set, c.n_filled
        new.status.word.copy_(c.status.word)      # an error of the kernels that made this state
        if c.big_prev is not None:
            new.big_prev = {k: _repeat(t, 0, c.HKV, beams) if isinstance(t, torch.Tensor) else t
                            for k, t in c.big_prev.items()}
        out_s.append(_repeat(states[li], 0, 1, beams))
        out_c.append(new)
    return out_s, out_c


class BeamStates:
    """The reordering of a decode state of groups x beams sequences whose first `shared` cached tokens are
    the same in all beams of a group. The plan is laid out again when the state holds other tensors than
    before (a cache that grew, a first bank)."""

    def __init__(self, states, kv_caches, groups: int, beams: int, shared: int):
        self.states, self.kv = states, kv_caches
        self.groups, self.beams, self.shared = groups, beams, shared
        self.plan = None

    def _items(self):
        from .bolt3 import Bolt3LayerState

        items = []
        for s, c in zip(self.states, self.kv):
            if isinstance(c, Bolt3LayerState):
                items += [(t, 0, None) for t in _layer_tensors(c)]
                if c.has_bank:
                    items.append((s, 0, None))
            else:
                items += [(t, 1, 3) for t in c.tensors()]
        return items

    def reorder(self, parent: torch.Tensor) -> None:
        """Every beam's state becomes that of its parent (int32 [groups, beams], as beam_select gives it)."""
        items = self._items()
        if self.plan is None or len(items) != len(self.plan.tensors) or any(
                a[0] is not b for a, b in zip(items, self.plan.tensors)):
            self.plan = K.BeamReorder(items, self.groups, self.beams)
        n = max((c.n for c in self.kv if hasattr(c, "tensors")), default=0)
        self.plan(parent, t0=min(self.shared, n), t1=n)


def backtrack(tokens: list, parents: list, pad: int) -> torch.Tensor:
    """The token sequences [groups, beams, steps] of the beams after the last step: step i's token of a beam
    is that of its ancestor, parents[i] leading from the beams after step i to those before."""
    steps = len(tokens)
    groups, beams = tokens[0].shape
    out = torch.full((groups, beams, steps), pad, dtype=torch.long, device=tokens[0].device)
    at = torch.arange(beams, device=out.device).expand(groups, beams)
    for i in range(steps - 1, -1, -1):
        out[:, :, i] = tokens[i].gather(1, at)
        at = parents[i].long().gather(1, at)
    return out


@torch.no_grad()
def beam_search(dec, ids: torch.Tensor, beams: int, max_new_tokens: int, eos_ids=()):
    """The `beams` best continuations of every row of ids [B, T] by the sum of their tokens' log
    probabilities, up to max_new_tokens tokens each or through the first of `eos_ids`. Returns (tokens
    [B, beams, n], scores fp32 [B, beams], lengths [B, beams]), best first; positions past a length hold
    eos_ids[0] (of a set, which has no order, the lowest). A finished beam keeps its score and its place
    among the beams. Stops early once all beams have finished (looked at every 16 tokens)."""
    if beams < 1 or beams > 16 or max_new_tokens < 1:
        raise ValueError(f"{beams} beams and {max_new_tokens} tokens: 1 to 16 beams, at least one token")
    eos = tuple(int(e) for e in (sorted(eos_ids) if isinstance(eos_ids, (set, frozenset)) else eos_ids))
    B, T = ids.shape
    dev = ids.device
    h, states, kv = dec.prefill(ids, max_kv_len=T + max_new_tokens + 64)
    logits = dec.model.lm_head(h[:, -1, :]).repeat_interleave(beams, dim=0)
    states, kv = expand_beams(dec.model, states, kv, beams)
    moves = BeamStates(states, kv, B, beams, shared=T)
    scores = torch.full((B, beams), float("-inf"), device=dev)
    scores[:, 0] = 0.0
    finished = torch.zeros(B, beams, dtype=torch.bool, device=dev) if eos else None
    tokens, parents = [], []
    runner = dec.step_graph(states, kv) if dec.graphs_supported(dev) else None
    for i in range(max_new_tokens):
        scores, parent, token, done = K.beam_select(logits, scores, finished, eos_ids=eos)
        finished = done if eos else None
        tokens.append(token)
        parents.append(parent)
        if i + 1 == max_new_tokens or (eos and i % 16 == 15 and bool(done.all())):
            break
        moves.reorder(parent)
        nxt = token.view(B * beams, 1)
        h = runner.step(nxt, T + i) if runner is not None else dec.step(nxt, T + i, states, kv)[0]
        logits = dec.model.lm_head(h[:, -1, :])
    if runner is not None:
        runner.close()
    dec.check_status(kv)
    out = backtrack(tokens, parents, eos[0] if eos else 0)
    order = torch.argsort(scores, dim=1, descending=True, stable=True)
    out, scores = out.gather(1, order[..., None].expand_as(out)), scores.gather(1, order)
    n = out.shape[2]
    lengths = torch.full((B, beams), n, dtype=torch.long, device=dev)
    if eos:
        hit = torch.isin(out, torch.tensor(eos, device=dev))
        lengths = torch.where(hit.any(-1), hit.int().argmax(-1) + 1, lengths)
        out = torch.where(torch.arange(n, device=dev) < lengths[..., None], out, eos[0])
    return out, scores, lengths
