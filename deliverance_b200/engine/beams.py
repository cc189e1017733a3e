"""Beam search on the engine's model and paged cache.

Every prompt keeps ``num_beams`` hypotheses, one row of the decode batch each. A step feeds every beam's newest token, scores all continuations
(``ops.beam.beam_select``: ``2 * num_beams`` candidates, so that ended hypotheses leave enough others), and lets the best that have not ended live on. A beam
shares its parent's full pages by reference; the page that is still being filled is its own, and its rows, like recurrent states, are taken over from the parent in
place (``ops.beam.beam_reorder``). Hypotheses end with an end token, which counts as one of their tokens, or at the length limit, and rank by ``log-probability / tokens **
length_penalty``. A prompt is done when ``num_beams`` of them have ended and the best beam alive, at its present length, ranks behind the last of those.
"""
from __future__ import annotations

import time
from dataclasses import dataclass, field

import torch

from .. import ops
from ..models.batch import make_batch
from ..ops.beam import MAX_CANDIDATES, beam_reorder, beam_select
from ..params import FinishReason, GeneratorParameters, Response

_NONE = float("-inf")


@dataclass
class _Beam:
    pages: list
    slot: int  # recurrent state, -1: none
    tokens: list = field(default_factory=list)
    score: float = _NONE  # sum of log-probabilities; -inf: not in use


@dataclass
class _Search:
    request: object
    beams: list
    steps: int  # most tokens of a hypothesis
    ended: list = field(default_factory=list)  # (rank value, tokens, reason), best first
    done: bool = False


class BeamSearch:
    def __init__(self, engine, params: GeneratorParameters):
        params.validate()
        self.e, self.params, self.W = engine, params, params.num_beams
        if self.W > engine.config.max_seqs:
            raise ValueError(f"{self.W} beams do not fit max_seqs={engine.config.max_seqs}")

    # ------------------------------------------------------------------------------------------------ memory
    def _limits(self, prompt: list) -> tuple:
        """(most new tokens, pages that prompt and beams may come to need)."""
        e, p = self.e, self.params
        ctx = e.cfg.max_position_embeddings
        steps = min(p.ntokens or ctx, ctx) - len(prompt)
        if p.max_tokens is not None:
            steps = min(steps, p.max_tokens)
        ps = e.page_size
        shared = len(prompt) // ps
        return steps, shared + self.W * ((len(prompt) + max(steps, 0) + ps - 1) // ps - shared)

    def run(self, prompts: list) -> list:
        e = self.e
        if not (e.waiting or e.running):
            e._drain()  # the step that was launched ahead of a request's last token
        if e.has_work():
            raise RuntimeError("beam search and scheduled requests do not share an engine at the same time")
        most = max(1, e.config.max_seqs // self.W)
        if e.hybrid:
            most = max(1, len(e.kv.free_slots) // self.W)
            if len(e.kv.free_slots) < self.W:
                raise MemoryError(f"{self.W} beams need as many recurrent-state slots")
        for prompt in prompts:  # (all of them before the first search: an error in the last one costs no answers)
            e._limit_of(prompt, self.params)
            need = self._limits(prompt)[1]
            if not e.kv.can_allocate(need):
                raise MemoryError(f"{self.W} beams of this prompt may need {need} pages, which the KV cache does not have")
        out, group, pages = [], [], 0
        for prompt in prompts:
            steps, need = self._limits(prompt)
            if group and (len(group) >= most or not e.kv.can_allocate(pages + need)):
                out += self._search(group)
                group, pages = [], 0
            group.append((prompt, steps))
            pages += need
        if group:
            out += self._search(group)
        if e.device.type == "cuda":
            ops.check_status(e.device.index)
        for i, hypotheses in enumerate(out):
            if not hypotheses:
                raise RuntimeError(f"beam search found no continuation of prompt {i} that has a finite log-probability: the model's logits are NaN or infinite")
        return out

    def _search(self, group: list) -> list:
        e = self.e
        searches: list[_Search] = []
        try:
            first: dict = {}
            for prompt, steps in group:
                r = e._new_request(prompt, self.params)
                if not e._admit(r):
                    raise MemoryError("a prompt cannot be admitted: KV cache too small")
                searches.append(_Search(r, [_Beam(r.pages, r.state_slot)], steps))
            while len(first) < len(searches):
                todo = [s.request for s in searches if s.request.computed < len(s.request.fill)]
                if e._prefill_step(todo, lambda reqs, logits: [first.update({r.rid: logits[i : i + 1]}) for i, r in enumerate(reqs)] and []) is None:
                    raise MemoryError("the KV cache is too small for the prompts")
            self._fork(searches, torch.cat([first[s.request.rid] for s in searches]))
            while True:
                alive = [s for s in searches if not s.done]
                if not alive:
                    break
                self._step(alive)
            return [self._responses(s) for s in searches]
        finally:
            for s in searches:
                self._drop(s)

    def _drop(self, s: _Search) -> None:
        e, r = self.e, s.request
        for b in s.beams[1:]:  # (the first one's pages and state are the request's)
            e.kv.release_pages(b.pages)
            if b.slot >= 0:
                e.kv.free_state_slot(b.slot)
        s.beams = []
        if r in e.running:
            e.running.remove(r)
        if r in e.waiting:  # (preempted by another prompt of the group: it holds nothing)
            e.waiting.remove(r)
        e._release(r)

    # ------------------------------------------------------------------------------------------------ steps
    def _candidates(self, logits: torch.Tensor, scores: list) -> list:
        """Per search ``[(value, beam, token)]``, best first."""
        e = self.e
        logits = e._full(logits)
        k = min(2 * self.W, MAX_CANDIDATES, len(scores[0]) * logits.shape[1])
        got = beam_select(logits, torch.tensor(scores, dtype=torch.float32).to(logits.device), k, None, e.cfg.final_softcap, e._inv_logit_scale())
        values, parents, tokens = (t.tolist() for t in got)
        return [[c for c in zip(v, p, t) if c[2] >= 0] for v, p, t in zip(values, parents, tokens)]

    def _choose(self, s: _Search, candidates: list) -> list:
        """Ended hypotheses join ``s.ended``; returns the beams that live on, ``(value, parent, token)``, ``num_beams`` at most."""
        e, W, lp = self.e, self.W, self.params.length_penalty
        n = len(s.beams[0].tokens) + 1
        last = n >= s.steps
        chosen = []
        for rank, (value, parent, token) in enumerate(candidates):
            ends = token in e.eos_ids
            if ends or last:
                if rank < W:  # (a worse candidate ends only where it would have lived on)
                    s.ended.append((value / n**lp, s.beams[parent].tokens + [token], FinishReason.STOP_TOKEN if ends else FinishReason.MAX_TOKENS))
            elif len(chosen) < W:
                chosen.append((value, parent, token))
        s.ended.sort(key=lambda h: -h[0])
        del s.ended[W:]
        s.done = last or not chosen or (len(s.ended) >= W and max(v for v, _, _ in chosen) / n**lp <= s.ended[-1][0])
        return chosen

    def _fork(self, searches: list, logits: torch.Tensor) -> None:
        """From the prompts' logits to ``num_beams`` beams each, all of them children of the prompt."""
        e = self.e
        for s, cand in zip(searches, self._candidates(logits, [[0.0]] * len(searches))):
            r = s.request
            r.t_first = time.perf_counter()
            chosen = self._choose(s, cand)
            if s.done:
                continue
            full = len(r.fill) // e.page_size
            for _ in range(self.W - 1):
                slot = e.kv.alloc_state_slot() if e.hybrid else -1
                b = _Beam([], slot)
                s.beams.append(b)
                for p in s.beams[0].pages[:full]:
                    e.kv.allocator.retain(p)
                    b.pages.append(p)
                e.kv.ensure_pages(b.pages, len(r.fill))
            self._continue(s, chosen)
        alive = [s for s in searches if not s.done]
        if alive:
            self._move(alive, [[0] * self.W for _ in alive])

    def _continue(self, s: _Search, chosen: list) -> list:
        """Tokens and scores of the beams that live on; returns every beam's parent. Beams without a continuation go out of use."""
        old = [b.tokens for b in s.beams]
        parents = []
        for j, b in enumerate(s.beams):
            value, parent, token = chosen[j] if j < len(chosen) else (_NONE, j, 0)
            b.tokens, b.score = (old[parent] if len(old) > parent else []) + [token], value
            parents.append(parent)
        return parents

    def _move(self, searches: list, parents: list) -> None:
        """What the beams' rows and states hold follows their parents (full pages have done so already)."""
        e = self.e
        dev, ps = e.device, e.page_size
        par = torch.tensor(parents, dtype=torch.int64).to(dev)
        if e.hybrid:
            slots = torch.tensor([[b.slot for b in s.beams] for s in searches], dtype=torch.int64).to(dev)
            beam_reorder(par, states=[t for layers in e.kv.state.values() for t in layers.values()], slots=slots)
        part = [i for i, s in enumerate(searches) if self._cached(s) % ps]
        if part:
            pages = torch.tensor([[b.pages[self._cached(searches[i]) // ps] for b in searches[i].beams] for i in part], dtype=torch.int64).to(dev)
            rows = torch.tensor([self._cached(searches[i]) % ps for i in part], dtype=torch.int32).to(dev)
            caches = [t for t in e.kv.k + e.kv.v if t is not None]
            beam_reorder(par if len(part) == len(searches) else par[torch.tensor(part, device=dev)], caches=caches, pages=pages, rows=rows)

    @staticmethod
    def _cached(s: _Search) -> int:
        """Rows in the cache: all tokens but the newest, which the next step feeds."""
        return len(s.request.fill) + len(s.beams[0].tokens) - 1

    def _step(self, searches: list) -> None:
        e = self.e
        seqs = []
        for s in searches:
            at = self._cached(s)
            for b in s.beams:
                e.kv.ensure_pages(b.pages, at + 1)
                seqs.append({"tokens": [b.tokens[-1]], "start": at, "pages": b.pages, "state_slot": max(b.slot, 0)})
                if e.needs_prev:
                    seqs[-1]["prev"] = b.tokens[-2] if len(b.tokens) > 1 else s.request.fill[-1]
        e.metrics["decode_steps"] += 1
        e.metrics["decode_tokens"] += len(seqs)
        if e.use_graphs and len(seqs) <= 256:
            logits = e._graph_decode(seqs)[: len(seqs)]
        else:
            batch = make_batch(seqs, e.page_size, e.device)
            batch.decode_splits = e._splits(len(seqs))
            logits = e.model.forward(batch, e.kv)
        moved, parents = [], []
        for s, cand in zip(searches, self._candidates(logits, [[b.score for b in s.beams] for s in searches])):
            chosen = self._choose(s, cand)
            if s.done:
                continue
            full = (self._cached(s) + 1) // e.page_size  # pages that this step's row has filled belong to whoever needs them
            par = self._continue(s, chosen)
            lists = [s.beams[p].pages[:full] for p in par]
            for pages in lists:
                for p in pages:
                    e.kv.allocator.retain(p)
            for b, pages in zip(s.beams, lists):
                for p in b.pages[:full]:
                    e.kv.allocator.release(p)
                b.pages[:full] = pages
            moved.append(s)
            parents.append(par)
        if moved:
            self._move(moved, parents)

    # ------------------------------------------------------------------------------------------------ results
    def _responses(self, s: _Search) -> list:
        r = s.request
        out = []
        for value, tokens, reason in s.ended:
            resp = Response()
            resp.token_ids, resp.score, resp.finish_reason = list(tokens), value, reason
            resp.prompt_tokens, resp.generated_tokens = len(r.prompt), len(tokens)
            resp.prefix_hit_tokens = r.prefix_hit
            resp.ttft_ms = (r.t_first - r.t_submit) * 1e3
            resp.total_ms = (time.perf_counter() - r.t_submit) * 1e3
            resp.avg_ms_per_token = resp.total_ms / max(1, len(tokens))
            out.append(resp)
        return out
