"""Beam search over the paged cache, on the device from the prompts' last logits to the finished hypotheses.

A batch of R requests with W beams each is a decode step of R * W rows.  One step is a replay of the recorded model step and four
operators: the best continuations of every request (`ops.beam_select`), which of them go on and which are finished
(`ops.beam_keep`), the cache following the beams (`ops.beam_reorder`), and the next step's positions, lengths and new pages
(`ops.step_build`).  None of them waits for the host; it launches step after step and looks now and then whether every request is done.

Where things lie.  The prompt is computed once, by an ordinary request; its full pages are shared by all beams.  Beam 0 goes on in
that request's last page and state slot, the others get a page, a slot and copies of both by the first reordering.  The pages that the beams
will fill are taken from the ledger before the search begins (all or none) and handed out on the device; pages that no
beam refers to any more come back with the rest when the search ends.  A search takes W pages for every page of generated tokens.

The reference decodes greedily or by sampling (crates/engine/workloads/src/sampling.rs); beam search is this engine's own.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Hashable, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..cache.pages import OutOfPages
from ..csrc import ops
from .batch import StepEntry
from .graphs import BUCKETS

LOOK_EVERY = 8             # steps between two looks at whether all requests are done


@dataclass
class BeamHypothesis:
    """`score`: the sum of the tokens' log probabilities / (their number ^ length penalty).  `finish_reason`: "eos" (the last token is a stop
    token) or "length"."""
    tokens: List[int]
    score: float
    finish_reason: str


class BeamSearch:
    def __init__(self, engine, beams: int, max_new_tokens: int, stops: Sequence[int], length_penalty: float = 1.0,
                 early_stopping: bool = False) -> None:
        self.engine = engine
        self.runner = engine.runner
        self.beams, self.last = int(beams), int(max_new_tokens)
        self.penalty, self.early = float(length_penalty), bool(early_stopping)
        self.stops = sorted(set(int(t) for t in stops))
        self.best = self.beams * (1 + len(self.stops))
        graphs = getattr(self.runner, "graphs", None)
        if not 0 < self.beams <= ops.BEAM_MAX:
            raise ValueError(f"up to {ops.BEAM_MAX} beams are served, found {beams}")
        if self.best > ops.BEAM_MAX_BEST:
            raise ValueError(f"{self.beams} beams with {len(self.stops)} stop tokens need {self.best} candidates a step, {ops.BEAM_MAX_BEST} are served")
        if self.last <= 0:
            raise ValueError("max_new_tokens must be positive")
        if not np.isfinite(self.penalty):
            raise ValueError("the length penalty must be a number")
        if not ops.beam_penalty_served(self.penalty, self.last):
            raise ValueError(f"{self.last} tokens to the power of {self.penalty}: up to 2 ^ {ops.BEAM_MAX_POWER:g}, or its inverse, is served")
        if graphs is None or not graphs.whole or self.runner.spec.token_extras:
            raise ValueError("beam search needs a model whose whole step is recorded as one graph and that takes no inputs per token beside ids "
                             "and positions")

    # ------------------------------------------------------------------ sizing
    def _blocks(self, group, tokens: int) -> int:
        return -(-(tokens // group.need.stride) // group.page_size)

    def _own_blocks(self, group, prompt: int, total: int) -> int:
        """Blocks from the prompt's last, partly filled one on (or the first behind it), that every beam has for itself."""
        return self._blocks(group, total) - prompt // group.need.stride // group.page_size

    def _beam_tokens(self, prompt: int, total: int) -> int:
        """Tokens that a beam's ledger entry is made for so that every group gets the pages it will need."""
        return max([0] + [self._own_blocks(g, prompt, total) * g.page_size * g.need.stride for g in self.runner.cache.groups])

    def _pages(self, prompt: int) -> Dict[int, int]:
        """Pages of a request in every group, at most: the prompt and its first beam, and the other beams."""
        total = prompt + self.last - 1
        extra = self._beam_tokens(prompt, total)
        return {g.index: self._blocks(g, total) + (self.beams - 1) * self._blocks(g, extra) for g in self.runner.cache.groups}

    def batch_of(self, prompts: Sequence[Sequence[int]]) -> int:
        """How many of the next prompts run together: as slots, rows of a step and free pages allow."""
        cache = self.runner.cache
        most = min(cache.slots.num_free, BUCKETS[-1]) // self.beams
        if most < 1:
            raise OutOfPages(f"{self.beams} beams need as many state slots, {cache.slots.num_free} are free")
        free, n = cache.free_pages(), 0
        for p in prompts[:most]:
            need = self._pages(len(p))
            if any(need[g] > free[g] for g in free):
                break
            free = {g: free[g] - need[g] for g in free}
            n += 1
        if n == 0:
            raise OutOfPages(f"a search with {self.beams} beams from {len(prompts[0])} tokens over {self.last} needs pages {self._pages(len(prompts[0]))}, "
                             f"free {cache.free_pages()}")
        return n

    # ------------------------------------------------------------------ the search
    def run(self, prompts: Sequence[Sequence[int]]) -> List[List[BeamHypothesis]]:
        """Hypotheses of every prompt, best first."""
        found: List[List[BeamHypothesis]] = []
        while len(found) < len(prompts):
            rest = prompts[len(found):]
            found += self._run_batch(rest[:self.batch_of(rest)])
        return found

    def _run_batch(self, prompts: Sequence[Sequence[int]]) -> List[List[BeamHypothesis]]:
        cache = self.runner.cache
        R, W = len(prompts), self.beams
        # (names that no request of a caller has)
        ids: List[Hashable] = [(self, r, w) for r in range(R) for w in range(W)]
        try:
            first = self._prefill(prompts, ids)
            slots = []
            for r, p in enumerate(prompts):
                total = len(p) + self.last - 1
                cache.ensure(ids[r * W], total)
                slots.append(cache.slot_of(ids[r * W]))
                for w in range(1, W):
                    slots.append(cache.begin(ids[r * W + w]))
                    cache.ensure(ids[r * W + w], self._beam_tokens(len(p), total))
            return self._decode(prompts, ids, slots, first)
        finally:
            for i in ids:
                if cache.has(i):
                    cache.release(i)

    def _prefill(self, prompts, ids) -> torch.Tensor:
        """Every prompt through the model in portions; its last logits [R, vocab]."""
        W, config = self.beams, self.engine.scheduler.config
        out = torch.empty((len(prompts), self.runner.spec.vocab_size), dtype=torch.float32, device=self.runner.device)
        at = [0] * len(prompts)
        while any(a < len(p) for a, p in zip(at, prompts)):
            budget, entries, ends = config.max_num_batched_tokens, [], []
            for r, p in enumerate(prompts):
                n = min(len(p) - at[r], config.prefill_chunk_tokens, budget)
                if n <= 0 or len(entries) >= config.max_num_seqs:
                    continue
                whole = at[r] + n == len(p)
                entries.append(StepEntry(ids[r * W], p[at[r]:at[r] + n], [n - 1] if whole else []))
                if whole:
                    ends.append(r)
                at[r] += n
                budget -= n
            logits = self.runner.step(entries)
            if ends:
                out[torch.tensor(ends, device=out.device)] = logits[:len(ends)]
        return out

    def _layout(self, prompts, ids, slots, ctx) -> Tuple[List[ops.StepPages], torch.Tensor]:
        """Fill the step's arrays for rows whose prompts are cached; the groups' pages that are still to be handed out."""
        cache, device = self.runner.cache, self.runner.device
        R, W = len(prompts), self.beams
        n, bucket = R * W, ctx.n_seqs
        for t, head, rest in ((ctx.positions, [len(p) - 1 for p in prompts for _ in range(W)], 0), (ctx.kv_len, [len(p) for p in prompts for _ in range(W)], 0),
                              (ctx.slots, slots, -1)):
            t.copy_(torch.tensor(list(head) + [rest] * (bucket - n), dtype=torch.int32))
        ctx.tokens.zero_()
        ctx.seq_of_token.copy_(torch.arange(bucket, dtype=torch.int32))
        ctx.cu_q.copy_(torch.arange(bucket + 1, dtype=torch.int32))
        ctx.logit_rows.copy_(torch.arange(bucket, dtype=torch.int32))
        pages = []
        for g in cache.groups:
            rows, free = np.full((bucket, ctx.block_tables[g.index].shape[1]), -1, dtype=np.int32), []
            for r, p in enumerate(prompts):
                have = len(p) // g.need.stride
                full, part = have // g.page_size, have % g.page_size != 0
                shared = cache.block_table(g.index, ids[r * W])
                for w in range(W):
                    own = shared[full:] if w == 0 else cache.block_table(g.index, ids[r * W + w])[:self._own_blocks(g, len(p), len(p) + self.last - 1)]
                    rows[r * W + w, :full] = shared[:full]
                    if part:
                        rows[r * W + w, full] = own[0]
                    free += own[1 if part else 0:]
            ctx.block_tables[g.index].copy_(torch.from_numpy(rows))
            pages.append(ops.StepPages(ctx.block_tables[g.index][:n], torch.tensor(free, dtype=torch.int32).to(device),
                                       torch.zeros(1, dtype=torch.int32, device=device), g.page_size, g.need.stride))
        return pages, torch.ones(n, dtype=torch.int32, device=device)

    def _decode(self, prompts, ids, slots, first: torch.Tensor) -> List[List[BeamHypothesis]]:
        r_, cache, device = self.runner, self.runner.cache, self.runner.device
        R, W, k = len(prompts), self.beams, self.best
        n = R * W
        longest = max(len(p) for p in prompts) + self.last - 1
        key, rec, ctx, ints = r_.graphs.beam_step(n, W, longest)
        pages, ones = self._layout(prompts, ids, slots, ctx)
        state = cache.beam_state()
        track = ops.BeamTrack.make(R, W, self.last, device)
        track.tokens = ctx.tokens[:n].view(R, W)              # the tokens that go on are the next step's
        cand = [torch.empty((R, k), dtype=t, device=device) for t in (torch.int32, torch.int32, torch.float32)]
        bad, any_bad, alive = (torch.zeros(n, dtype=torch.int32, device=device) for _ in range(3))
        refused = torch.zeros(1, dtype=torch.int32, device=device)
        stops = torch.tensor(self.stops, dtype=torch.int32, device=device) if self.stops else None
        seen, looked = torch.zeros(R, dtype=torch.int32).pin_memory(), None
        lens, positions, tables = ctx.kv_len[:n], ctx.positions[:n], [p.table for p in pages]
        ops.scope("beam search")
        # the prompts' logits: one row a request, before there are beams
        ops.beam_select(first, torch.zeros((R, 1), device=device), *cand, any_bad[:R])
        for step in range(self.last):
            if step:
                rec = r_.graphs.run_beams(key, rec, ctx, ints)
                r_.steps_run += 1
                r_.tokens_run += n
                ops.scope("beam search")
                ops.beam_select(rec.logits[:n], track.scores, *cand, bad)
                # (a beam that has no tokens keeps its row, whose pages hold anything)
                torch.gt(track.scores.view(-1), float("-inf"), out=alive)
                any_bad.addcmul_(bad, alive)
            ops.beam_keep(*cand, stops, track, step, self.last, self.penalty, self.early)
            if step + 1 == self.last:
                break
            if looked is not None and looked.query():
                if bool((seen != 0).all()):
                    break
                looked = None
            if looked is None and step % LOOK_EVERY == 0:
                seen.copy_(track.done, non_blocking=True)
                looked = torch.cuda.Event()
                looked.record(torch.cuda.current_stream(device))
            ops.beam_reorder(state, track.parents, lens, tables, ctx.slots[:n])
            ops.step_build(ones, lens, lens, positions, ctx.seq_of_token[:n], ctx.cu_q[:n + 1], pages, refused)
        ops.scope("other")
        if int(any_bad.max()) != 0:
            raise ValueError("invalid logits (a NaN or an infinity) in a beam search")
        if int(refused) != 0:
            raise RuntimeError(f"a step of a beam search was refused ({int(refused)})")
        ops.check_device_errors()
        return self._walk_back(track, R)

    def _walk_back(self, track, R: int) -> List[List[BeamHypothesis]]:
        counts, scores = track.done_count.tolist(), track.done_scores.tolist()
        steps, parents, tokens = track.done_steps.tolist(), track.done_parents.tolist(), track.done_tokens.tolist()
        past_parents, past_tokens = track.past_parents.cpu().numpy(), track.past_tokens.cpu().numpy()
        out = []
        for r in range(R):
            hyps = []
            for i in range(counts[r]):
                step, beam, toks = steps[r][i], parents[r][i], [tokens[r][i]]
                for s in range(step - 1, -1, -1):
                    toks.append(int(past_tokens[s, r, beam]))
                    beam = int(past_parents[s, r, beam])
                toks.reverse()
                hyps.append(BeamHypothesis(toks, scores[r][i], "eos" if toks[-1] in self.stops else "length"))
            out.append(hyps)
        return out
