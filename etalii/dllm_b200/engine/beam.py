"""Beam search: the prompts enter the cache in one step, then every step runs all beams of all sequences, chooses the next ones
on the device (`ops.beam_select`), and moves what each beam takes over (`ops.beam_reorder`), captured as one CUDA graph. The host
reads the histories every few steps.

Beams share the pages of their prompt; from the page that holds the prompt's end on, each has pages of its own for all it may
still write. Which page of which beam an older position lies in is the page tables' affair, on the device
(csrc/beam_reorder.cu)."""
from __future__ import annotations

import hashlib
import math
from dataclasses import dataclass
from typing import Sequence

import numpy as np
import torch

from ..kernels import ops
from ..sampling.beams import BeamOptions, BeamState
from ..sampling.options import SamplingOptions
from .decode import DecodeGraph
from .generate import ContextLengthError


@dataclass(frozen=True)
class BeamResult:
    tokens: tuple[int, ...]
    score: float
    """Sum of the tokens' log probabilities (and the stop token's), over their count ** length_penalty."""
    prompt_tokens: int
    finish_reason: str
    """"stop" (the text ended with a stop token) or "length" (max_new_tokens or the context window)."""

    @property
    def fingerprint(self) -> str:
        """SHA-256 of the ids as little-endian int32, as `GenerationResult.fingerprint`."""
        return hashlib.sha256(np.asarray(self.tokens, dtype="<i4").tobytes()).hexdigest()


class SharedRows:
    """For the attention parts of a step whose tokens share pages (`ops.attention_shared`): each token's slot, the groups'
    first tokens, the pages that a group's table rows have in common, the most tokens of a group."""

    __slots__ = ("slots", "groups", "shared", "max_rows")

    def __init__(self, slots, groups, shared, max_rows: int) -> None:
        self.slots, self.groups, self.shared, self.max_rows = slots, groups, shared, int(max_rows)


def beam_pages(length: int, new_tokens: int, beams: int, page_size: int) -> int:
    """Pages that a search holds: the prompt's full pages once, and for each beam its own from there to the end."""
    full = length // page_size
    return full + beams * (-(-(length + new_tokens) // page_size) - full)


def plan_beam_batches(lengths: Sequence[int], limits: Sequence[int], beams: int, page_size: int, total_pages: int,
                      total_slots: int, max_batch: int | None = None) -> list[list[int]]:
    """Splits requests, in order, into batches that fit the cache; raises if one alone does not fit."""
    batches: list[list[int]] = []
    current: list[int] = []
    pages = 0
    most = total_slots // beams
    if most < 1:
        raise ContextLengthError(f"{beams} beams need as many cache slots; there are {total_slots}")
    limit = min(most, max_batch) if max_batch else most
    for index, (length, new) in enumerate(zip(lengths, limits)):
        need = beam_pages(length, new, beams, page_size)
        if need > total_pages:
            raise ContextLengthError(f"request {index} needs {need * page_size} cached tokens with {beams} beams; the cache "
                                     f"holds {total_pages * page_size}")
        if current and (pages + need > total_pages or len(current) >= limit):
            batches.append(current)
            current, pages = [], 0
        current.append(index)
        pages += need
    if current:
        batches.append(current)
    return batches


class BeamRun:
    """One sequence's search as the host sees it: the tokens and parents of every step, [step][beam]."""

    def __init__(self, prompt_tokens: int, limit: int) -> None:
        self.prompt_tokens, self.limit = prompt_tokens, limit
        self.tokens: list[Sequence[int]] = []
        self.parents: list[Sequence[int]] = []

    @property
    def produced(self) -> int:
        return len(self.tokens)

    def text(self, count: int, beam: int) -> tuple[int, ...]:
        """The first `count` tokens of the text that is in place `beam` after `count` steps."""
        out = []
        for step in range(count - 1, -1, -1):
            out.append(int(self.tokens[step][beam]))
            beam = int(self.parents[step][beam])
        return tuple(reversed(out))

    def results(self, options: BeamOptions, scores, finished, finished_at, done: bool) -> list[BeamResult]:
        """The best texts, best first: those that have ended and, unless the search is over, those still running."""
        out = [BeamResult(self.text(int(at[0]), int(at[1])), float(score), self.prompt_tokens, "stop")
               for score, at in zip(finished, finished_at) if score > -math.inf]
        if not done:
            divisor = max(1, self.produced) ** options.length_penalty
            out += [BeamResult(self.text(self.produced, beam), float(score) / divisor, self.prompt_tokens, "length")
                    for beam, score in enumerate(scores) if score > -math.inf]
        out.sort(key=lambda result: -result.score)  # (stable: ended texts first among equals)
        return out[:options.beams]


class BeamGraph(DecodeGraph):
    """A beam search's step for `sequences` x options.beams beams: forward, choice, move, advance."""

    def __init__(self, engine, sequences: int, options: BeamOptions, use_graph: bool = True, max_context: int | None = None,
                 min_tokens: int = 0, stops: tuple = ()) -> None:
        super().__init__(engine, sequences * options.beams, SamplingOptions(), use_graph=use_graph, max_context=max_context)
        device = engine.rt.device
        self.n, self.beams, self.search = sequences, options.beams, options
        self.search_min_tokens = int(min_tokens)
        self.stops = torch.tensor(sorted(stops), dtype=torch.int32, device=device) if stops else None
        self.state = BeamState(sequences, options.beams, device)
        self.parents = torch.zeros((sequences, options.beams), dtype=torch.int32, device=device)
        self.parent_history = torch.zeros((self.CAPACITY, sequences, options.beams), dtype=torch.int32, device=device)
        self.tickets = torch.zeros(sequences, dtype=torch.int32, device=device)
        cuts = torch.arange(0, (sequences + 1) * options.beams, options.beams, dtype=torch.int32, device=device)
        self.shared = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.batch.shared = SharedRows(self.batch.slots, cuts, self.shared, options.beams)
        self.rows = engine.cache.beam_rows()

    def _body(self) -> None:
        engine, batch = self.engine, self.batch
        logits = self.logits = engine.model.forward(batch)
        choose(engine, self.parents, self.chosen, self.state, logits, self.produced, self.tickets, self.search, self.stops,
               self.search_min_tokens, steps=self.counter, history=self.parent_history)
        ops.beam_reorder(self.rows, batch.slots, self.parents, batch.start, ahead=1)
        ops.decode_advance(batch.tokens, batch.tok_pos, batch.start, self.chosen, self.history, self.counter, self.b)

    def load_search(self, slots, tokens, starts, produced: int, shared: Sequence[int]) -> None:
        self.load(slots, tokens, starts, produced)
        self.shared.copy_(torch.tensor(list(shared), dtype=torch.int32))

    def histories(self, steps: int) -> tuple[np.ndarray, np.ndarray]:
        """(tokens, parents) of the last `steps` steps since the load, [step, sequence, beam]. (Waits for them.)"""
        tokens = self.history[: steps * self.b].view(steps, self.n, self.beams).cpu().numpy()
        return tokens, self.parent_history[:steps].cpu().numpy()


def choose(engine, parents, tokens, state: BeamState, logits, produced, tickets, options: BeamOptions, stops, min_tokens: int,
           steps=None, history=None, scores=None) -> None:
    """`ops.beam_select` with the engine's work buffer for scratch; `scores`: those of the rows of `logits` where they are not the
    state's own (the first choice, of one row a sequence)."""
    scores = state.scores if scores is None else scores
    sequences, rows = scores.shape
    floats = ops.beam_select_scratch(sequences, rows, logits.shape[1], options.beams)
    ops.beam_select(parents, tokens.view(parents.shape), state.tensors(), logits, (scores, *state.tensors()[1:]), produced,
                    engine.rt.ws.buffer("beam_scratch", (floats,), torch.float32), tickets, stop_ids=stops, steps=steps,
                    min_tokens=min_tokens, length_penalty=options.length_penalty, early=options.early_stopping, history=history)


def search_batch(engine, prompts: Sequence[np.ndarray], limits: Sequence[int], options: BeamOptions, stops: frozenset,
                 min_tokens: int) -> list[list[BeamResult]]:
    """One batch of prompts through `engine` (every limit is at least 1); results in their order."""
    cache, device, beams, n = engine.cache, engine.rt.device, options.beams, len(prompts)
    slots: list[list[int]] = []
    results: list[list[BeamResult] | None] = [None] * n
    runs = [BeamRun(len(p), limit) for p, limit in zip(prompts, limits)]
    stop_ids = torch.tensor(sorted(stops), dtype=torch.int32, device=device) if stops else None
    held: list[int] = []
    try:
        for _ in range(n):
            slots.append(engine.open(beams))
            held += slots[-1]
        # the prompts, once each, in their first beams' slots; then pages for everything the beams may write
        logits = engine.step([s[0] for s in slots], prompts)
        for mine, limit in zip(slots, limits):
            cache.fork(mine[0], mine[1:], limit)
        cache.sync_tables()
        state = BeamState(n, beams, device)
        parents = torch.zeros((n, beams), dtype=torch.int32, device=device)
        chosen = torch.zeros((n, beams), dtype=torch.int32, device=device)
        produced = torch.zeros(1, dtype=torch.int32, device=device)
        choose(engine, parents, chosen, state, logits, produced, torch.zeros(n, dtype=torch.int32, device=device), options, stop_ids,
               min_tokens, scores=torch.zeros((n, 1), dtype=torch.float32, device=device))
        ops.beam_reorder(cache.beam_rows(), torch.tensor(slots, dtype=torch.int32, device=device), parents,
                         torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=device))
        for run, tokens, came in zip(runs, chosen.tolist(), parents.tolist()):
            run.tokens.append(tokens)
            run.parents.append(came)
        ops.raise_if_failed()
        running = list(range(n))
        while True:
            scores, finished, finished_at, done = (t.tolist() for t in state.tensors())
            still = []
            for row, index in enumerate(running):
                run = runs[index]
                if done[row] or run.produced >= run.limit:
                    results[index] = run.results(options, scores[row], finished[row], finished_at[row], bool(done[row]))
                    engine.close(slots[index])
                    held = [s for s in held if s not in slots[index]]
                else:
                    still.append(row)
            if not still:
                return results  # type: ignore[return-value]
            count = runs[running[still[0]]].produced  # (all sequences start together)
            steps = min(engine.decode_chunk, DecodeGraph.CAPACITY, min(runs[running[row]].limit - count for row in still))
            keep = [running[row] for row in still]
            longest = max(len(prompts[i]) + count + steps for i in keep)
            graph = engine._beam_graph(len(keep), options, longest, min_tokens, tuple(sorted(stops)))
            graph.state.take(state, still)
            graph.load_search([s for i in keep for s in slots[i]], [t for i in keep for t in runs[i].tokens[-1]],
                              [len(prompts[i]) + count - 1 for i in keep for _ in range(beams)], count,
                              [len(prompts[i]) // cache.page_size for i in keep])
            graph.replay(steps)
            engine.steps_run += steps
            tokens, came = graph.histories(steps)
            ops.raise_if_failed()
            for row, index in enumerate(keep):
                runs[index].tokens += list(tokens[:, row])
                runs[index].parents += list(came[:, row])
                for slot in slots[index]:
                    cache.advance(slot, steps)
            state = BeamState(len(keep), beams, device)
            state.take(graph.state, list(range(len(keep))))
            running = keep
    finally:
        if held:
            engine.close(held)
