"""Beam search on the GPU: the choice, the move and the attention over shared pages alone against the plain implementation in
64 bits (tests/plain_beams.py), then whole searches through the engine.

Tolerances, from the arithmetic:
  choice: a row's sum is up to 512 float32 additions a thread deep and joined from a few hundred parts, exp2 is good to 2^-22, so its
    logarithm is off by less than 6e-5; totals of up to 100 are rounded twice to 24 bits (1.2e-5).
  attention in bfloat16: weights and the result are rounded to 8 bits once each: 2^-9 of the largest value twice; float32 scores and
    sums add less than 2^-12 of it at these sizes.
  attention in float32: a score of n products is off by less than n 2^-24 of the sum of their sizes, which moves weights by twice
    that; sums of k weights by k 2^-24."""
import math
import os
import re
import subprocess
import sys

import numpy as np
import pytest
import torch

import gaperax_cases
import plain_beams as PB
import plain_llama as P
import revupel_cases
import satavik_cases
import tezinex_cases
import tisalorn_cases
import zivazen_cases
from helpers import PlainLogits, host, make_engine, model_case, prompts_for, rel_error

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOTAL_TOL = 8e-5


def ops():
    from etalii.dllm_b200.kernels import ops as module

    return module


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---- the choice ------------------------------------------------------------------------------------------------------


class Choice:
    """Inputs of a choice with outputs of their own (or the inputs', `in_place`)."""

    def __init__(self, n, rows, beams, vocab, seed, stops=(), produced=7, in_place=False):
        g = torch.Generator().manual_seed(seed)
        self.n, self.rows, self.beams, self.vocab = n, rows, beams, vocab
        self.logits = torch.randn((n * rows, vocab), generator=g) * 3
        top = torch.randint(0, vocab, (n * rows, 12), generator=g)
        self.logits.scatter_reduce_(1, top, torch.rand((n * rows, 12), generator=g) * 12 + 4, "amax")
        self.scores = -torch.rand((n, rows), generator=g) * 9 - 2
        self.stops = list(stops)
        self.finished = torch.sort(-torch.rand((n, beams), generator=g) * 3, dim=1, descending=True).values
        self.finished[:, max(1, beams // 2):] = -math.inf
        self.finished_at = torch.stack([torch.arange(n * beams).view(n, beams) % max(produced, 1),
                                        torch.arange(n * beams).view(n, beams) % rows], dim=2).to(torch.int32)
        self.finished_at[self.finished == -math.inf] = -1
        self.done = torch.zeros(n, dtype=torch.int32)
        self.produced, self.in_place = produced, in_place and rows == beams

    def run(self, min_tokens=0, penalty=1.0, early=False, steps=None, history=None, repeat=1):
        o = ops()
        state = tuple(t.to(DEV).contiguous() for t in (self.scores, self.finished, self.finished_at, self.done))
        out = state if self.in_place else (torch.full((self.n, self.beams), 7.0, device=DEV), torch.full_like(state[1], 7.0),
                                           torch.full_like(state[2], 77), torch.full_like(state[3], 7))
        parents, tokens = (torch.full((self.n, self.beams), 99, dtype=torch.int32, device=DEV) for _ in range(2))
        scratch = torch.full((o.beam_select_scratch(self.n, self.rows, self.vocab, self.beams),), math.nan, device=DEV)
        self.tickets = torch.zeros(self.n, dtype=torch.int32, device=DEV)
        for _ in range(repeat):
            o.beam_select(parents, tokens, out, self.logits.to(DEV), state, _i32([self.produced]), scratch, self.tickets,
                          stop_ids=_i32(self.stops) if self.stops else None, min_tokens=min_tokens, length_penalty=penalty,
                          early=early, steps=steps, history=history)
        assert int(self.tickets.abs().sum()) == 0
        return [t.cpu() for t in (parents, tokens, *out)]

    def check(self, got, min_tokens=0, penalty=1.0, early=False, produced=None):
        parents, tokens, scores, finished, finished_at, done = got
        produced = self.produced if produced is None else produced
        for b in range(self.n):
            pool = [(float(s), tuple(w)) for s, w in zip(self.finished[b].tolist(), self.finished_at[b].tolist()) if s > -math.inf]
            if self.done[b]:
                assert scores[b].tolist() == [-math.inf] * self.beams and tokens[b].tolist() == [0] * self.beams
                assert parents[b].tolist() == [min(i, self.rows - 1) for i in range(self.beams)] and done[b] == 1
                assert torch.equal(finished[b], self.finished[b]) and torch.equal(finished_at[b], self.finished_at[b])
                continue
            logits = self.logits[b * self.rows:(b + 1) * self.rows].double().numpy()
            places, merged, over = PB.select(logits, self.scores[b].double().tolist(), self.beams, set(self.stops), pool, produced,
                                             min_tokens, penalty, early)
            assert [(int(p), int(t)) for p, t in zip(parents[b], tokens[b])] == [(p, t) for _, p, t in places], b
            want = np.array([s for s, _, _ in places])
            np.testing.assert_array_equal(np.isfinite(want), np.isfinite(scores[b].numpy()))
            live = np.isfinite(want)
            assert np.abs(scores[b].numpy()[live] - want[live]).max(initial=0) <= TOTAL_TOL
            assert [tuple(w) for w in finished_at[b].tolist()][:len(merged)] == [w for _, w in merged]
            assert finished[b].tolist()[len(merged):] == [-math.inf] * (self.beams - len(merged))
            for s, (w, _) in zip(finished[b].tolist(), merged):
                assert abs(s - w) <= TOTAL_TOL
            assert bool(done[b]) == over


@pytest.mark.parametrize("n,rows,beams,vocab", [(1, 1, 1, 1), (2, 1, 4, 3), (1, 4, 4, 5), (3, 4, 4, 401), (2, 3, 5, 2047),
                                                (2, 6, 4, 2049), (1, 16, 16, 4097), (1, 32, 32, 1003), (1, 17, 17, 8195),
                                                (20, 2, 2, 515), (1, 4, 4, 49152), (2, 8, 8, 20001), (1, 1, 32, 30)])
@pytest.mark.parametrize("stops", [(), (2,), (0, 1, 400, 2046)])
def test_choice(n, rows, beams, vocab, stops):
    case = Choice(n, rows, beams, vocab, seed=vocab + rows, stops=stops)
    if n > 1:
        case.done[1] = 1
    case.check(case.run(penalty=0.7, early=True), penalty=0.7, early=True)


@pytest.mark.parametrize("n,rows,beams,vocab", [(1, 16, 16, 33001), (1, 32, 32, 16003), (2, 9, 9, 30011), (1, 16, 32, 9001),
                                                (5, 16, 16, 12289)])
@pytest.mark.parametrize("what", ["any", "one row", "equal rows", "few"])
def test_choice_among_many_lists(n, rows, beams, vocab, what):
    """More candidates in the stretches' lists than a block holds at a time: it goes by the lists' first."""
    case = Choice(n, rows, beams, vocab, seed=vocab + beams, stops=(3, vocab - 1))
    if what == "one row":
        case.scores[:, 1:] = -math.inf  # (one beam lives)
    elif what == "equal rows":
        case.logits[:] = case.logits[0].round()  # (totals tie in every row and list)
        case.scores[:] = -1.0
    elif what == "few":
        case.logits[:, 7:] = -math.inf  # (fewer candidates than lists)
    case.check(case.run(penalty=0.7), penalty=0.7)


@pytest.mark.parametrize("penalty,early", [(0.0, False), (1.0, False), (1.3, True)])
@pytest.mark.parametrize("produced,min_tokens", [(0, 0), (3, 5), (5, 5), (900, 5)])
def test_choice_of_lengths_and_ends(penalty, early, produced, min_tokens):
    case = Choice(4, 4, 4, 300, seed=produced, stops=(1, 7), produced=produced, in_place=True)
    case.logits[::3, 1] = 15.0  # (some texts end)
    if produced == 0:
        case.scores[:, 1:] = -math.inf
    got = case.run(min_tokens=min_tokens, penalty=penalty, early=early)
    case.check(got, min_tokens=min_tokens, penalty=penalty, early=early)


@pytest.mark.parametrize("what", ["equal", "coarse", "ascending", "descending", "one value", "lowest"])
@pytest.mark.parametrize("vocab", [700, 33000])
def test_choice_among_equals_goes_by_the_lower_token(what, vocab):
    """A single row: logits decide, then tokens. (Lists of candidates that do not fit are given up for whole passes.)"""
    case = Choice(1, 1, 8, vocab, seed=3, stops=(5,))
    x = case.logits[0]
    if what == "equal":
        x[:] = 0.25
    elif what == "coarse":
        x.copy_(x.round())
    elif what == "ascending":
        x.copy_(x.sort().values)
    elif what == "descending":
        x.copy_(x.sort(descending=True).values)
    elif what == "one value":
        x[:] = -math.inf
        x[vocab - 1] = 3.0
    else:
        x[:] = torch.finfo(torch.float32).min
    case.check(case.run())


def test_choice_of_rows_without_a_likelihood():
    case = Choice(6, 3, 3, 1000, seed=9, stops=(4,))
    case.logits[0] = -math.inf                 # a row of which nothing is left
    case.logits[4, 500] = math.nan             # not a number
    case.logits[8, 999] = math.inf
    case.logits[9:12] = -math.inf              # a sequence with nothing: over
    case.scores[4] = torch.tensor([-math.inf, -1.0, -math.inf])
    case.scores[5] = torch.tensor([math.nan, -math.inf, -2.0])
    case.logits[15, 10:] = -math.inf           # a grammar that lets ten tokens through
    got = case.run()
    case.scores[5, 0] = -math.inf              # (a score that is not a number is none)
    case.check(got)
    assert got[5].tolist() == [0, 0, 0, 1, 0, 0]


def test_choice_of_the_lowest_value_masks():
    """Masks of the type's lowest value instead of -inf leave a row with candidates of weight 0, in the order of the tokens."""
    case = Choice(1, 2, 4, 50, seed=1)
    case.logits[:] = torch.finfo(torch.float32).min
    case.logits[0, 7], case.logits[1, 9] = 2.0, 3.0
    parents, tokens, scores, *_ = case.run()
    by_score = sorted(zip(scores[0].tolist(), parents[0].tolist(), tokens[0].tolist()), reverse=True)
    best = sorted([(float(case.scores[0, 0]), 0, 7), (float(case.scores[0, 1]), 1, 9)], reverse=True)
    assert [c[1:] for c in by_score[:2]] == [c[1:] for c in best]
    assert by_score[2][0] < -1e38


def test_choice_by_steps_keeps_the_parents():
    case = Choice(3, 4, 4, 500, seed=4, stops=(3,), produced=2)
    case.done[2] = 1
    history = torch.full((6, 3, 4), -5, dtype=torch.int32, device=DEV)
    for step in (0, 4, 5, 6):
        got = case.run(min_tokens=5, steps=_i32([step]), history=history)
        case.check(got, min_tokens=5, produced=2 + step)
        if step < 6:
            assert torch.equal(history[step].cpu(), got[0])
    assert (history[1:4] == -5).all()


def test_choice_twice_gives_the_same_bits_and_runs_on_a_stream_of_its_own():
    case = Choice(5, 8, 8, 50000, seed=6, stops=(3, 9))
    first = case.run()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        second = case.run(repeat=3)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_choice_refusals():
    o = ops()
    good = dict(n=2, rows=4, beams=4, vocab=50, seed=0)

    def call(change):
        case = Choice(**good)
        args = dict(parents=torch.zeros((2, 4), dtype=torch.int32, device=DEV), tokens=torch.zeros((2, 4), dtype=torch.int32, device=DEV),
                    logits=case.logits.to(DEV), scores=case.scores.to(DEV), scratch=torch.zeros(
                        o.beam_select_scratch(2, 4, 50, 4), device=DEV), tickets=torch.zeros(2, dtype=torch.int32, device=DEV),
                    stop_ids=None, history=None)
        args.update(change)
        rest = tuple(t.to(DEV) for t in (case.finished, case.finished_at, case.done))
        o.beam_select(args["parents"], args["tokens"], (torch.zeros((2, 4), device=DEV), *rest), args["logits"], (args["scores"], *rest),
                      _i32([1]), args["scratch"], args["tickets"], stop_ids=args["stop_ids"], history=args["history"])

    call({})
    for change, says in [({"parents": torch.zeros((2, 33), dtype=torch.int32, device=DEV)}, "1 to 32"),
                         ({"stop_ids": _i32(list(range(9)))}, "at most 8"), ({"logits": torch.zeros((7, 50), device=DEV)}, "do not"),
                         ({"logits": torch.zeros((8, 50), dtype=torch.bfloat16, device=DEV)}, "float32"),
                         ({"tokens": torch.zeros((2, 4), dtype=torch.int64, device=DEV)}, "int32"),
                         ({"scratch": torch.zeros(3, device=DEV)}, "scratch"), ({"logits": torch.zeros((8, 50))}, "CUDA"),
                         ({"history": torch.zeros((3, 2, 4), dtype=torch.int32, device=DEV)}, "needs steps"),
                         ({"tickets": torch.zeros(1, dtype=torch.int32, device=DEV)}, "do not")]:
        with pytest.raises(o.KernelError, match=says):
            call(change)
    with pytest.raises(o.KernelError):
        o.beam_select_scratch(0, 4, 50, 4)


def test_choice_refuses_numbers_that_are_not_there():
    case = Choice(1, 2, 2, 50, seed=0)
    case.run(steps=_i32([0]))
    with pytest.raises(ops().KernelError, match="number each"):
        case.run(steps=_i32([]))
    state = tuple(t.to(DEV) for t in (case.scores, case.finished, case.finished_at, case.done))
    out = torch.zeros((1, 2), dtype=torch.int32, device=DEV)
    with pytest.raises(ops().KernelError, match="number each"):
        ops().beam_select(out, out.clone(), state, case.logits.to(DEV), state, _i32([]), torch.zeros(ops().beam_select_scratch(1, 2, 50, 2), device=DEV),
                          _i32([0]))


# ---- the move --------------------------------------------------------------------------------------------------------


def _moved(storage, table, states, slots, parents, lengths, kv_heads, key_dim, value_dim):
    """What beams have after the move, computed on copies (numpy views of whole pages, read before written)."""
    before, table_before = storage.clone(), table.clone()
    states_before = [s.clone() for s in states]
    want, want_table, want_states = storage.clone(), table.clone(), [s.clone() for s in states]
    keys = kv_heads * 64 * key_dim
    for b, length in enumerate(lengths):
        full, rows = length // 64, length % 64
        for i, p in enumerate(parents[b]):
            here, there = int(slots[b][i]), int(slots[b][p])
            want_table[here, :full] = table_before[there, :full]
            if rows:
                mine, theirs = int(table_before[here, full]), int(table_before[there, full])
                for cut, dim in ((slice(0, keys), key_dim), (slice(keys, None), value_dim)):
                    if dim:
                        to = want[:, mine, cut].reshape(storage.shape[0], kv_heads, 64, dim)
                        to[:, :, :rows] = before[:, theirs, cut].reshape(storage.shape[0], kv_heads, 64, dim)[:, :, :rows]
                        want[:, mine, cut] = to.reshape(storage.shape[0], -1)
            for state, old in zip(want_states, states_before):
                state[here] = old[there]
    return want, want_table, want_states


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("beams,kind", [(2, "ring"), (4, "random"), (5, "ring"), (8, "first"), (11, "random"), (32, "random"), (3, "stay")])
@pytest.mark.parametrize("kv_heads,key_dim,value_dim", [(2, 16, 16), (1, 24, 8), (3, 40, 0)])
def test_move(dtype, beams, kind, kv_heads, key_dim, value_dim):
    from etalii.dllm_b200.cache.beams import CacheRows

    g = torch.Generator().manual_seed(beams + key_dim)
    lengths = [0, 1, 63, 64, 65, 150]
    n = len(lengths)
    pages = n * beams * 3 + 4
    per_page = kv_heads * 64 * (key_dim + value_dim)
    storage = torch.randn((3, pages, per_page), generator=g).to(dtype)
    ids = torch.randperm(pages, generator=g)[: n * beams * 3].to(torch.int32).view(n * beams, 3)
    table = torch.full((n * beams + 2, 4), 0, dtype=torch.int32)
    slots = torch.randperm(n * beams + 2, generator=g)[: n * beams].to(torch.int32).view(n, beams)
    table[slots.view(-1).long(), :3] = ids
    states = [torch.randn((n * beams + 2, *shape), generator=g) for shape in ((3,), (5, 7, 11), (40, 130), (4,))]
    parents = {"ring": torch.arange(beams).roll(1).repeat(n, 1), "first": torch.zeros((n, beams), dtype=torch.long),
               "stay": torch.arange(beams).repeat(n, 1),
               "random": torch.randint(0, beams, (n, beams), generator=g)}[kind].to(torch.int32)
    want = _moved(storage, table, states, slots, parents.tolist(), lengths, kv_heads, key_dim, value_dim)
    dev = storage.to(DEV), table.to(DEV), [s.to(DEV) for s in states]
    rows = CacheRows([(dev[0], dev[1], kv_heads, key_dim, value_dim)], dev[2], 64)
    # lengths one a beam, one short (`ahead`): a sequence's first counts
    each = (torch.tensor(lengths)[:, None] - 1 + torch.arange(beams)[None, :] * 1000).to(torch.int32).to(DEV).contiguous()
    ops().beam_reorder(rows, slots.to(DEV), parents.to(DEV), each, ahead=1)
    assert torch.equal(dev[0].cpu(), want[0]) and torch.equal(dev[1].cpu(), want[1])
    # (at length 0 nothing has been computed yet: states stay)
    for got, state, old in zip(dev[2], want[2], states):
        state[slots[0].long()] = old[slots[0].long()]
        assert torch.equal(got.cpu(), state)


def test_move_leaves_alone_what_does_not_exist():
    """Parents, slots and page numbers outside their ranges are skipped: nothing is read or written there."""
    from etalii.dllm_b200.cache.beams import CacheRows

    storage = torch.randn((1, 4, 64 * 32), device=DEV)
    table = _i32([[0, 9], [1, 1], [2, 2]])
    state = torch.randn((3, 8), device=DEV)
    before = storage.clone(), state.clone(), table.clone()
    rows = CacheRows([(storage, table, 1, 16, 16)], [state], 64)
    ops().beam_reorder(rows, _i32([[0, 1]]), _i32([[7, -1]]), _i32([10]))   # no such parents
    ops().beam_reorder(rows, _i32([[0, 50]]), _i32([[1, 0]]), _i32([10]))   # no such slot
    ops().beam_reorder(rows, _i32([[0, 1]]), _i32([[1, 1]]), _i32([300]))   # positions beyond the table's row
    torch.cuda.synchronize()
    assert torch.equal(storage, before[0])
    assert torch.equal(state[1:], before[1][1:]) and torch.equal(table[1:], before[2][1:])


def test_move_refusals():
    from etalii.dllm_b200.cache.beams import CacheRows

    o, state = ops(), torch.zeros((4, 8), device=DEV)
    rows = CacheRows([], [state], 64)
    for slots, parents, lengths, says in [
            (_i32([[0, 1]]), _i32([list(range(33))]), _i32([1]), "1 to 32"), (_i32([[0, 1, 2]]), _i32([[0, 1]]), _i32([1]), "slots"),
            (_i32([[0, 1]]), _i32([[0, 1]]), _i32([1, 2, 3]), "lengths"), (_i32([[0, 1]]).long(), _i32([[0, 1]]), _i32([1]), "int32"),
            (_i32([[0, 1]]).cpu(), _i32([[0, 1]]), _i32([1]), "CUDA")]:
        with pytest.raises(o.KernelError, match=says):
            o.beam_reorder(rows, slots, parents, lengths)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
def test_move_is_over_before_the_attention_behind_it_reads(dtype, dim):
    """Attention asks for positions, page tables and rows of earlier steps ahead of its wait: right behind a move, in one graph, it
    gives what it gives when the move has long been over."""
    from types import SimpleNamespace

    from etalii.dllm_b200.cache.beams import CacheRows
    from etalii.dllm_b200.cache.paged import KvView

    o, beams, n, layers, kv_heads, length = ops(), 8, 3, 24, 4, 300
    g = torch.Generator().manual_seed(dim)
    count = n * beams
    storage = torch.randn((layers, count * 6, 2, kv_heads, 64, dim), generator=g).to(dtype).to(DEV)
    table = torch.randperm(count * 6, generator=g).to(torch.int32).view(count, 6).contiguous().to(DEV)
    slots, parents = _i32(list(range(count))), _i32([[(i + 1) % beams for i in range(beams)]] * n)
    q = (torch.randn((count, 2 * kv_heads * dim), generator=g) * 1.5).to(dtype).to(DEV)
    rows = CacheRows([(storage, table, kv_heads, dim, dim)], [], 64)
    view = KvView(storage[layers - 1], table, 64, kv_heads, dim, None)
    batch = SimpleNamespace(tok_pos=_i32([length - 1] * count), tok_seq=_i32(list(range(count))), slots=slots, n_seqs=count, n_tokens=count,
                            max_new=1, max_context=length, tile_seq=_i32([0]), tile_first=_i32([0]), cu_seqlens=_i32(list(range(count + 1))),
                            n_tiles=0)
    lengths = _i32([length] * n)

    def attend(out):
        kernel = o.attention_decode_cluster if dtype == torch.bfloat16 else o.attention_blocks
        kernel(out, q, view, 2 * kv_heads, dim ** -0.5, 0, batch)

    behind, alone = torch.empty_like(q), torch.empty_like(q)
    attend(behind)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            o.beam_reorder(rows, slots.view(n, beams), parents, lengths)
            attend(behind)
    for _ in range(20):
        graph.replay()
        torch.cuda.synchronize()
        attend(alone)
        torch.cuda.synchronize()
        assert torch.equal(behind, alone)
    o.raise_if_failed()


# ---- attention over shared pages -------------------------------------------------------------------------------------


class Pages:
    """Groups of tokens over a paged entry. groups: a list of (common positions, [each token's position]); "beams": every token
    has a row of the table of its own, full pages of `common` in all of them; "chunk": one row for all. `join`: pages that
    neighbouring beams have in common behind them, as lines that part late."""

    def __init__(self, kind, groups, heads, kv_heads, dim, dtype, seed=0, join=False, values=1.0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.dtype = heads, kv_heads, dim, dtype
        rows, self.slots, self.positions, self.shared, self.cuts, used = [], [], [], [], [0], 0
        for common, newest in groups:
            last = max(max(newest), 0) // 64 + 1
            full = common // 64 if kind == "beams" else last
            prefix = list(range(used, used + full))
            used += full
            for i in range(len(newest) if kind == "beams" else 1):
                rows.append(prefix + [used + j * len(newest) + (i - i % 2 if join and j < last - full - 1 else i)
                                      for j in range(last - full)])
            used += (last - full) * len(newest)
            self.slots += list(range(len(rows) - len(newest), len(rows))) if kind == "beams" else [len(rows) - 1] * len(newest)
            self.positions += newest
            self.shared.append(full)
            self.cuts.append(len(self.positions))
        self.width = max(len(r) for r in rows) + 1
        perm = torch.randperm(used + 2, generator=g)
        self.table = torch.zeros((len(rows), self.width), dtype=torch.int32)
        for i, r in enumerate(rows):
            self.table[i, :len(r)] = perm[torch.tensor(r, dtype=torch.long)].to(torch.int32)
        self.storage = (torch.randn((used + 2, 2, kv_heads, 64, dim), generator=g) * values).to(dtype)
        self.q = (torch.randn((len(self.positions), heads * dim), generator=g) * 1.5).to(dtype)
        self.max_rows = max(len(p) for _, p in groups)
        self.max_context = max(max(max(p) for _, p in groups) + 1, 1)
        self.scale = dim ** -0.5

    def run(self, window=0, scale=None, shared=None, repeat=1, max_rows=None):
        from etalii.dllm_b200.cache.paged import KvView

        o = ops()
        view = KvView(self.storage.to(DEV), self.table.to(DEV), 64, self.kv_heads, self.dim, window or None)
        floats, words = o.attention_shared_scratch(view, self.heads, len(self.cuts) - 1, max_rows or self.max_rows, self.max_context)
        scratch = torch.full((max(floats, 1),), math.nan, device=DEV)
        tickets = torch.zeros(words, dtype=torch.int32, device=DEV)
        q = self.q.to(DEV)
        out = torch.full_like(q, 7.0)
        for _ in range(repeat):
            o.attention_shared(out, q, view, self.heads, self.scale if scale is None else scale, window, _i32(self.slots),
                               _i32(self.positions), _i32(self.cuts), _i32(self.shared if shared is None else shared),
                               max_rows or self.max_rows, self.max_context, scratch, tickets)
        torch.cuda.synchronize()
        if max_rows is None:
            o.raise_if_failed()
        assert int(tickets.abs().sum()) == 0
        return out.float().cpu().numpy()

    def want(self, window=0, scale=None):
        return PB.attend(self.q.double().numpy(), self.storage.double().numpy(), self.table.numpy(), self.slots, self.positions, self.heads,
                         self.kv_heads, self.scale if scale is None else scale, window)

    def tolerance(self, scale=None):
        largest = float(self.storage[:, 1].double().abs().max())
        scale = abs(self.scale if scale is None else scale)
        sizes = float(self.q.double().abs().max()) * float(self.storage[:, 0].double().abs().max()) * self.dim * scale
        exact = (2 * (self.dim + 4) * sizes + self.max_context + 64) * 2.0 ** -24
        return largest * (exact if self.dtype == torch.float32 else 2.0 ** -8 + 2.0 ** -11)

    def check(self, window=0, scale=None, **how):
        got, want = self.run(window, scale, **how), self.want(window, scale)
        assert np.isfinite(got).all()
        assert np.abs(got - want).max() <= self.tolerance(scale)
        return got


DTYPES = [torch.float32, torch.bfloat16]
BEAMS = [(0, [0, 0, 0]), (70, [75, 75, 75, 75]), (128, [128, 128]), (200, [190 + 64] * 5), (63, [63])]
CHUNKS = [(0, [0, 1, 2]), (0, [62, 63, 64, 65, 66]), (0, [127]), (0, [300, 301]), (0, [63])]
HEADS = [(4, 2, 64), (9, 3, 64), (8, 2, 128), (6, 6, 80), (16, 1, 96), (8, 1, 112), (4, 2, 16), (6, 3, 32), (6, 2, 48), (6, 3, 24), (2, 1, 8),
         (4, 2, 72), (4, 1, 136), (2, 2, 256), (64, 1, 64), (40, 1, 128), (33, 1, 32)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("kind,groups", [("beams", BEAMS), ("chunk", CHUNKS)])
def test_attention_over_shared_pages(dtype, heads, kv_heads, dim, kind, groups):
    Pages(kind, groups, heads, kv_heads, dim, dtype, seed=dim, join=True).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 40, 64, 128])
@pytest.mark.parametrize("window", [1, 40, 64, 100, 129])
def test_attention_windows(dtype, dim, window):
    Pages("beams", BEAMS, 6, 2, dim, dtype, seed=window).check(window=window)
    Pages("chunk", CHUNKS, 6, 2, dim, dtype, seed=window).check(window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 40, 64, 128])
def test_attention_of_tokens_that_see_nothing(dtype, dim):
    pages = Pages("beams", [(70, [100, -1, 100, -1]), (5, [-1, -1]), (0, [-1, 0])], 6, 2, dim, dtype)
    got = pages.check()
    assert (got[[1, 3, 4, 5, 6]] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 40, 64, 128])
@pytest.mark.parametrize("splits", ["one", "several"])
def test_attention_leaves_alone_what_is_not_seen(dtype, dim, splits):
    """NaN and infinities in rows of a page that nobody has written, in the text of another beam, and in a later token of a chunk
    stay where they are; a token that sees one has it in its result."""
    copies = 1 if splits == "several" else 60
    beams = Pages("beams", [(70, [100, 100, 90])] * copies, 4, 2, dim, dtype)
    clean, tolerance = beams.run(), beams.tolerance() * 2  # (such a page may be added in another order)
    table = beams.table.long()
    beams.storage[table[0, 1], :, :, 101 - 64:] = math.nan           # nobody's rows
    beams.storage[table[1, 1], 1, :, 95 - 64] = math.inf             # the second beam's own text
    beams.storage[table[1, 1], 0, :, 96 - 64] = math.nan
    beams.storage[table[2, 1], 1, :, 91 - 64:] = -math.inf           # behind the third beam's position
    got = beams.run()
    keep = [t for t in range(len(beams.positions)) if t != 1]
    assert np.abs(got[keep] - clean[keep]).max() <= tolerance and np.isnan(got[1]).all()
    chunk = Pages("chunk", [(0, [70, 71, 72, 73])] * copies, 4, 2, dim, dtype)
    clean, tolerance = chunk.run(), chunk.tolerance() * 2
    page = chunk.table.long()[0, 1]
    chunk.storage[page, 1, 1, 72 - 64, 3] = math.nan                 # one value of the third token, kv head 1
    chunk.storage[page, 1, 1, 73 - 64, 5] = math.inf
    got = chunk.run().reshape(-1, 4, dim)
    clean = clean.reshape(-1, 4, dim)
    changed = np.zeros(got.shape, bool)
    changed[2:4, 2:, 3] = True
    changed[3, 2:, 5] = True
    assert np.isnan(got[2:4, 2:, 3]).all() and (got[3, 2:, 5] == np.inf).all()
    assert np.abs(got[~changed] - clean[~changed]).max() <= tolerance and np.isfinite(got[~changed]).all()


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 32), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_attention_of_long_contexts(dtype, dim):
    """Contexts of which every block has several steps; weights that keep growing (a maximum renewed in every step)."""
    pages = Pages("chunk", [(0, list(range(5000, 5006))), (0, [4099])], 8, 2, dim, dtype, seed=1)
    pages.check()
    grows = Pages("beams", [(3000, [3100] * 4)], 4, 1, dim, dtype, seed=2)
    q = grows.q.view(4, 4, dim)
    order = torch.arange(3200, dtype=torch.float64) / 3200 * 4
    for row in grows.table.long():
        for index in range(3100 // 64 + 1):
            at = order[index * 64:(index + 1) * 64]
            grows.storage[row[index], 0, 0, :len(at)] = (q[0, 0].double()[None, :] * at[:, None] / dim ** 0.5).to(dtype)
    grows.check()


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 32), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_attention_of_many_tokens_a_group(dtype, dim):
    """More tokens than a lane each (own pages are then walked token by token), more query rows than a tile, pages in common that
    the caller does not name, own pages that do not fit the list."""
    Pages("beams", [(64, [130] * 70), (10, [20] * 3)], 2, 2, dim, dtype, seed=3).check()
    Pages("chunk", [(0, list(range(100, 170)))], 6, 2, dim, dtype, seed=4).check()
    unnamed = Pages("beams", [(640, [700] * 6), (64, [80] * 6)], 4, 2, dim, dtype, seed=5)
    a, b = unnamed.check(), unnamed.check(shared=[0, 0])
    assert np.abs(a - b).max() <= unnamed.tolerance()
    Pages("beams", [(0, [1500] * 12)], 2, 1, dim, dtype, seed=6).check()


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 32), (torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_attention_scales(dtype, dim, scale):
    Pages("beams", BEAMS, 4, 2, dim, dtype, seed=7).check(scale=scale)


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 32), (torch.bfloat16, 64), (torch.bfloat16, 128)])
def test_attention_twice_gives_the_same_bits(dtype, dim):
    pages = Pages("chunk", [(0, [9000, 9001, 9002])], 8, 2, dim, dtype, seed=8)
    first = pages.run()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        assert np.array_equal(first, pages.run(repeat=3))


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 24), (torch.float32, 72), (torch.float32, 80), (torch.float32, 136), (torch.bfloat16, 48),
                                       (torch.bfloat16, 80), (torch.bfloat16, 96), (torch.bfloat16, 112), (torch.bfloat16, 136)])
def test_attention_of_several_clusters_whose_rows_do_not_divide_a_block(dtype, dim):
    """Contexts that several clusters share, head sizes whose rows' pieces do not end where a block's threads do, other values in the
    same scratch from call to call: each output row takes its maximum and sum from its own call."""
    from etalii.dllm_b200.cache.paged import KvView

    o = ops()
    both = [Pages("chunk", [(0, list(range(9000, 9008)))] * n, 8, 1, dim, dtype, seed=n, values=v) for n, v in ((1, 1.0), (2, 4.0))]
    sizes = [o.attention_shared_scratch(KvView(p.storage.to(DEV), p.table.to(DEV), 64, 1, dim, None), 8, len(p.cuts) - 1, 8, 9008) for p in both]
    assert all(floats > 0 and words > 0 for floats, words in sizes)  # (several clusters)
    scratch = torch.full((max(floats for floats, _ in sizes),), math.nan, device=DEV)
    tickets = torch.zeros(max(words for _, words in sizes), dtype=torch.int32, device=DEV)
    calls = []
    for p in both:
        view = KvView(p.storage.to(DEV), p.table.to(DEV), 64, 1, dim, None)
        q, want = p.q.to(DEV), p.want()
        calls.append((p, view, q, want, [_i32(x) for x in (p.slots, p.positions, p.cuts, p.shared)]))
    results = []
    for _ in range(3):
        for p, view, q, want, rest in calls:
            out = torch.full_like(q, 7.0)
            o.attention_shared(out, q, view, 8, p.scale, 0, *rest, 8, 9008, scratch, tickets)
            results.append(out.float().cpu().numpy())
            assert np.abs(results[-1] - want).max() <= p.tolerance()
    o.raise_if_failed()
    assert all(np.array_equal(results[i], results[i + 2]) for i in range(4)) and int(tickets.abs().sum()) == 0


def test_attention_in_storage_beyond_32_bits():
    """Pages whose values lie more than 2^32 bytes and 2^31 values from the entry's start."""
    from etalii.dllm_b200.cache.paged import KvView

    o = ops()
    for dtype, dim in ((torch.bfloat16, 128), (torch.float32, 64)):
        pages = (1 << 31) // (2 * 8 * 64 * dim) + 40
        storage = torch.zeros((pages, 2, 8, 64, dim), dtype=dtype, device=DEV)
        small = Pages("chunk", [(0, [140, 141])], 8, 8, dim, dtype, seed=9)
        last = pages - 1 - torch.arange(small.storage.shape[0])
        storage[last.to(DEV)] = small.storage.to(DEV)
        table = (pages - 1 - small.table).to(DEV)
        view = KvView(storage, table, 64, 8, dim, None)
        floats, words = o.attention_shared_scratch(view, 8, 1, 2, 142)
        out = torch.empty((2, 8 * dim), dtype=dtype, device=DEV)
        o.attention_shared(out, small.q.to(DEV), view, 8, small.scale, 0, _i32(small.slots), _i32(small.positions), _i32(small.cuts),
                           _i32(small.shared), 2, 142, torch.empty(max(floats, 1), device=DEV), torch.zeros(words, dtype=torch.int32, device=DEV))
        assert np.abs(out.float().cpu().numpy() - small.want()).max() <= small.tolerance()
        del storage, view


def test_attention_of_more_tokens_than_the_launch_was_told():
    o = ops()
    for dim, dtype in ((64, torch.bfloat16), (32, torch.bfloat16), (64, torch.float32)):
        Pages("chunk", [(0, list(range(100, 170)))], 6, 2, dim, dtype).run(max_rows=4)
        with pytest.raises(o.KernelError, match="max_rows"):
            o.raise_if_failed()
        o.raise_if_failed()


def test_attention_refusals():
    from etalii.dllm_b200.cache.paged import KvView

    o = ops()

    def call(dim=64, dtype=torch.bfloat16, page=64, heads=4, kv_heads=2, **change):
        view = KvView(torch.zeros((4, 2, kv_heads, page, dim), dtype=dtype, device=DEV), _i32([[0, 1]]), page, kv_heads, dim, None)
        q = torch.zeros((2, heads * dim), dtype=dtype, device=DEV)
        args = dict(out=torch.zeros_like(q), q=q, slots=_i32([0, 0]), positions=_i32([3, 4]), groups=_i32([0, 2]), shared=_i32([2]),
                    max_rows=2, max_context=100, scratch=torch.zeros(1 << 16, device=DEV), tickets=torch.zeros(64, dtype=torch.int32, device=DEV))
        args.update(change)
        o.attention_shared(args["out"], args["q"], view, heads, 0.1, 0, args["slots"], args["positions"], args["groups"], args["shared"],
                           args["max_rows"], args["max_context"], args["scratch"], args["tickets"])

    call()
    bad = torch.zeros((2, 256), device=DEV)
    for change, says in [(dict(dim=60), "multiple of 8"), (dict(dim=264), "multiple of 8"), (dict(page=32), "64"),
                         (dict(dtype=torch.float16), "float16"), (dict(heads=3), "heads"), (dict(q=bad), "q torch.float32"),
                         (dict(out=torch.zeros((1, 256), dtype=torch.bfloat16, device=DEV)), "out"), (dict(slots=_i32([0])), "slots"),
                         (dict(positions=_i32([3, 4]).long()), "int32"), (dict(scratch=torch.zeros(64, device=DEV, dtype=torch.float64)), "float32"),
                         (dict(max_context=200), "table rows"), (dict(max_rows=0), "unsupported|argument"),
                         (dict(q=torch.zeros((2, 256), dtype=torch.bfloat16)), "CUDA")]:
        with pytest.raises(o.KernelError, match=says):
            call(**change)
    long = Pages("chunk", [(0, [9000, 9001])], 4, 2, 64, torch.bfloat16)
    view = KvView(long.storage.to(DEV), long.table.to(DEV), 64, 2, 64, None)
    floats, words = o.attention_shared_scratch(view, 4, 1, 2, 9002)
    for scratch, tickets in ((floats - 1, words), (floats, words - 1)):
        with pytest.raises(o.KernelError, match="tickets"):
            o.attention_shared(long.q.to(DEV), long.q.to(DEV), view, 4, 0.1, 0, _i32(long.slots), _i32(long.positions), _i32(long.cuts),
                               _i32(long.shared), 2, 9002, torch.zeros(scratch, device=DEV), torch.zeros(tickets, dtype=torch.int32, device=DEV))


def test_attention_refuses_scratch_that_is_not_aligned():
    from etalii.dllm_b200.cache.paged import KvView

    o = ops()
    for dtype, dim in ((torch.float32, 64), (torch.bfloat16, 32), (torch.bfloat16, 128)):
        long = Pages("chunk", [(0, [9000, 9001])], 4, 2, dim, dtype)
        view = KvView(long.storage.to(DEV), long.table.to(DEV), 64, 2, dim, None)
        floats, words = o.attention_shared_scratch(view, 4, 1, 2, 9002)
        q = long.q.to(DEV)
        for offset in (1, 2, 3):
            with pytest.raises(o.KernelError, match="aligned"):
                o.attention_shared(torch.empty_like(q), q, view, 4, 0.1, 0, _i32(long.slots), _i32(long.positions), _i32(long.cuts),
                                   _i32(long.shared), 2, 9002, torch.zeros(floats + 4, device=DEV)[offset:],
                                   torch.zeros(words, dtype=torch.int32, device=DEV))


# ---- whole searches --------------------------------------------------------------------------------------------------


def _compare(found, want, tolerance):
    assert [r.tokens for r in found] == [tuple(t) for t, _, _ in want]
    assert [r.finish_reason for r in found] == [reason for _, _, reason in want]
    for result, (_, score, _) in zip(found, want):
        assert abs(result.score - score) <= tolerance


@pytest.mark.parametrize("tag", ["a", "b"])
@pytest.mark.parametrize("beams,penalty,early", [(1, 1.0, False), (3, 1.0, False), (4, 0.0, True), (6, 1.4, False)])
@pytest.mark.parametrize("graphs", [True, False])
def test_search_is_the_plain_search(tag, beams, penalty, early, graphs):
    """Prompts whose ends lie before, on and behind a page's end; texts that cross one; stop tokens that come up."""
    from etalii.dllm_b200.sampling.beams import BeamOptions

    config, weights = model_case(tag)
    engine = make_engine(config, weights, "float32", cuda_graphs=graphs, decode_chunk=5)
    logits_of = PlainLogits(config, weights)
    prompts = prompts_for(config, [5, 60, 64, 70])
    options = BeamOptions(beams=beams, length_penalty=penalty, early_stopping=early)
    for stops in ((), tuple(range(0, config["vocab_size"], 55))):
        found = engine.beam_search(prompts, 12, options, stop_token_ids=stops, ignore_eos=True, min_tokens=2 if stops else 0)
        for prompt, texts in zip(prompts, found):
            want = PB.search(lambda text: logits_of(text)[-1], prompt, beams, 12, stops, penalty, early, 2 if stops else 0)
            _compare(texts, want, 2e-3)
            assert all(r.prompt_tokens == len(prompt) for r in texts)
    engine.cache.check()
    assert engine.cache.slots.held == 0 and engine.cache.pages_held() == 0


@pytest.mark.parametrize("dtype,head_dim", [("float32", 32), ("float32", 64), ("bfloat16", 32), ("bfloat16", 64), ("bfloat16", 72)])
def test_search_whose_beams_read_shared_pages(dtype, head_dim, monkeypatch):
    """The same search with the attention that reads pages once and with the one that reads every beam's (what a step takes goes by
    its size otherwise): the same texts in float32, scores within the rounding of the logits."""
    from etalii.dllm_b200.parts import attention
    from etalii.dllm_b200.sampling.beams import BeamOptions

    config, _ = model_case("a")
    config = {**config, "num_attention_heads": 4, "num_key_value_heads": 2, "head_dim": head_dim, "max_position_embeddings": 512}
    weights = P.random_weights(config, 6, std=0.08)
    prompts = prompts_for(config, [20, 128, 200])
    found = []
    for least in (0, 1 << 60):
        monkeypatch.setattr(attention, "SHARED_FROM_BYTES", {d: (least, least) for d in attention.SHARED_FROM_BYTES})
        monkeypatch.setattr(attention, "reads_shared_pages",
                            lambda batch, cache, least=least: getattr(batch, "shared", None) is not None and least == 0)
        engine = make_engine(config, weights, dtype, max_tokens=4096)
        before = ops().launches
        found.append(engine.beam_search(prompts, 70, BeamOptions(beams=3), ignore_eos=True))
        assert ops().launches > before
    for one, other in zip(*found):
        if dtype == "float32":
            assert [r.tokens for r in one] == [r.tokens for r in other]
        assert abs(one[0].score - other[0].score) <= (1e-3 if dtype == "float32" else 0.06)


@pytest.fixture
def calls(monkeypatch):
    """How often each attention operator of single tokens has been called."""
    module, count = ops(), {}
    for name in ("attention_shared", "attention_decode_cluster", "attention_decode", "attention_blocks"):
        def counted(*a, name=name, inner=getattr(module, name), **k):
            count[name] = count.get(name, 0) + 1
            return inner(*a, **k)

        monkeypatch.setattr(module, name, counted)
    return count


@pytest.mark.parametrize("beams,taken,left", [(8, "attention_shared", "attention_decode_cluster"),
                                              (4, "attention_decode_cluster", "attention_shared")])
def test_search_reads_shared_pages_where_the_rule_says_so(beams, taken, left, calls):
    """8 kv heads of 128, contexts of up to 1,024: eight beams are 32 MB of keys and values a layer, four are 16."""
    from etalii.dllm_b200.sampling.beams import BeamOptions

    config, _ = model_case("a")
    config = {**config, "num_attention_heads": 16, "num_key_value_heads": 8, "head_dim": 128, "max_position_embeddings": 1024}
    engine = make_engine(config, P.random_weights(config, 6, std=0.08), "bfloat16", max_tokens=8192, max_length=1024)
    found = engine.beam_search(prompts_for(config, [200]), 20, BeamOptions(beams=beams), ignore_eos=True)
    assert calls.get(taken, 0) > 0 and calls.get(left, 0) == 0 and len(found[0]) == beams


@pytest.mark.parametrize("dtype,head_dim,other", [("float32", 64, "attention_blocks"), ("bfloat16", 64, "attention_decode_cluster"),
                                                  ("bfloat16", 128, "attention_decode_cluster")])
def test_search_finds_the_same_by_either_attention(dtype, head_dim, other, calls, monkeypatch):
    """The rule moved to either side: the operator that it names runs and the other does not; float32 finds the same texts."""
    from etalii.dllm_b200.parts import attention
    from etalii.dllm_b200.sampling.beams import BeamOptions

    config, _ = model_case("a")
    config = {**config, "num_attention_heads": 4, "num_key_value_heads": 2, "head_dim": head_dim, "max_position_embeddings": 512}
    weights = P.random_weights(config, 6, std=0.08)
    prompts = prompts_for(config, [20, 128, 200])
    reads, found = attention.reads_shared_pages, []
    for shared in (True, False):
        monkeypatch.setattr(attention, "SHARED_FROM_BYTES", {d: (0, 0) if shared else (1 << 60, 1 << 60) for d in attention.SHARED_FROM_BYTES})
        # (the MB for each prompt and kv head is the rule's too: a step that counts as many positions as that takes)
        monkeypatch.setattr(attention, "reads_shared_pages", lambda batch, cache: reads(
            type("Step", (), {**vars(batch), "max_context": 1 << 24}), cache) if getattr(batch, "shared", None) is not None else False)
        engine = make_engine(config, weights, dtype, max_tokens=4096)
        calls.clear()
        found.append(engine.beam_search(prompts, 40, BeamOptions(beams=3), ignore_eos=True))
        ran, kept = ("attention_shared", other) if shared else (other, "attention_shared")
        decoded = calls.get(ran, 0) - (config["num_hidden_layers"] if ran == "attention_blocks" else 0)  # (the prompt's step)
        assert decoded > 0
        assert calls.get(kept, 0) == (config["num_hidden_layers"] if kept == "attention_blocks" else 0)
    for one, two in zip(*found):
        if dtype == "float32":
            assert [r.tokens for r in one] == [r.tokens for r in two]
        assert abs(one[0].score - two[0].score) <= (1e-3 if dtype == "float32" else 0.06)


def test_one_beam_is_the_greedy_choice():
    from etalii.dllm_b200.sampling.beams import BeamOptions

    config, weights = model_case("a")
    for dtype in ("float32", "bfloat16"):
        engine = make_engine(config, weights, dtype)
        prompts = prompts_for(config, [3, 30])
        greedy = engine.generate(prompts, 20, ignore_eos=True)
        beams = engine.beam_search(prompts, 20, BeamOptions(beams=1), ignore_eos=True)
        if dtype == "float32":
            assert [b[0].tokens for b in beams] == [g.tokens for g in greedy]
        assert all(len(b) == 1 and len(b[0].tokens) == 20 and b[0].finish_reason == "length" for b in beams)


ARCHITECTURES = {"tisalorn": tisalorn_cases, "satavik": satavik_cases, "revupel": revupel_cases, "gaperax": gaperax_cases,
                 "tezinex": tezinex_cases, "zivazen": zivazen_cases}


@pytest.mark.parametrize("name", sorted(ARCHITECTURES))
def test_search_of_every_architecture(name):
    """Against a search that runs every text as a prompt of its own through the same engine's step function: states, windows,
    chunks and borrowed keys move with the beams. (float32, whose logits do not depend on how a text was cut.)"""
    from etalii.dllm_b200.sampling.beams import BeamOptions

    module = ARCHITECTURES[name]
    for tag, config in sorted(module.CASES.items())[:2]:
        config = config() if callable(config) else config
        weights = module.make_weights(config, 1) if hasattr(module, "make_weights") else module.random_weights(config, 1)
        engine = module.make_engine(config, weights, "float32", max_tokens=4096, decode_chunk=4)
        prompts = module.tokens_for(config, [9, 61, 130])

        def logits_of(text):
            slot = engine.open(1)
            out = host(engine.step(slot, [text]))[0]
            engine.close(slot)
            return out

        found = engine.beam_search(prompts, 9, BeamOptions(beams=3), stop_token_ids=[7], ignore_eos=True)
        for prompt, texts in zip(prompts, found):
            _compare(texts, PB.search(logits_of, prompt, 3, 9, (7,)), 5e-3)


def test_search_in_bfloat16_finds_texts_as_good():
    """bfloat16 rounds activations, so texts may differ where scores are close: the best text's score is within the error of the
    logits of the plain search's."""
    from etalii.dllm_b200.sampling.beams import BeamOptions

    config, weights = model_case("a")
    config = {**config, "num_attention_heads": 2, "num_key_value_heads": 1, "head_dim": 64, "max_position_embeddings": 512}
    weights = P.random_weights(config, 3, std=0.08)
    engine = make_engine(config, weights, "bfloat16", max_tokens=4096)
    logits_of = PlainLogits(config, weights)
    prompts = prompts_for(config, [20, 127, 200])
    found = engine.beam_search(prompts, 10, BeamOptions(beams=4), ignore_eos=True)
    for prompt, texts in zip(prompts, found):
        want = PB.search(lambda text: logits_of(text)[-1], prompt, 4, 10)
        for result in texts:  # each text's own score
            rows = PB.log_probabilities(logits_of(list(prompt) + list(result.tokens))[len(prompt) - 1:-1])
            own = sum(rows[i][t] for i, t in enumerate(result.tokens)) / 10
            assert abs(own - result.score) <= 0.06
        assert texts[0].score >= want[0][1] - 0.06


def test_search_in_batches_and_its_limits():
    from etalii.dllm_b200.engine.generate import ContextLengthError
    from etalii.dllm_b200.sampling.beams import BeamOptions

    config, weights = model_case("a")
    engine = make_engine(config, weights, "float32", max_tokens=640)
    prompts = prompts_for(config, [5, 9, 70, 100])
    options = BeamOptions(beams=3)
    together = make_engine(config, weights, "float32", max_tokens=8192).beam_search(prompts, 30, options, ignore_eos=True)
    assert engine.beam_search(prompts, 30, options, ignore_eos=True) == together  # (several batches)
    assert engine.beam_search(prompts, 30, options, ignore_eos=True, max_batch=1) == together
    assert len(together[3][0].tokens) == 28  # the context window (128)
    assert engine.beam_search([[1, 2]], 0, options)[0][0].tokens == ()
    with pytest.raises(ContextLengthError):
        make_engine(config, weights, "float32", max_tokens=128).beam_search(prompts, 30, options)
    with pytest.raises(ValueError, match="at most 8"):
        engine.beam_search(prompts, 30, options, stop_token_ids=range(20))
    with pytest.raises(ValueError, match="min_tokens"):
        engine.beam_search(prompts, 30, options, min_tokens=-1)
    assert engine.cache.slots.held == 0 and engine.cache.pages_held() == 0
    assert engine.generate(prompts[:1], 4, ignore_eos=True)[0].tokens  # the engine goes on as before


@pytest.mark.parametrize("penalty", [20.0, 1e30, 1e300])
def test_search_refuses_a_penalty_that_leaves_no_score(penalty):
    """(tokens) ** penalty beyond float32 would give every text that has ended the score -0, or raise in the middle of a search."""
    from etalii.dllm_b200.sampling.beams import BeamOptions

    config, weights = model_case("a")
    engine = make_engine(config, weights, "float32")
    prompts = prompts_for(config, [5, 9])
    with pytest.raises(ValueError, match="length_penalty"):
        engine.beam_search(prompts, 40, BeamOptions(beams=2, length_penalty=penalty), stop_token_ids=range(0, 8), ignore_eos=True)
    assert engine.cache.slots.held == 0
    found = engine.beam_search(prompts, 40, BeamOptions(beams=2, length_penalty=8.0), ignore_eos=True)
    assert all(np.isfinite(text.score) and text.score < 0 for texts in found for text in texts)


@pytest.mark.parametrize("penalty", [math.inf, math.nan, 1e300])
def test_choice_refuses_a_penalty_that_is_no_float32(penalty):
    case = Choice(1, 2, 2, 50, seed=0)
    case.run()
    with pytest.raises(ops().KernelError, match="length_penalty"):
        case.run(penalty=penalty)


@pytest.mark.parametrize("dtype,tolerance", [("float32", 2e-5), ("bfloat16", 2e-2)])
def test_short_chunks_over_the_whole_device(dtype, tolerance):
    """Steps of a few tokens each, keys cut over the device: the logits of the engine that walks them."""
    config, weights = model_case("a")
    config = {**config, "num_attention_heads": 2, "num_key_value_heads": 1, "head_dim": 64, "max_position_embeddings": 2048}
    weights = P.random_weights(config, 5, std=0.08)
    plain, cut = (make_engine(config, weights, dtype, max_tokens=8192, split_chunks=n) for n in (0, 8))
    prompts = prompts_for(config, [1500, 63, 5])
    outs = []
    for engine in (plain, cut):
        slots = engine.open(3)
        engine.step(slots, prompts)
        before = engine.steps_run
        a = host(engine.step(slots, [p[:n] for p, n in zip(prompts, (8, 1, 3))], [[0, 7], [0], [0, 1, 2]]))
        b = host(engine.step(slots, [p[:2] for p in prompts]))
        assert engine.steps_run == before + 2
        outs.append(np.concatenate([a, b]))
        assert (getattr(engine.last_batch, "shared", None) is not None) == (engine is cut)
    assert rel_error(outs[1], outs[0]) <= tolerance


def test_short_chunks_of_short_contexts_are_steps_like_any_other():
    """An engine that splits chunks runs a step below 768 positions as one that does not: from the launcher of all layers where
    there is one, to the same bits."""
    config, _ = model_case("a")
    config = {**config, "num_attention_heads": 4, "num_key_value_heads": 2, "head_dim": 64, "hidden_size": 128,
              "intermediate_size": 320, "max_position_embeddings": 1024}
    weights = P.random_weights(config, 5, std=0.05)
    prompts = prompts_for(config, [700] + [90] * 8)
    outs = []
    for n in (0, 8):
        engine = make_engine(config, weights, "bfloat16", max_tokens=8192, max_length=1024, split_chunks=n)
        launched, run = [], engine.model.native_layers.run
        engine.model.native_layers.run = lambda *a, launched=launched, run=run: (launched.append(1), run(*a))
        slots = engine.open(9)
        engine.step(slots, prompts)
        outs.append(host(engine.step(slots, [p[:8] for p in prompts])))   # 72 tokens on at most 708 positions
        assert len(launched) == 2 and getattr(engine.last_batch, "shared", None) is None
        engine.step(slots, [p[:60] for p in prompts])
        host(engine.step(slots, [p[:8] for p in prompts]))                # on 776
        assert len(launched) == (4 if n == 0 else 3) and (getattr(engine.last_batch, "shared", None) is not None) == (n > 0)
    assert np.array_equal(*outs)


def test_short_chunks_over_the_whole_device_wait_for_nothing():
    """What a step tells the attention over shared pages is made on the device, behind what is running there."""
    config, weights = model_case("a")
    config = {**config, "max_position_embeddings": 1024}
    engine = make_engine(config, P.random_weights(config, 5, std=0.05), "float32", max_tokens=8192, max_length=1024, split_chunks=4)
    slots = engine.open(3)
    engine.step(slots, prompts_for(config, [800, 70, 5]))
    engine.step(slots, [[1, 2, 3], [4], [5, 6, 7, 8]])
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        shared = engine._shared_rows(engine.last_batch)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert shared.slots.tolist() == [slots[0]] * 3 + [slots[1]] + [slots[2]] * 4 and shared.slots.dtype == torch.int32
    assert shared.shared.tolist() == [engine.cache.max_pages] * 3 and shared.max_rows == 4
    assert shared.groups.tolist() == [0, 3, 4, 8]


def test_the_command_line(tmp_path):
    from etalii.dllm_b200.weights.random_init import write_model

    config, weights = model_case("b")
    write_model(str(tmp_path), config, {k: torch.from_numpy(v).to(torch.bfloat16) for k, v in weights.items()})
    rounded = {k: torch.from_numpy(v).to(torch.bfloat16).float().numpy() for k, v in weights.items()}
    logits_of = PlainLogits(config, rounded)

    def run(*arguments):
        command = [sys.executable, os.path.join(ROOT, "bin", "dllm-b200"), "--model", str(tmp_path), "--dtype", "float32", "generate",
                   "--prompt-ids", "5,9,200,31", "--ignore-eos", *arguments]
        done = subprocess.run(command, capture_output=True, text=True, timeout=600)
        return done.returncode, done.stdout, done.stderr

    code, out, err = run("--max-tokens", "7", "--beams", "3", "--length-penalty", "0.5", "--stop-token-id", "40")
    assert code == 0
    want = PB.search(lambda text: logits_of(text)[-1], [5, 9, 200, 31], 3, 7, (40,), 0.5)
    assert [tuple(int(t) for t in line.split()) for line in out.splitlines()] == [t for t, _, _ in want]
    scores = [float(s) for s in re.findall(r"score: (-?[0-9.]+)  fingerprint: [0-9a-f]{64}  tokens: \d+  finish: (?:stop|length)", err)]
    assert len(scores) == 3 and all(abs(s - w) < 2e-3 for s, (_, w, _) in zip(scores, want))
    assert run("--beams", "3", "--temperature", "1")[0] == 2 and run("--beams", "40")[0] == 2
