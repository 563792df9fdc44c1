"""Beam search's bookkeeping (no GPU): options, plans, texts traced back through the histories, pages that sequences share,
the list of what beams move."""
import math

import numpy as np
import pytest
import torch

import plain_beams as PB
from etalii.dllm_b200.cache.allocators import CacheError
from etalii.dllm_b200.cache.beams import CacheRows
from etalii.dllm_b200.cache.paged import CacheNeed, PagedCache
from etalii.dllm_b200.engine.beam import BeamRun, beam_pages, plan_beam_batches
from etalii.dllm_b200.engine.generate import ContextLengthError
from etalii.dllm_b200.sampling.beams import BeamOptions


@pytest.mark.parametrize("wrong", [{"beams": 0}, {"beams": 33}, {"length_penalty": -0.1}, {"length_penalty": math.nan}])
def test_options_refuse(wrong):
    with pytest.raises(ValueError):
        BeamOptions(**wrong)


@pytest.mark.parametrize("penalty", [math.inf, -math.inf, 1e400])
def test_options_refuse_a_penalty_that_is_no_number(penalty):
    with pytest.raises(ValueError, match="finite"):
        BeamOptions(length_penalty=penalty)


@pytest.mark.parametrize("tokens,largest", [(1, 96.0), (2047, 96 / 11), (65535, 6.0)])
def test_options_refuse_a_penalty_that_leaves_no_score(tokens, largest):
    BeamOptions(length_penalty=largest * 0.999).check_length(tokens)
    for penalty in (largest * 1.001, 1e300):
        with pytest.raises(ValueError, match="2 \\*\\* 96"):
            BeamOptions(length_penalty=penalty).check_length(tokens)
    BeamOptions(length_penalty=1e300).check_length(0)
    # at the bound the least log probability that a token can have (1 - 2^-24 as a probability) is still a normal float32
    assert np.float32(2.0 ** -24) / np.float32(2.0 ** 96) >= np.finfo(np.float32).tiny


def test_options_defaults():
    assert (BeamOptions().beams, BeamOptions().length_penalty, BeamOptions().early_stopping) == (4, 1.0, False)


@pytest.mark.parametrize("length,new,beams,pages", [(1, 1, 4, 4), (63, 1, 4, 4), (64, 1, 4, 5), (63, 2, 4, 8), (130, 62, 3, 5),
                                                    (130, 63, 3, 8), (128, 64, 1, 3)])
def test_pages_of_a_search(length, new, beams, pages):
    assert beam_pages(length, new, beams, 64) == pages


def test_batches_fit_the_cache():
    # 5 pages each (1 + 4 x 1): pool of 11 holds two; slots for three; the last one alone
    assert plan_beam_batches([100, 100, 100], [20] * 3, 4, 64, 11, 12) == [[0, 1], [2]]
    assert plan_beam_batches([100, 100, 100], [20] * 3, 4, 64, 100, 9) == [[0, 1], [2]]
    assert plan_beam_batches([100, 100, 100], [20] * 3, 4, 64, 100, 100, max_batch=1) == [[0], [1], [2]]
    with pytest.raises(ContextLengthError, match="needs"):
        plan_beam_batches([100], [200], 4, 64, 11, 12)
    with pytest.raises(ContextLengthError, match="slots"):
        plan_beam_batches([100], [2], 4, 64, 11, 3)


def test_texts_are_traced_back_through_the_parents():
    run = BeamRun(5, 3)
    run.tokens = [[10, 11, 12], [20, 21, 22], np.array([30, 31, 32])]
    run.parents = [[0, 0, 0], [2, 1, 2], np.array([1, 0, 0])]
    assert run.text(3, 0) == (11, 21, 30) and run.text(3, 1) == (12, 20, 31) and run.text(3, 2) == (12, 20, 32)
    assert run.text(2, 2) == (12, 22) and run.text(0, 1) == ()
    results = run.results(BeamOptions(beams=3, length_penalty=2.0), [-9.0, -math.inf, -18.0], [-1.5, -math.inf, -math.inf],
                          [[2, 1], [-1, -1], [-1, -1]], False)
    assert [(r.tokens, r.score, r.finish_reason) for r in results] == [
        ((11, 21, 30), -1.0, "length"), ((11, 21), -1.5, "stop"), ((12, 20, 32), -2.0, "length")]
    over = run.results(BeamOptions(beams=3), [-9.0, -9.0, -9.0], [-1.5, -2.5, -math.inf], [[2, 1], [0, 0], [-1, -1]], True)
    assert [(r.tokens, r.finish_reason) for r in over] == [((11, 21), "stop"), ((), "stop")]


def _cache():
    needs = [CacheNeed("kv", 2, 16), CacheNeed("kv", 1, 32, window=100), None, CacheNeed("state", state_shape=(3, 4))]
    return PagedCache(needs, max_tokens=64 * 40, max_length=640, device=None)


@pytest.mark.parametrize("length,new", [(1, 1), (63, 1), (64, 1), (64, 64), (150, 100), (128, 300)])
def test_fork_shares_full_pages_and_nothing_else(length, new):
    cache = _cache()
    source, *others = cache.acquire(4)
    cache.reserve(source, length)
    cache.advance(source, length)
    cache.fork(source, others, new)
    full, end = length // 64, -(-(length + new) // 64)
    for group in cache._groups:
        rows = group.table_host[[source, *others], :end]
        assert (rows[:, :full] == rows[0, :full]).all()  # the prompt's full pages in common
        own = rows[:, full:].reshape(-1).tolist()
        assert len(set(own)) == len(own) and not set(own) & set(rows[0, :full].tolist())
        assert group.dirty >= set(others)
    assert all(cache.length(s) == length for s in others)
    cache.check()
    for slot in (source, *others):
        cache.advance(slot, new)
        cache.reserve(slot, 0)  # everything is there already
    cache.check()
    cache.release([source, *others])
    cache.check()
    assert cache.pages_held() == 0


def test_fork_refusals():
    cache = _cache()
    source, other, used = cache.acquire(3)
    for slot in (source, used):
        cache.reserve(slot, 70)
        cache.advance(slot, 70)
    with pytest.raises(CacheError, match="not a new"):
        cache.fork(source, [used], 10)
    with pytest.raises(CacheError, match="not in use"):
        cache.fork(30, [other], 10)
    with pytest.raises(CacheError, match="exceeds"):
        cache.fork(source, [other], 1000)
    more = cache.acquire(20)
    with pytest.raises(CacheError, match="out of pages"):
        cache.fork(source, [other, *more], 560)
    cache.check()
    cache.release([source, other, used, *more])
    assert cache.pages_held() == 0


def test_the_list_of_what_beams_move():
    storage = torch.zeros((2, 5, 3 * 64 * (16 + 8)), dtype=torch.bfloat16)  # two entries, values smaller than keys
    only = torch.zeros((1, 4, 1 * 64 * 40), dtype=torch.float32)
    table = torch.zeros((6, 7), dtype=torch.int32)
    state = torch.zeros((6, 5000), dtype=torch.float32)
    narrow = torch.zeros((6, 3), dtype=torch.float32)
    rows = CacheRows([(storage, table, 3, 16, 8), (only, table, 1, 40, 0)], [state, narrow], 64)
    pieces = rows.pieces.numpy()
    # 2 entries x 3 heads x 2 halves of keys and of values, a table; 1 x 1 x 2 of keys, a table; 20,000 bytes in three pieces; 12 in one
    assert rows.n_pieces == len(pieces) == 12 + 12 + 1 + 2 + 1 + 3 + 1
    kinds, sizes = pieces[:, 4] >> 32, pieces[:, 5] & 0xFFFFFFFF
    assert kinds.tolist() == [0] * 24 + [2, 0, 0, 2, 1, 1, 1, 1]
    assert sizes[:24].tolist() == [32] * 12 + [16] * 12 and sizes[25] == 160 and sizes[28:].tolist() == [8192, 8192, 3616, 12]
    assert pieces[14, 0] - storage.data_ptr() == 3 * 64 * 16 * 2 + 64 * 8 * 2  # values of head 1 of entry 0
    assert pieces[15, 0] - pieces[14, 0] == 32 * 8 * 2                          # and their other half
    assert pieces[18, 0] - pieces[12, 0] == storage[0].numel() * 2 and (pieces[:24, 1] == 3 * 64 * 24 * 2).all()
    first, count = pieces[:24, 6] & 0xFFFFFFFF, pieces[:24, 6] >> 32
    assert first.tolist() == [0, 32] * 12 and (count == 32).all()
    assert (pieces[-1, 5] >> 32) == 4 and (pieces[0, 5] >> 32) == 16


def test_the_list_refuses():
    storage, table = torch.zeros((1, 4, 64 * 40), dtype=torch.float32), torch.zeros((6, 7), dtype=torch.int32)
    with pytest.raises(CacheError, match="values"):
        CacheRows([(storage, table, 1, 40, 8)], [], 64)
    with pytest.raises(CacheError, match="int32"):
        CacheRows([(storage, table.long(), 1, 40, 0)], [], 64)
    with pytest.raises(CacheError, match="contiguous"):
        CacheRows([], [torch.zeros((3, 8))[:, ::2]], 64)
    with pytest.raises(CacheError, match="nothing"):
        CacheRows([], [], 64)
    with pytest.raises(CacheError, match="multiple of 4"):
        CacheRows([(torch.zeros((1, 2, 64 * 1), dtype=torch.bfloat16), table, 1, 1, 0)], [], 64)


@pytest.mark.parametrize("scratch,tickets,says", [(0x10008, 0x20000, "unsupported"), (0x10004, 0x20000, "unsupported"),
                                                  (0, 0x20000, "argument"), (0x10000, 0, "argument")])
@pytest.mark.parametrize("dtype,dim", [(0, 64), (1, 32), (1, 64)])
def test_attention_over_shared_pages_refuses_its_scratch(scratch, tickets, says, dtype, dim):
    """Two tokens on 9,000 positions, which several clusters share: the entry point looks at the scratch's address before it
    launches anything. (The addresses are nobody's.)"""
    from etalii.dllm_b200.kernels import ops

    assert ops._shared_shape(dtype, 4, 2, dim, 1, 2, 9002)[0] > 0
    call = ops._ATTENTION_SHARED.pack(*[0x1000 * (i + 1) for i in range(8)], scratch, tickets, 0x30000, 0, 200, 2, 141, 64, dtype, 4, 2, dim, 1,
                                      2, 9002, 0, 0.1)
    status = ops._fn("attention_shared", "dllm_attention_shared")(call, ops._ATTENTION_SHARED.size)
    assert says in ops._STATUS[status]


def test_choice_refuses_to_go_without_a_step_number():
    """A null address where the number of tokens so far is read. (The other addresses are nobody's: nothing is launched.)"""
    from etalii.dllm_b200.kernels import ops

    at = [0x1000 * (i + 1) for i in range(17)]
    call = ops._BEAM_SELECT.pack(at[0], 50, at[1], at[2], at[3], at[4], 0, 0, 0, *at[5:11], 0, at[11], at[12], 0, 0, 0, 1, 4, 4, 50, 0, 0, 1.0)
    assert ops._STATUS[ops._fn("beam_select", "dllm_beam_select")(call, ops._BEAM_SELECT.size)] == "bad argument"


def _step(tokens, context, groups=1, decode=True, shared=True):
    from types import SimpleNamespace

    from etalii.dllm_b200.engine.beam import SharedRows

    cuts = torch.zeros(groups + 1, dtype=torch.int32)
    batch = SimpleNamespace(is_decode=decode, n_tokens=tokens, max_context=context)
    if shared:
        batch.shared = SharedRows(None, cuts, None, tokens // groups)
    return batch


def _entry(kv_heads, dim, dtype, value_dim=0, keys_only=False, page=64):
    from etalii.dllm_b200.cache.paged import KvView

    return KvView(torch.zeros(1, dtype=dtype), torch.zeros((1, 4), dtype=torch.int32), page, kv_heads, dim, None, value_dim, keys_only)


@pytest.mark.parametrize("kv_heads,dim,dtype,tokens,groups,least", [
    (3, 64, torch.bfloat16, 64, 8, (128 << 20) / (64 * 768)), (3, 64, torch.bfloat16, 4, 1, (128 << 20) / (4 * 768)),
    (8, 128, torch.bfloat16, 64, 8, (64 << 20) / (64 * 4096)),   # (eight prompts of eight kv heads: a MB each)
    (8, 128, torch.bfloat16, 8, 1, (32 << 20) / (8 * 4096)), (32, 64, torch.bfloat16, 32, 8, (256 << 20) / (32 * 8192)),
    (3, 64, torch.float32, 64, 8, (64 << 20) / (64 * 1536)), (8, 128, torch.float32, 8, 1, (64 << 20) / (8 * 8192))])
def test_from_which_contexts_on_beams_read_shared_pages(kv_heads, dim, dtype, tokens, groups, least):
    """By the bytes of keys and values counted for every beam."""
    from etalii.dllm_b200.parts.attention import reads_shared_pages

    cache = _entry(kv_heads, dim, dtype)
    first = math.ceil(least)
    assert reads_shared_pages(_step(tokens, first, groups), cache) and not reads_shared_pages(_step(tokens, first - 1, groups), cache)
    assert not reads_shared_pages(_step(tokens, 1 << 30, groups, shared=False), cache)


def test_what_else_decides_whether_a_step_reads_shared_pages():
    from etalii.dllm_b200.parts.attention import reads_shared_pages

    for dtype in (torch.float32, torch.bfloat16):
        cache = _entry(2, 64, dtype)  # a few tokens appended: by the longest context
        assert reads_shared_pages(_step(2, 768, decode=False), cache) and not reads_shared_pages(_step(2, 767, decode=False), cache)
        for other in (_entry(2, 60, dtype), _entry(2, 264, dtype), _entry(2, 64, dtype, value_dim=32), _entry(2, 64, dtype, keys_only=True),
                      _entry(2, 64, dtype, page=32)):
            assert not reads_shared_pages(_step(64, 1 << 20, 8), other)
    assert not reads_shared_pages(_step(64, 1 << 20, 8), _entry(2, 64, torch.float16))
    # bfloat16 heads that the cluster kernel of single tokens does not take
    assert reads_shared_pages(_step(4, 10), _entry(2, 72, torch.bfloat16)) and not reads_shared_pages(_step(4, 10), _entry(2, 80, torch.bfloat16))


def test_plain_choice_by_hand():
    """Two beams, four tokens, token 3 ends a text: worked out on paper."""
    logits = np.log(np.array([[0.5, 0.3, 0.1, 0.1], [0.05, 0.05, 0.1, 0.8]]))
    places, pool, done = PB.select(logits, [math.log(0.5), math.log(0.4)], 2, {3}, [], 4, 0, 1.0, False)
    # totals: 0.32 (beam 1 ends), 0.25 (0, token 0), 0.15 (0, token 1): both go on from beam 0, the first stays in its place
    assert [(round(math.exp(s), 9), p, t) for s, p, t in places] == [(0.25, 0, 0), (0.15, 0, 1)]
    assert [(round(math.exp(s * 5), 9), w) for s, w in pool] == [(0.32, (4, 1))] and not done
    _, pool, done = PB.select(logits, [math.log(0.5), math.log(0.4)], 2, {3}, [(-0.1, (0, 0))], 4, 0, 1.0, True)
    assert [w for _, w in pool] == [(0, 0), (4, 1)] and done
    _, pool, _ = PB.select(logits, [math.log(0.5), math.log(0.4)], 2, {3}, [], 4, 5, 1.0, False)
    assert pool == []
