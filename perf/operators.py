"""Beam search's device work, as cases that can be timed and checked: the choice of the next beams, the reordering of what
the beams keep, and the attention of tokens that share cached pages.

  select:  logits [sequences x beams, vocabulary] and the beams' scores -> the next beams (whom each continues, with which
           token, at which score) and the pool of finished texts.
  reorder: every beam takes over the cache of the beam that it continues: page table, rows of the page that is being
           filled, fixed-size states. In place.
  attend:  attention of a few new tokens a group over the paged cache, where the group's tokens share pages: the beams of
           one prompt (common pages of the prompt, pages of their own behind them) or the tokens of a short chunk that
           is appended to one sequence (all pages in common, each token sees up to itself).

Sizes are those of the models that this repository's benchmark and tests run (`MODELS` in cases.py): 135M (30 layers, 9
heads on 3 of 64, vocabulary 49,152), 8B (32 layers, 32 heads on 8 of 128, vocabulary 128,256) and the recurrent layers of
width 2,048 (16 heads of 128 x 128)."""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
PAGE = 64  # positions a cache page holds
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases -------------------------------------------------------------------------------------------------------
def _select(name, n, beams_in, beams, vocab, stops=1, produced=3, min_tokens=0, penalty=1.0, early=False, allowed=1.0):
    return {"name": name, "op": "select", "n": n, "beams_in": beams_in, "beams": beams, "vocab": vocab, "stops": stops,
            "produced": produced, "min_tokens": min_tokens, "penalty": penalty, "early": early, "allowed": allowed}


def _reorder(name, n, beams, kept, length, layers, kv_heads, dim, dtype, states=0, state_heads=0, state_dim=0):
    return {"name": name, "op": "reorder", "n": n, "beams": beams, "kept": kept, "length": length, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "states": states, "state_heads": state_heads,
            "state_dim": state_dim}


def _attend(name, kind, n, rows, context, tail, heads, kv_heads, dim, dtype, window=0, idle=0):
    return {"name": name, "op": "attend", "kind": kind, "n": n, "rows": rows, "context": context, "tail": tail,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "window": window, "idle": idle}


def listed():
    return [
        # one person's request to the small model: nothing but latency
        _select("select_1x4_49k", 1, 4, 4, 49152),
        # the first choice of a batch: one row of logits a prompt, from which the beams start; no stop token yet
        _select("select_first_24x5_49k", 24, 1, 5, 49152, produced=0, min_tokens=1),
        # a step of a served batch over a large vocabulary, several stop tokens
        _select("select_8x8_128k", 8, 8, 8, 128256, stops=3, produced=40, penalty=0.8),
        # the widest search of an offline job, constrained to half the vocabulary
        _select("select_32x16_128k", 32, 16, 16, 128256, produced=200, penalty=0.6, early=True, allowed=0.5),
        # four beams of the small model, between two steps
        _reorder("reorder_135m_1x4", 1, 4, 2, 143, 30, 3, 64, "bfloat16"),
        # the same for a batch on the large model
        _reorder("reorder_8b_8x8", 8, 8, 3, 300, 32, 8, 128, "bfloat16"),
        # the 32-bit path, every beam moves (they change places in a ring)
        _reorder("reorder_135m_fp32_ring_3x5", 3, 5, 0, 125, 30, 3, 64, "float32"),
        # recurrent layers: matrices of a megabyte a layer and beam, beside a few layers of keys and values
        _reorder("reorder_states_4x4", 4, 4, 2, 97, 4, 4, 128, "bfloat16", 12, 16, 128),
        # four beams on a short prompt of the small model
        _attend("attend_beams_135m_1x4", "beams", 1, 4, 90, 21, 9, 3, 64, "bfloat16"),
        # a batch of eight prompts, eight beams each, a layer of the large model
        _attend("attend_beams_8b_8x8", "beams", 8, 8, 2000, 150, 32, 8, 128, "bfloat16"),
        # eight tokens appended to each of two long contexts
        _attend("attend_chunk_8b_2x8_40k", "chunk", 2, 8, 40000, 0, 32, 8, 128, "bfloat16"),
        # the 32-bit path, one beam of each prompt has ended
        _attend("attend_beams_135m_fp32_2x5", "beams", 2, 5, 700, 70, 9, 3, 64, "float32", idle=1),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    op = rng.choice(["select", "reorder", "attend"])
    if op == "select":
        beams = _log(rng, 1, 16)
        beams_in = rng.choice([1, beams, beams, beams])
        vocab = _log(rng, 400, 152000)
        n = _log(rng, 1, 48)
        while n > 1 and n * beams_in * vocab > 500 * 128000:
            n //= 2
        produced = rng.choice([0, 1, 7, 120, 900])
        case = _select("", n, beams_in, beams, vocab, rng.randint(0, 4), produced, rng.choice([0, 0, 5]),
                       rng.choice([0.0, 0.7, 1.0, 1.3]), rng.random() < 0.5, rng.choice([1.0, 1.0, 0.3, 0.02]))
    elif op == "reorder":
        beams, n, layers = _log(rng, 2, 16), _log(rng, 1, 12), _log(rng, 1, 32)
        kv_heads, dim = rng.choice([(3, 64), (8, 128), (32, 64), (4, 128), (2, 24), (1, 80)])
        while n > 1 and n * beams * layers * kv_heads * dim > 64 * 32 * 8 * 128:
            n //= 2
        while layers > 1 and n * beams * layers * kv_heads * dim > 64 * 32 * 8 * 128:
            layers //= 2
        length = _log(rng, 1, 700)
        states = rng.choice([0, 0, 1, 6]) if n * beams <= 24 else 0
        case = _reorder("", n, beams, rng.randint(0, beams - 1), length, layers, kv_heads, dim,
                        rng.choice(["bfloat16", "bfloat16", "float32"]), states, rng.choice([1, 5, 16]),
                        rng.choice([33, 64, 128]))
    else:
        kind = rng.choice(["beams", "chunk"])
        heads, kv_heads, dim = rng.choice([(9, 3, 64), (32, 8, 128), (32, 32, 64), (16, 4, 128), (8, 1, 80), (6, 2, 32)])
        rows, n = _log(rng, 1, 16), _log(rng, 1, 12)
        context = _log(rng, 1, 40000)
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        while n * rows * context * kv_heads * dim > 16 * 36000 * 1024 * (1 if dtype == "bfloat16" else 0.25) and context > 8:
            context = context * 3 // 5
        tail = 0 if kind == "chunk" else _log(rng, 1, 260)
        case = _attend("", kind, n, rows, context, tail, heads, kv_heads, dim, dtype, rng.choice([0, 0, 0, 100, 1000]),
                       rng.choice([0, 0, rows // 3]))
    del case["name"]
    return case


# ---- what a program has in hand before the call ------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 7919 + 17)
    return {"select": _prepare_select, "reorder": _prepare_reorder, "attend": _prepare_attend}[case["op"]](case, g)


def _uniform(g, shape, low=0.0, high=1.0):
    return torch.rand(shape, generator=g, device=DEVICE) * (high - low) + low


def _places(g, rows, count, among):
    """`count` different whole numbers below `among` in each of `rows` rows."""
    return _uniform(g, (rows, among)).argsort(dim=1)[:, :count]


def _prepare_select(case, g):
    n, kin, beams, vocab = case["n"], case["beams_in"], case["beams"], case["vocab"]
    logits = torch.randn((n * kin, vocab), generator=g, device=DEVICE) * 2.0
    # a few tokens of a row are likely, as after training; so are the stop tokens, now and then
    top = min(24, vocab)
    at = torch.randint(0, vocab, (n * kin, top), generator=g, device=DEVICE)
    logits.scatter_reduce_(1, at, _uniform(g, (n * kin, top), 5.0, 19.0), "amax")  # (a place drawn twice: the same in any order)
    stops = torch.arange(case["stops"], device=DEVICE, dtype=torch.int32) * 3 + 2
    logits[:, stops.long()] = _uniform(g, (n * kin, case["stops"]), 0.0, 19.0)
    if case["allowed"] < 1.0:  # what a grammar does not let through
        logits.masked_fill_(_uniform(g, logits.shape) >= case["allowed"], -math.inf)
    scores = torch.zeros((n, kin), device=DEVICE) if case["produced"] == 0 else -_uniform(g, (n, kin), 4.0, 14.0)
    if case["produced"] == 0 and kin > 1:
        scores[:, 1:] = -math.inf  # beams that are copies of the first
    have = torch.arange(beams, device=DEVICE)[None, :] < (torch.arange(n, device=DEVICE)[:, None] * 2 % (beams + 1))
    have &= torch.tensor(case["produced"] > 1, device=DEVICE)
    length = max(1.0, case["produced"] / 2) ** case["penalty"]
    finished = (-_uniform(g, (n, beams), 4.0, 16.0) / length).sort(dim=1, descending=True).values
    step = torch.randint(0, max(1, case["produced"]), (n, beams, 1), generator=g, device=DEVICE, dtype=torch.int32)
    who = torch.randint(0, kin, (n, beams, 1), generator=g, device=DEVICE, dtype=torch.int32)
    done = torch.zeros(n, dtype=torch.int32, device=DEVICE)
    done[7::8] = 1  # an eighth of a batch has ended
    return {"case": case, "logits": logits, "stops": stops, "scores": scores,
            "finished": torch.where(have, finished, -math.inf).contiguous(),
            "finished_at": torch.where(have[:, :, None], torch.cat([step, who], 2), -1).to(torch.int32).contiguous(),
            "done": done, "produced": torch.tensor([case["produced"]], dtype=torch.int32, device=DEVICE),
            "parents": torch.zeros((n, beams), dtype=torch.int32, device=DEVICE),
            "tokens": torch.zeros((n, beams), dtype=torch.int32, device=DEVICE),
            "out": (torch.zeros((n, beams), device=DEVICE), torch.zeros((n, beams), device=DEVICE),
                    torch.zeros((n, beams, 2), dtype=torch.int32, device=DEVICE),
                    torch.zeros(n, dtype=torch.int32, device=DEVICE))}


def _sources(case):
    """(beams of a sequence that others continue, beams that move): `kept` survivors stay in their places and share the other
    places out between them; with none kept the beams change places in a ring."""
    kept, beams = case["kept"], case["beams"]
    return (beams, beams) if kept == 0 else (min(kept, beams - kept), beams - kept)


def _prepare_reorder(case, g):
    n, beams, kept, length = case["n"], case["beams"], case["kept"], case["length"]
    order = _places(g, n, beams, beams)
    parents = torch.arange(beams, device=DEVICE).repeat(n, 1)
    if kept == 0:
        parents.scatter_(1, order, order.roll(1, dims=1))
    elif kept < beams:
        spread = torch.arange(beams - kept, device=DEVICE) % kept
        parents.scatter_(1, order[:, kept:], order[:, :kept][:, spread])
    full, last = length // PAGE, -(-(length + 1) // PAGE)  # pages that are full; pages with the one that is filled next
    slots = (torch.randperm(n * beams + 3, generator=g, device=DEVICE)[: n * beams]).to(torch.int32).view(n, beams)
    pages = n * beams * last + 5
    ids = torch.randperm(pages, generator=g, device=DEVICE)[: n * beams * last].to(torch.int32)
    table = torch.zeros((n * beams + 3, last + 2), dtype=torch.int32, device=DEVICE)
    table[slots.view(-1).long(), :last] = ids.view(n * beams, last)
    kind = TYPES[case["dtype"]]
    storage = torch.empty((case["layers"], pages, 2, case["kv_heads"], PAGE, case["dim"]), dtype=kind, device=DEVICE)
    for layer in storage:
        layer.copy_(torch.randn(layer.shape, generator=g, device=DEVICE, dtype=torch.bfloat16))
    shape = (n * beams + 3, case["state_heads"], case["state_dim"], case["state_dim"])
    states = [torch.randn(shape, generator=g, device=DEVICE) for _ in range(case["states"])]
    lengths = torch.full((n,), length, dtype=torch.int32, device=DEVICE)
    return {"case": case, "storage": storage, "table": table, "states": states, "slots": slots.contiguous(),
            "parents": parents.to(torch.int32).contiguous(), "lengths": lengths, "full": full}


def _groups(case):
    """For each group (first position of its new tokens or of its beams' own text, positions of its rows): the contexts of
    a batch differ, the chunks of three sequences in a row are of two lengths."""
    out = []
    for g in range(case["n"]):
        context = max(1, case["context"] - case["context"] * g // (2 * case["n"]))
        rows = case["rows"] if case["kind"] == "beams" else max(1, case["rows"] - (g % 3 == 2))
        live = rows - min(case["idle"], rows - 1)
        newest = [context + (case["tail"] - 1 if case["kind"] == "beams" else r) for r in range(live)]
        out.append((context, newest + [-1] * (rows - live)))
    return out


def _owner(beam, depth):
    """Whose page a beam reads `depth` pages before the one that it fills: of lines that go back to ever fewer beams."""
    return beam & ~((1 << min(depth, 10)) - 1)


def _prepare_attend(case, g):
    groups, beams = _groups(case), case["kind"] == "beams"
    kind = TYPES[case["dtype"]]
    table_rows, slots, positions, shared, cuts, used = [], [], [], [], [0], 0
    for context, newest in groups:
        last = max(newest) // PAGE + 1
        common = context // PAGE if beams else last
        prefix = list(range(used, used + common))
        used += common
        for r in range(len(newest) if beams else 1):
            own_pages = [used + j * len(newest) + _owner(r, last - 1 - j - common) for j in range(last - common)]
            table_rows.append(prefix + own_pages)
        used += (last - common) * len(newest)
        slots += range(len(table_rows) - len(newest), len(table_rows)) if beams else [len(table_rows) - 1] * len(newest)
        positions += newest
        shared.append(common)
        cuts.append(len(positions))
    width = max(len(row) for row in table_rows) + 2
    table = torch.zeros((len(table_rows), width), dtype=torch.int64)
    for i, row in enumerate(table_rows):
        table[i, : len(row)] = torch.tensor(row)
    pages = torch.randperm(used + 3, generator=g, device=DEVICE)
    table = pages[table.to(DEVICE)].to(torch.int32).contiguous()
    seat = torch.randperm(len(table_rows), generator=g, device=DEVICE)  # which row of the table a sequence has
    placed = torch.empty_like(table)
    placed[seat] = table
    storage = torch.empty((used + 3, 2, case["kv_heads"], PAGE, case["dim"]), dtype=kind, device=DEVICE)
    for part in storage.split(512):
        part.copy_(torch.randn(part.shape, generator=g, device=DEVICE, dtype=kind))
    q = torch.randn((len(positions), case["heads"] * case["dim"]), generator=g, device=DEVICE) * 1.5
    as_int = lambda values: torch.tensor(values, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return {"case": case, "q": q.to(kind), "storage": storage, "table": placed,
            "slots": seat[torch.tensor(slots, device=DEVICE)].to(torch.int32).contiguous(),
            "positions": as_int(positions), "groups": as_int(cuts), "shared": as_int(shared),
            "max_rows": max(len(p) for _, p in groups), "max_context": max(max(p) for _, p in groups) + 1,
            "scale": case["dim"] ** -0.5, "out": torch.empty((len(positions), case["heads"] * case["dim"]), dtype=kind, device=DEVICE)}


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"select": _own_select, "reorder": _own_reorder, "attend": _own_attend}[op](state)
    return {"select": _plain_select, "reorder": _plain_reorder, "attend": _plain_attend}[op](state)


def _own_select(s):
    from etalii.dllm_b200.kernels import ops

    case = s["case"]
    if "scratch" not in s:  # the work buffers that a program keeps for all its steps
        s["scratch"] = torch.empty(ops.beam_select_scratch(case["n"], case["beams_in"], case["vocab"], case["beams"]), device=DEVICE)
        s["tickets"] = torch.zeros(case["n"], dtype=torch.int32, device=DEVICE)
    ops.beam_select(s["parents"], s["tokens"], s["out"], s["logits"], (s["scores"], s["finished"], s["finished_at"], s["done"]),
                    s["produced"], s["scratch"], s["tickets"], stop_ids=s["stops"], min_tokens=case["min_tokens"],
                    length_penalty=case["penalty"], early=case["early"])
    scores, finished, finished_at, done = s["out"]
    return {"parents": s["parents"], "tokens": s["tokens"], "scores": scores, "finished": finished, "finished_at": finished_at,
            "done": done}


def _own_reorder(s):
    from etalii.dllm_b200.kernels import ops

    if "rows" not in s:  # the list of what a beam keeps, made once for a cache
        from etalii.dllm_b200.cache.beams import CacheRows

        case = s["case"]
        s["rows"] = CacheRows([(s["storage"], s["table"], case["kv_heads"], case["dim"], case["dim"])], s["states"], PAGE)
    ops.beam_reorder(s["rows"], s["slots"], s["parents"], s["lengths"])
    return {"storage": s["storage"], "table": s["table"], "states": s["states"]}


def _own_attend(s):
    from etalii.dllm_b200.kernels import ops

    case = s["case"]
    if "view" not in s:  # the view of the cache and the work buffers that a program keeps
        from etalii.dllm_b200.cache.paged import KvView

        s["view"] = KvView(s["storage"], s["table"], PAGE, case["kv_heads"], case["dim"], case["window"] or None)
        floats, tickets = ops.attention_shared_scratch(s["view"], case["heads"], case["n"], s["max_rows"], s["max_context"])
        s["scratch"] = torch.empty(floats, device=DEVICE)
        s["tickets"] = torch.zeros(tickets, dtype=torch.int32, device=DEVICE)
    ops.attention_shared(s["out"], s["q"], s["view"], case["heads"], s["scale"], case["window"], s["slots"], s["positions"],
                         s["groups"], s["shared"], s["max_rows"], s["max_context"], s["scratch"], s["tickets"])
    return {"out": s["out"]}


def _key(value, index):
    """An int64 that orders by value (float32, descending means larger) and then by the lower index."""
    bits = (value + 0.0).view(torch.int32)
    ordered = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
    return ordered * (1 << 32) + ((1 << 32) - 1 - index)


def _before(a, b):
    """Which candidates (total, beam, logit, token) come before which: a larger total; of equal ones the lower beam's, and of
    one beam's that with the larger logit, then the lower token. [n, count of b, count of a]."""
    (t, k, x, v), (u, l, y, w) = [[part[:, None, :] for part in a], [part[:, :, None] for part in b]]
    return (t > u) | ((t == u) & ((k < l) | ((k == l) & ((x > y) | ((x == y) & (v < w))))))


def _plain_select(s):
    case = s["case"]
    n, kin, beams, vocab = case["n"], case["beams_in"], case["beams"], case["vocab"]
    x, scores, stops = s["logits"].view(n, kin, vocab), s["scores"], s["stops"].long()
    largest = x.amax(dim=2, keepdim=True)
    log_sum = largest + torch.log(torch.exp(x - largest).sum(dim=2, keepdim=True))
    total_of = lambda logit, row: (logit - log_sum[:, :, 0].gather(1, row)) + scores.gather(1, row)  # noqa: E731
    valid = lambda total: torch.where(total > -math.inf, total, -math.inf)  # noqa: E731  (no likelihood: no candidate)
    # each row's best tokens that do not end the text, then the best of a sequence's rows
    on = x.clone()
    on[:, :, stops] = -math.inf
    width = min(beams, vocab)
    token = _key(on, torch.arange(vocab, device=DEVICE)).topk(width, dim=2).indices
    logit = on.gather(2, token).view(n, kin * width)
    token = token.view(n, kin * width)
    parent = torch.arange(kin, device=DEVICE).repeat_interleave(width)[None, :].expand(n, kin * width)
    live = valid(total_of(logit, parent))
    best = _key(live, torch.arange(kin * width, device=DEVICE)).topk(min(beams, kin * width), dim=1).indices
    fill = torch.zeros((n, beams - best.shape[1]), dtype=torch.int64, device=DEVICE)
    live, parent, token, logit = (torch.cat([t.gather(1, best), (fill - math.inf if t.is_floating_point() else fill).to(t.dtype)], 1)
                                  for t in (live, parent, token, logit))
    is_live = live > -math.inf
    candidates = (live, parent, logit, token)
    # who continues whom: the best continuation of a beam stays in the beam's place, the others take the free places in order
    order = torch.arange(beams, device=DEVICE)
    earlier = order[None, :, None] > order[None, None, :]
    repeated = ((parent[:, :, None] == parent[:, None, :]) & earlier & is_live[:, None, :]).any(dim=2)
    stays = is_live & ~repeated & (parent < beams)
    taken = ((parent[:, :, None] == order[None, None, :]) & stays[:, :, None]).any(dim=1)
    free_first = torch.argsort(taken.to(torch.int32) * beams + order[None, :], dim=1)  # free places ascending, then the others
    place = torch.where(stays, parent, free_first.gather(1, ((~stays).cumsum(dim=1) - 1).clamp(min=0)))
    idle = torch.clamp(order, max=kin - 1)[None, :].expand(n, beams)  # a place without a beam keeps to itself
    here = torch.empty_like(place).scatter_(1, place, order[None, :].expand(n, beams))
    next_live, parent, token, is_live = (t.gather(1, here) for t in (live, parent, token, is_live))
    parent, token = torch.where(is_live, parent, idle), torch.where(is_live, token, 0)
    # texts that end here: stop tokens among the first `beams` of all candidates
    length = float(case["produced"] + 1) ** case["penalty"]
    finished, finished_at = s["finished"], s["finished_at"]
    if len(stops) and case["produced"] >= case["min_tokens"]:
        stop_parent = torch.arange(kin, device=DEVICE).repeat_interleave(len(stops))[None, :].expand(n, kin * len(stops))
        stop_logit = x[:, :, stops].reshape(n, kin * len(stops))
        stop_total = valid(total_of(stop_logit, stop_parent))
        ending = (stop_total, stop_parent, stop_logit, stops.repeat(kin)[None, :].expand(n, kin * len(stops)))
        before = _before(ending, ending).sum(dim=2)
        ended = torch.where((before + _before(candidates, ending).sum(dim=2) < beams) & (stop_total > -math.inf),
                            stop_total / length, -math.inf)
        by_rank = before.argsort(dim=1)
        ended, at = ended.gather(1, by_rank), stop_parent.gather(1, by_rank)
        at = torch.stack([torch.full_like(at, case["produced"]), at], 2).to(torch.int32)
        at = torch.where((ended > -math.inf)[:, :, None], at, -1)
        pool, by_score = torch.cat([finished, ended], 1).sort(dim=1, descending=True, stable=True)
        finished = pool[:, :beams].contiguous()
        finished_at = torch.cat([finished_at, at], 1).gather(1, by_score[:, :beams, None].expand(n, beams, 2))
    worst, best = finished[:, -1], next_live.amax(dim=1)
    over = (worst > -math.inf) & ((worst >= best / length) | case["early"]) | (best == -math.inf)
    was = s["done"] > 0
    w = was[:, None]
    return {"parents": torch.where(w, idle, parent).to(torch.int32), "tokens": torch.where(w, 0, token).to(torch.int32),
            "scores": torch.where(w, -math.inf, next_live), "finished": torch.where(w, s["finished"], finished),
            "finished_at": torch.where(w[:, :, None], s["finished_at"], finished_at), "done": (was | over).to(torch.int32)}


def _plain_reorder(s):
    case, table, storage = s["case"], s["table"], s["storage"]
    n, beams, full, rows = case["n"], case["beams"], s["full"], case["length"] % PAGE
    slots = s["slots"].long()
    source = slots.gather(1, s["parents"].long()).view(-1)
    slots = slots.view(-1)
    before = table[source]
    if rows:
        there, here = before[:, full].long(), table[slots, full].long()
        storage[:, here, :, :, :rows] = storage[:, there, :, :, :rows]
    table[slots, :full] = before[:, :full]
    for held in s["states"]:
        held[slots] = held[source]
    return {"storage": storage, "table": table, "states": s["states"]}


def _plain_attend(s):
    case, q = s["case"], s["q"]
    tokens, heads, kv_heads, dim = q.shape[0], case["heads"], case["kv_heads"], case["dim"]
    pages = -(-s["max_context"] // PAGE)
    index = s["table"][s["slots"].long(), :pages].long()
    wide = lambda which: s["storage"][index, which].float().permute(0, 2, 1, 3, 4).reshape(tokens, kv_heads, pages * PAGE, dim)  # noqa: E731
    score = torch.matmul(q.float().view(tokens, kv_heads, heads // kv_heads, dim), wide(0).transpose(2, 3)) * s["scale"]
    at, position = torch.arange(pages * PAGE, device=DEVICE), s["positions"][:, None]
    sees = at[None, :] <= position
    if case["window"]:
        sees &= at[None, :] > position - case["window"]
    score = torch.where(sees[:, None, None, :], score, -math.inf)
    largest = score.amax(dim=3, keepdim=True)
    weight = torch.exp(score - torch.where(largest > -math.inf, largest, 0.0))
    total = weight.sum(dim=3, keepdim=True)
    out = torch.matmul(weight, wide(1)) / torch.where(total > 0, total, 1.0)  # (a token that sees nothing: zeros)
    return {"out": out.reshape(tokens, heads * dim).to(q.dtype)}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "select":
        running = case["n"] - (case["n"] // 8)
        live = 1 if case["produced"] == 0 else case["beams_in"]
        values = running * live * case["vocab"]
        return {"bytes": 4 * values + case["n"] * case["beams"] * 40, "flops": 4 * values}
    if case["op"] == "reorder":
        sources, moved = _sources(case)
        size = {"bfloat16": 2, "float32": 4}[case["dtype"]]
        beam = case["layers"] * 2 * case["kv_heads"] * case["dim"] * size * (case["length"] % PAGE) \
            + case["states"] * case["state_heads"] * case["state_dim"] ** 2 * 4 + 4 * (case["length"] // PAGE)
        return {"bytes": case["n"] * beam * (sources + moved) + case["n"] * case["beams"] * 8, "flops": 0}
    size = {"bfloat16": 2, "float32": 4}[case["dtype"]]
    window, keys, seen, tokens = case["window"] or 1 << 40, 0, 0, 0
    for context, newest in _groups(case):
        end, live = max(newest) + 1, [p for p in newest if p >= 0]
        first = max(0, min(live) + 1 - window)
        tokens += len(newest)
        seen += sum(min(p + 1, window) for p in live)
        common = context // PAGE * PAGE if case["kind"] == "beams" else end
        keys += max(0, common - first)
        if case["kind"] == "beams":
            last = (end - 1) // PAGE
            for page in range(common // PAGE, last + 1):
                owners = len({_owner(r, last - page) for r in range(len(live))})
                keys += owners * max(0, min(end, (page + 1) * PAGE) - max(first, page * PAGE))
    width = case["heads"] * case["dim"]
    return {"bytes": keys * 2 * case["kv_heads"] * case["dim"] * size + 2 * tokens * width * size, "flops": 4 * seen * width}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"select": _exact_select, "reorder": _exact_reorder, "attend": _exact_attend}[case["op"]](case, s)


def _exact_select(case, s):
    n, kin, beams, vocab = case["n"], case["beams_in"], case["beams"], case["vocab"]
    stops = set(s["stops"].tolist())
    length = float(case["produced"] + 1) ** case["penalty"]
    scores_out = np.full((n, beams), -math.inf)
    pool_out = s["finished"].double().cpu().numpy().copy()
    done = s["done"].tolist()
    for b in range(n):
        if done[b]:
            continue
        rows = s["logits"][b * kin:(b + 1) * kin].double()
        likely = torch.log_softmax(rows, dim=1) + s["scores"][b].double()[:, None]
        likely = torch.where(likely > -math.inf, likely, -math.inf).reshape(-1)
        count = min(likely.numel(), beams * (1 + len(stops)) + kin * len(stops))
        best = likely.topk(count)
        chosen, ended = [], []
        for rank, (value, at) in enumerate(sorted(zip(best.values.tolist(), best.indices.tolist()), key=lambda c: (-c[0], c[1]))):
            if value == -math.inf:
                break
            if at % vocab in stops:
                if rank < beams:
                    ended.append(value / length)
            elif len(chosen) < beams:
                chosen.append((value, at // vocab))
        places = [None] * beams
        others = []
        for value, parent in chosen:
            if parent < beams and places[parent] is None:
                places[parent] = value
            else:
                others.append(value)
        for value in others:
            places[places.index(None)] = value
        scores_out[b] = [-math.inf if value is None else value for value in places]
        if case["produced"] >= case["min_tokens"]:
            pool_out[b] = sorted(list(pool_out[b]) + ended, reverse=True)[:beams]
    return {"parents": None, "tokens": None, "scores": scores_out, "finished": pool_out, "finished_at": None, "done": None}


def _exact_reorder(case, s):
    """(Moving values computes nothing: what comes out are the inputs' own values, element for element.)"""
    return None


def _exact_attend(case, s):
    q, heads, kv_heads, dim = s["q"].double(), case["heads"], case["kv_heads"], case["dim"]
    group = heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
    for t, (slot, position) in enumerate(zip(s["slots"].tolist(), s["positions"].tolist())):
        if position < 0:
            continue
        first = max(0, position + 1 - case["window"]) if case["window"] else 0
        at = torch.arange(first, position + 1, device=DEVICE)
        page, row = s["table"][slot, at // PAGE].long(), at % PAGE
        keys, values = s["storage"][page, 0, :, row].double(), s["storage"][page, 1, :, row].double()
        for h in range(heads):
            weight = torch.softmax(keys[:, h // group] @ q[t, h * dim:(h + 1) * dim] * s["scale"], dim=0)
            out[t, h * dim:(h + 1) * dim] = weight @ values[:, h // group]
    return {"out": out}
