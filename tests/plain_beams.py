"""Beam search in plain Python and numpy, in 64 bits: the choice of the next beams, what beams take over from one another,
attention of tokens over pages, and the whole search above a function that gives a text's logits. Shares no code with the
library."""
import math

import numpy as np


def log_probabilities(logits):
    """Rows of log probabilities; a row that holds a NaN or +inf, or nothing above -inf, has none."""
    x = np.asarray(logits, dtype=np.float64)
    out = np.full(x.shape, -math.inf)
    for i, row in enumerate(x):
        if np.isnan(row).any() or (row == math.inf).any() or not (row > -math.inf).any():
            continue
        top = row.max()
        out[i] = row - (top + math.log(np.exp(row - top).sum()))
    return out


def candidates(logits, scores):
    """All (total, beam, logit, token) of a sequence, in the order of the choice."""
    x = np.asarray(logits, dtype=np.float64)
    likely = log_probabilities(x)
    out = [(likely[k, t] + scores[k], k, x[k, t], t) for k in range(x.shape[0]) for t in range(x.shape[1])
           if scores[k] > -math.inf and likely[k, t] > -math.inf]
    out.sort(key=lambda c: (-c[0], c[1], -c[2], c[3]))
    return out


def select(logits, scores, beams, stops, pool, produced, min_tokens, penalty, early):
    """One sequence's choice. pool: [(score, (step, beam))], best first, at most `beams`. Returns (places: [(score, parent,
    token)], pool, done)."""
    rows = len(scores)
    chosen, ended = [], []
    length = float(produced + 1) ** penalty
    for rank, (total, beam, _, token) in enumerate(candidates(logits, scores)):
        if token in stops:
            if rank < beams and produced >= min_tokens:
                ended.append((total / length, (produced, beam)))
        elif len(chosen) < beams:
            chosen.append((total, beam, token))
        if rank >= beams and len(chosen) == beams:
            break
    if produced < min_tokens:  # (stop tokens count for nothing: not in the ranks either)
        ended = []
    places = [None] * beams
    rest = []
    for one in chosen:
        if one[1] < beams and places[one[1]] is None:
            places[one[1]] = one
        else:
            rest.append(one)
    for one in rest:
        places[places.index(None)] = one
    best = max((p[0] for p in places if p is not None), default=-math.inf)
    places = [(-math.inf, min(i, rows - 1), 0) if p is None else p for i, p in enumerate(places)]
    merged = sorted(list(pool) + ended, key=lambda entry: -entry[0])[:beams]  # (stable: those that were there first)
    full = len(merged) == beams
    done = best == -math.inf or (full and (early or merged[-1][0] >= best / length))
    return places, merged, done


def search(logits_of, prompt, beams, new_tokens, stops=(), penalty=1.0, early=False, min_tokens=0):
    """The best texts behind `prompt`: [(tokens, score, "stop" | "length")], best first. logits_of(text) -> the logits behind it."""
    texts, scores, pool = [()], [0.0], []
    for step in range(new_tokens):
        rows = np.stack([np.asarray(logits_of(list(prompt) + list(text)), dtype=np.float64) if score > -math.inf
                         else np.zeros_like(rows[0]) if step else None for text, score in zip(texts, scores)])
        places, merged, done = select(rows, scores, beams, set(stops), [(s, w) for s, w, _ in pool], step, min_tokens, penalty,
                                      early)
        known = {w: t for _, w, t in pool}
        pool = [(s, w, known[w] if w in known else texts[w[1]]) for s, w in merged]
        texts = [texts[parent] + (token,) for _, parent, token in places]
        scores = [score for score, _, _ in places]
        if done:
            break
    out = [(text, score, "stop") for score, _, text in pool]
    if not done:
        divisor = max(1, len(texts[0])) ** penalty
        out += [(text, score / divisor, "length") for text, score in zip(texts, scores) if score > -math.inf]
    out.sort(key=lambda entry: -entry[1])
    return out[:beams]


def attend(q, storage, table, slots, positions, heads, kv_heads, scale, window=0, page=64):
    """q [tokens, heads * dim]; storage [pages, 2, kv_heads, page, dim]. A token at -1: zeros."""
    q, storage = np.asarray(q, np.float64), np.asarray(storage, np.float64)
    dim = storage.shape[-1]
    out = np.zeros_like(q)
    for t, (slot, position) in enumerate(zip(slots, positions)):
        if position < 0:
            continue
        at = np.arange(max(0, position + 1 - window) if window else 0, position + 1)
        pages, rows = np.asarray(table)[slot, at // page], at % page
        for h in range(heads):
            g = h // (heads // kv_heads)
            keys, values = storage[pages, 0, g, rows], storage[pages, 1, g, rows]
            with np.errstate(invalid="ignore", over="ignore"):
                s = keys @ q[t, h * dim:(h + 1) * dim] * scale
                w = np.exp(s - s.max())
                out[t, h * dim:(h + 1) * dim] = (w[:, None] * values).sum(0) / w.sum()
    return out
