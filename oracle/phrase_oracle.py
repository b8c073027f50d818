"""Plain restatements, in 64 bits on the CPU, of the phrase operators (include/tonehip.h: tone_frames_*, tone_token_scores,
tone_ctc_align): numpy only, one request / row / sequence at a time, straight from the definitions."""

from __future__ import annotations

import itertools

import numpy as np


def plan(table, queue, cursors, rows_in, rows_out, first, length, keep, add, page, max_add):
    """Returns (table, queue, cursors, slots) after the requests; the caller gives valid ones."""
    before, table, queue = np.array(table), np.array(table), np.array(queue)
    head, tail = (int(c) for c in cursors)
    free = [int(queue[i % len(queue)]) for i in range(head, tail)]
    slots = np.full((len(first), max_add), -1, np.int64)
    released = []
    taken = 0
    for b in range(len(first)):
        held = {}
        for f in range(first[b], length[b]):
            held[f // page] = int(before[rows_in[b], f // page - first[b] // page])
        kept, end = max(first[b], keep[b]), length[b] + add[b]
        wanted = sorted({f // page for f in range(kept, end)})
        released += [held[p] for p in sorted(held) if p not in wanted]
        for p in wanted:
            if p not in held:
                held[p] = free[taken]
                taken += 1
        table[rows_out[b]] = -1
        for j, p in enumerate(wanted):
            table[rows_out[b], j] = held[p]
        for f in range(length[b], end):
            if f >= kept:
                slots[b, f - length[b]] = held[f // page] * page + f % page
    for i, p in enumerate(released):
        queue[(tail + i) % len(queue)] = p
    return table, queue, np.array([head + taken, tail + len(released)]), slots


def slots(table, rows, first, begin, count, page, n_pages, max_count):
    out = np.full((len(rows), max_count), -1, np.int64)
    for b in range(len(rows)):
        for j in range(min(count[b], max_count)):
            f = begin[b] + j
            at = f // page - first[b] // page
            if 0 <= rows[b] < table.shape[0] and first[b] >= 0 and f >= first[b] and at < table.shape[1] \
                    and 0 <= table[rows[b], at] < n_pages:
                out[b, j] = int(table[rows[b], at]) * page + f % page
    return out


def scores(row, token, k):
    """One row (float64): (logprob, rank, entropy, [(id, logprob)] * k, mean |z|) with z = row - max under the softmax."""
    v = row.size
    order = sorted(range(v), key=lambda i: (-row[i], i))
    high = row.max()
    if high == -np.inf:
        lp, entropy, mean = np.full(v, -np.inf), 0.0, 0.0
    else:
        z = row - high
        e = np.exp(z)
        s = e.sum()
        lp = z - np.log(s)
        p = e / s
        some = p > 0
        entropy, mean = float(-(p[some] * lp[some]).sum()), float(-(p[some] * z[some]).sum())
    given = 0 <= token < v
    return (lp[token] if given else 0.0, order.index(token) if given else -1, entropy, [(i, lp[i]) for i in order[:k]], mean)


def align(frames, tokens, blank):
    """frames (F, V) float64, tokens a list: (score, total, labels, spans), None for the last two where no path fits."""
    f, vocab = frames.shape
    lab = [blank]
    for t in tokens:
        lab += [t, blank]
    n = len(lab)

    def emit(t, s):
        if not 0 <= lab[s] < vocab or (s % 2 and lab[s] == blank):
            return -np.inf
        return frames[t, lab[s]] if abs(frames[t, lab[s]]) < 6e4 else -np.inf      # (NaN compares false)

    if f == 0:
        ok = not tokens
        return (0.0, 0.0, [], []) if ok else (-np.inf, -np.inf, None, None)
    best = np.full((f, n), -np.inf)
    total = np.full((f, n), -np.inf)
    came = np.zeros((f, n), int)
    for t in range(f):
        for s in range(n):
            if t == 0:
                prev, sums = [0.0 if s < 2 else -np.inf], [0.0 if s < 2 else -np.inf]
            else:
                steps = [s - d for d in range(3) if s >= d and (d < 2 or (s % 2 and s > 1 and lab[s] != lab[s - 2]))]
                prev, sums = [best[t - 1, i] for i in steps], [total[t - 1, i] for i in steps]
            j = int(np.argmax(prev))            # the first of equals
            came[t, s] = j
            best[t, s] = prev[j] + emit(t, s)
            h = max(sums)
            total[t, s] = h if h == -np.inf else h + np.log(sum(np.exp(v - h) for v in sums)) + emit(t, s)
    ends = [n - 1] + ([n - 2] if n > 1 else [])
    score = max(best[f - 1, s] for s in ends)
    h = max(total[f - 1, s] for s in ends)
    tot = h if h == -np.inf else h + np.log(sum(np.exp(total[f - 1, s] - h) for s in ends))
    if score == -np.inf:
        return score, tot, None, None
    s = n - 1 if best[f - 1, n - 1] == score else n - 2
    labels, spans = [0] * f, [[-1, -1] for _ in tokens]
    for t in range(f - 1, -1, -1):
        labels[t] = lab[s]
        if s % 2:
            spans[s // 2][0] = t
            spans[s // 2][1] = max(spans[s // 2][1], t + 1)
        s -= came[t, s]
    return score, tot, labels, spans


def align_by_paths(frames, tokens, blank):
    """(score, total) from every label sequence of the frames' length that reads as ``tokens`` (tiny cases only)."""
    f, vocab = frames.shape
    scores_ = []
    for path in itertools.product(range(vocab), repeat=f):
        said = [c for i, c in enumerate(path) if c != blank and (i == 0 or path[i - 1] != c)]
        if said == list(tokens):
            scores_.append(sum(frames[t, c] for t, c in enumerate(path)))
    if not scores_:
        return -np.inf, -np.inf
    h = max(scores_)
    return h, h if h == -np.inf else h + np.log(np.exp(np.array(scores_) - h).sum())
