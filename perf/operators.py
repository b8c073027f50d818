"""What a server does with the frames of a phrase once the model has answered, as measured cases.

A streaming CTC model answers with a row of log probabilities per 30 ms frame.  A server that wants more than the greedy
text (confidences, alternatives, word times, the score of a given transcript) has to hold those rows until the phrase
ends, in pages of a shared pool, and then ask what they say about given tokens.  Four operators:

  paging   page tables and slot maps built on the GPU from the streams' frame counts (``frames_plan`` for the frames a
           step appends, ``frames_slots`` for the frames a phrase reads back)
  put      the rows of a step written through such a slot map (``frames_put``)
  scores   the log probability of a given token per row, its rank, the row's entropy and its top alternatives
           (``token_scores``), over dense rows or rows of the pool
  align    the best CTC path of given token sequences, each token's frames, and the sequences' total log probability
           (``ctc_align``)
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
BLANK = 34          # the blank of the 35-token head; wider vocabularies here keep it


def listed():
    return [
        # one step of a full card: 4096 streams append the 10 frames of a 300 ms chunk, finished phrases leave
        {"name": "plan-step", "op": "plan", "streams": 4096, "page": 64, "window": 2064, "add": 10, "ragged": False},
        # a few recordings imported at once: thousands of new frames each, page size not a power of two
        {"name": "plan-import", "op": "plan", "streams": 96, "page": 48, "window": 20000, "add": 18000, "ragged": True},
        # one phrase read back: the smallest call of the set
        {"name": "slots-phrase", "op": "slots", "streams": 1, "page": 64, "window": 2064, "count": 187},
        # the rows of a 4096-stream step put into their pages
        {"name": "put-step", "op": "put", "streams": 4096, "add": 10, "vocab": 35, "src": "fp32", "pool": "fp32"},
        # the rows of imported recordings, held in half the bytes
        {"name": "put-import", "op": "put", "streams": 96, "add": 18000, "vocab": 35, "src": "fp32", "pool": "fp16"},
        # the frames of one phrase, read from the pool: confidences and five alternatives
        {"name": "scores-phrase", "op": "scores", "rows": 187, "vocab": 35, "dtype": "fp32", "k": 5, "paged": True,
         "pad": 0, "masked": False},
        # every frame of a 4096-stream step, with the alternatives a host beam search keeps
        {"name": "scores-step", "op": "scores", "rows": 40960, "vocab": 35, "dtype": "fp32", "k": 8, "paged": False,
         "pad": 0, "masked": False},
        # one row over a wide vocabulary: a decoder's next token
        {"name": "scores-token", "op": "scores", "rows": 1, "vocab": 65536, "dtype": "bf16", "k": 20, "paged": False,
         "pad": 0, "masked": True},
        # a batch of texts over a wide, odd vocabulary
        {"name": "scores-wide", "op": "scores", "rows": 2048, "vocab": 65537, "dtype": "bf16", "k": 10, "paged": False,
         "pad": 0, "masked": True},
        # one finished phrase of a few seconds
        {"name": "align-phrase", "op": "align", "seqs": 1, "frames": 187, "tokens": 43, "vocab": 35, "dtype": "fp32",
         "paged": True, "total": False, "share": 1},
        # eight hypotheses for each of 24 phrases, scored on the same frames
        {"name": "align-nbest", "op": "align", "seqs": 192, "frames": 400, "tokens": 110, "vocab": 35, "dtype": "fp16",
         "paged": True, "total": True, "share": 8},
        # the longest phrases a splitter lets through (2000 frames, a minute of speech), many streams at once
        {"name": "align-long", "op": "align", "seqs": 48, "frames": 2000, "tokens": 700, "vocab": 35, "dtype": "fp32",
         "paged": False, "total": True, "share": 1},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "slots", "put", "scores", "scores", "scores", "align", "align"])
    if op == "plan":
        page = rng.choice([1, 7, 16, 32, 48, 64, 100])
        streams = _log(rng, 1, 4096)
        add = _log(rng, 1, max(1, min(18000, 1600000 // streams)))
        window = page * _log(rng, 2, max(2, min(400, 800000 // streams))) + add
        return {"op": op, "streams": streams, "page": page, "window": window, "add": add, "ragged": rng.random() < 0.5}
    if op == "slots":
        streams = _log(rng, 1, 2048)
        count = _log(rng, 1, max(1, min(20000, 1600000 // streams)))
        return {"op": op, "streams": streams, "page": rng.choice([1, 7, 16, 32, 48, 64, 100]), "window": count + _log(rng, 1, 500),
                "count": count}
    if op == "put":
        streams, vocab = _log(rng, 1, 4096), _log(rng, 2, 1024)
        return {"op": op, "streams": streams, "add": _log(rng, 1, max(1, min(18000, 60000000 // (streams * vocab)))),
                "vocab": vocab, "src": rng.choice(sorted(DTYPES)), "pool": rng.choice(sorted(DTYPES))}
    if op == "scores":
        vocab = rng.choice([35, _log(rng, 2, 64), _log(rng, 65, 2048), _log(rng, 2049, 131072)])
        return {"op": op, "rows": _log(rng, 1, max(1, min(60000, 130000000 // vocab))), "vocab": vocab, "dtype": rng.choice(sorted(DTYPES)),
                "k": min(vocab, rng.choice([0, 1, 4, 5, 8, 10, 16, 20, 32, 64])), "paged": rng.random() < 0.4,
                "pad": rng.choice([0, 0, 1, 5, 8]), "masked": rng.random() < 0.5}
    frames = _log(rng, 1, 2000)
    tokens = _log(rng, 1, max(1, frames // 2))
    share = rng.choice([1, 1, 4, 8])
    seqs = share * _log(rng, 1, max(1, min(48, 60000000 // (frames * (2 * tokens + 1))) // share))
    return {"op": "align", "seqs": seqs, "frames": frames, "tokens": tokens, "vocab": rng.choice([35, 35, _log(rng, 36, 600)]),
            "dtype": rng.choice(sorted(DTYPES)), "paged": rng.random() < 0.5, "total": rng.random() < 0.6, "share": share}


# --- inputs ---------------------------------------------------------------------------------------------------------

def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def _held(first, end, page):
    """Pages [lo, hi) that hold the frames [first, end)."""
    lo = first // page
    return lo, np.where(first < end, -(-end // page), lo)


def _paged_streams(rs, n, page, window, end_of):
    """A pool in use: frames [first, length) of n streams, each stream's page table row, the queue of free pages."""
    length = rs.integers(0, 4 * window, n)
    kept = end_of(length)
    first = length - kept
    lo, hi = _held(first, length, page)
    held = int((hi - lo).sum())
    return first, length, lo, hi, held


def _prepare_plan(c, rs):
    n, page, window, add_max = c["streams"], c["page"], c["window"], c["add"]
    room = max(0, window - add_max)
    first, length, lo, hi, held = _paged_streams(rs, n, page, max(1, room), lambda ln: np.minimum(ln, rs.integers(0, room + 1, n)))
    add = rs.integers(0, add_max + 1, n) if c["ragged"] else np.full(n, add_max)
    # most streams stay inside their phrase; some finish one and let its frames go; a few are closed
    what = rs.random(n)
    keep = np.where(what < 0.9, first, np.where(what < 0.98, first + (length - first) * rs.random(n), length + add)).astype(np.int64)
    width = -(-window // page) + 1
    pages = n * (width - (-add_max // page) + 1) + 5
    perm = rs.permutation(pages).astype(np.int32)
    rows = rs.permutation(2 * n)
    table = np.full((2 * n, width), -1, np.int32)
    at = 0
    for b in range(n):
        table[rows[b], : hi[b] - lo[b]] = perm[at : at + hi[b] - lo[b]]
        at += int(hi[b] - lo[b])
    head = int(rs.integers(0, 10 * pages))
    queue = np.full(pages, -1, np.int32)
    queue[(head + np.arange(pages - held)) % pages] = perm[held:]
    i32 = lambda a: _dev(np.asarray(a, np.int32))  # noqa: E731
    return {"op": "plan", "page": page, "add_max": add_max, "table": _dev(table), "queue": _dev(queue),
            "cursors_in": _dev(np.array([head, head + pages - held], np.int64)), "cursors_out": torch.zeros(2, dtype=torch.int64, device=DEV),
            "rows_in": i32(rows[:n]), "rows_out": i32(rows[n:]), "first": i32(first), "length": i32(length), "keep": i32(keep), "add": i32(add)}


def _prepare_slots(c, rs):
    n, page, window, most = c["streams"], c["page"], c["window"], c["count"]
    count = rs.integers(1, most + 1, n)
    count[0] = most
    length = rs.integers(window, 4 * window + 1, n)
    first = length - window
    begin = first + (rs.random(n) * (window - count + 1)).astype(np.int64)
    lo, hi = _held(first, length, page)
    width = -(-window // page) + 1
    pages = int((hi - lo).sum()) + 3
    perm = rs.permutation(pages).astype(np.int32)
    table = np.full((2 * n, width), -1, np.int32)
    rows = rs.permutation(2 * n)[:n]
    at = 0
    for b in range(n):
        table[rows[b], : hi[b] - lo[b]] = perm[at : at + hi[b] - lo[b]]
        at += int(hi[b] - lo[b])
    i32 = lambda a: _dev(np.asarray(a, np.int32))  # noqa: E731
    return {"op": "slots", "page": page, "pages": pages, "most": most, "table": _dev(table), "rows": i32(rows), "first": i32(first),
            "begin": i32(begin), "count": i32(count)}


def _logits(c, rows, vocab, gen):
    """Rows as a trained head gives them: one token well ahead in most rows, the rest spread out."""
    x = torch.randn(rows, vocab, device=DEV, generator=gen).mul_(2.0)
    top = torch.randint(0, vocab, (rows, 1), device=DEV, generator=gen)
    return x.scatter_add_(1, top, 10.0 * torch.rand(rows, 1, device=DEV, generator=gen)), top


def _prepare_put(c, rs, gen):
    n = c["streams"] * c["add"]
    x, _ = _logits(c, n, c["vocab"], gen)
    src = torch.log_softmax(x, -1).to(DTYPES[c["src"]]).view(c["streams"], c["add"], c["vocab"])
    total = n + n // 8 + 7
    runs = torch.randperm((total + 15) // 16, device=DEV, generator=gen)              # pages of 16 in any order
    slots = (runs[:, None] * 16 + torch.arange(16, device=DEV)).reshape(-1)
    slots = torch.where(slots < total, slots, -1)[:n].contiguous()
    slots = torch.where(torch.rand(n, device=DEV, generator=gen) < 0.02, -1, slots).view(c["streams"], c["add"])
    return {"op": "put", "src": src, "slots": slots, "pool": torch.zeros(total, c["vocab"], dtype=DTYPES[c["pool"]], device=DEV)}


def _prepare_scores(c, rs, gen):
    n, vocab = c["rows"], c["vocab"]
    held = n + n // 4 + 3 if c["paged"] else n
    x, top = _logits(c, held, vocab, gen)
    if c["masked"]:      # tokens that a grammar forbids
        x.masked_fill_(torch.rand(held, vocab, device=DEV, generator=gen) < 0.1, float("-inf"))
    wide = torch.zeros(held, vocab + c["pad"], dtype=DTYPES[c["dtype"]], device=DEV)
    wide[:, :vocab] = x
    rows = None
    if c["paged"]:
        rows = torch.randperm(held, device=DEV, generator=gen)[:n].contiguous()
        rows = torch.where(torch.rand(n, device=DEV, generator=gen) < 0.05, -1, rows)
        top = top[rows.clamp(min=0)]
    given = torch.where(torch.rand(n, device=DEV, generator=gen) < 0.6, top[:, 0],
                        torch.randint(-1, vocab, (n,), device=DEV, generator=gen)).to(torch.int32)
    return {"op": "scores", "x": wide[:, :vocab], "rows": rows, "tokens": given, "k": c["k"]}


def _prepare_align(c, rs, gen):
    seqs, frames, most, vocab, share = c["seqs"], c["frames"], c["tokens"], c["vocab"], c["share"]
    phrases = seqs // share
    flen = rs.integers(max(1, frames // 2), frames + 1, phrases)
    flen[0] = frames
    tlen = np.minimum(rs.integers(max(1, most // 2), most + 1, phrases), np.maximum(flen // 2, 1))
    tlen[0] = most
    ids = rs.integers(0, vocab - 1, (phrases, most))
    ids[ids >= BLANK] += 1
    said = np.full((phrases, frames), BLANK)
    for p in range(phrases):          # each token at a frame of its own, blanks between
        said[p, ((np.arange(tlen[p]) + 0.5) * flen[p] / tlen[p]).astype(int)] = ids[p, : tlen[p]]
    x = torch.randn(phrases * frames, vocab, device=DEV, generator=gen).mul_(1.5)
    x.scatter_add_(1, _dev(said).view(-1, 1), 6.0 * torch.rand(phrases * frames, 1, device=DEV, generator=gen))
    x = torch.log_softmax(x, -1).to(DTYPES[c["dtype"]])
    hyp = np.repeat(ids, share, 0)
    other = rs.integers(0, vocab - 1, hyp.shape)
    other[other >= BLANK] += 1
    hyp = np.where((rs.random(hyp.shape) < 0.1) & (np.arange(seqs) % share > 0)[:, None], other, hyp)
    tokens = np.where(np.arange(most) < np.repeat(tlen, share)[:, None], hyp, -1)
    state = {"op": "align", "tokens": _dev(tokens.astype(np.int32)), "token_lens": _dev(np.repeat(tlen, share).astype(np.int32)),
             "frame_lens": _dev(np.repeat(flen, share).astype(np.int32)), "total": c["total"], "rows": None}
    if c["paged"] or share > 1:
        perm = torch.randperm(phrases * frames, device=DEV, generator=gen)
        pool = torch.empty_like(x)
        pool[perm] = x
        rows = perm.view(phrases, frames)
        rows = torch.where(torch.arange(frames, device=DEV) < _dev(flen)[:, None], rows, -1)
        return state | {"x": pool, "rows": rows.repeat_interleave(share, 0).contiguous()}
    return state | {"x": x.view(phrases, frames, vocab)}


def prepare(case, seed):
    rs = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    if op == "plan":
        return _prepare_plan(case, rs)
    if op == "slots":
        return _prepare_slots(case, rs)
    return {"put": _prepare_put, "scores": _prepare_scores, "align": _prepare_align}[op](case, rs, gen)


# --- the plain forms -------------------------------------------------------------------------------------------------

def _plain_plan(s):
    page, table, queue, n_pages = s["page"], s["table"], s["queue"], s["queue"].numel()
    first, length, keep, add = (s[k].long() for k in ("first", "length", "keep", "add"))
    rows_in, rows_out = s["rows_in"].long(), s["rows_out"].long()
    head, tail = s["cursors_in"][0], s["cursors_in"][1]
    kept, end = torch.maximum(first, keep), length + add
    had, has = first < length, kept < end
    lo0, lo1 = first // page, kept // page
    hi0, hi1 = torch.where(had, -(-length // page), lo0), torch.where(has, -(-end // page), lo1)
    start = torch.where(had, torch.maximum(hi0, lo1), lo1)
    take = torch.where(has, hi1 - start, 0)
    drop = torch.where(had, torch.where(has, torch.minimum(hi0, lo1), hi0) - lo0, 0)
    t0, d0 = torch.cumsum(take, 0) - take, torch.cumsum(drop, 0) - drop
    width = table.shape[1]
    legal = (first >= 0) & (first <= length) & (add >= 0) & (add <= s["add_max"]) & (keep >= 0) & (keep <= end)
    status = (take.sum() > tail - head).int() + 2 * (hi1 - lo1 > width).any().int() + 4 * (~legal).any().int()
    ok = status == 0
    before = table[rows_in]
    j = torch.arange(width, device=table.device)
    at = lo1[:, None] + j
    old = before.gather(1, (at - lo0[:, None]).clamp(0, width - 1))
    new = queue[(head + t0[:, None] + at - start[:, None]) % n_pages]
    after = torch.where(at < hi1[:, None], torch.where(had[:, None] & (at < hi0[:, None]), old, new), -1)
    after = torch.where(ok, after, before)
    table[rows_out] = after
    goes = ok & (j < drop[:, None])
    to = torch.where(goes, (tail + d0[:, None] + j) % n_pages, n_pages)
    wider = torch.cat([queue, queue[:1]])
    wider.scatter_(0, to.view(-1), before.view(-1))
    queue.copy_(wider[:n_pages])
    s["cursors_out"].copy_(torch.stack([head + torch.where(ok, take.sum(), 0), tail + torch.where(ok, drop.sum(), 0)]))
    i = torch.arange(s["add_max"], device=table.device)
    frame = length[:, None] + i
    slot = after.gather(1, (frame // page - lo1[:, None]).clamp(0, width - 1)).long() * page + frame % page
    slots = torch.where(ok & (i < add[:, None]) & (frame >= kept[:, None]), slot, -1)
    return {"table": table, "queue": queue, "cursors": s["cursors_out"], "slots": slots, "status": status.int().view(1)}


def _plain_slots(s):
    page, table = s["page"], s["table"]
    first, begin, count = (s[k].long() for k in ("first", "begin", "count"))
    i = torch.arange(s["most"], device=table.device)
    frame = begin[:, None] + i
    at = frame // page - (first // page)[:, None]
    got = table[s["rows"].long()].gather(1, at.clamp(0, table.shape[1] - 1)).long()
    fine = (i < count[:, None]) & (frame >= first[:, None]) & (at < table.shape[1]) & (got >= 0) & (got < s["pages"])
    return {"slots": torch.where(fine, got * page + frame % page, -1)}


def _plain_put(s):
    pool = s["pool"]
    slots = s["slots"].view(-1)
    src = s["src"].float().view(slots.numel(), -1).to(pool.dtype)
    fine = (slots >= 0) & (slots < pool.shape[0])
    # rows without a slot go behind the pool's copy and are cut off again
    wider = torch.cat([pool, pool[:1]])
    wider[torch.where(fine, slots, pool.shape[0])] = src
    pool.copy_(wider[: pool.shape[0]])
    return {"pool": pool}


def _plain_scores(s):
    x, tokens, rows, k = s["x"], s["tokens"].long(), s["rows"], s["k"]
    if rows is not None:
        here = (rows >= 0) & (rows < x.shape[0])
        x = x[rows.clamp(0, x.shape[0] - 1)]
    else:
        here = torch.ones_like(tokens, dtype=torch.bool)
    x = x.float()
    vocab = x.shape[1]
    high = x.amax(1, keepdim=True)
    left = high > float("-inf")
    z = torch.where(left, x - high, float("-inf"))
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    z0 = torch.where(e > 0, z, 0.0)
    entropy = torch.where(left, lse - (e * z0).sum(1, keepdim=True) / total, 0.0)[:, 0]
    given = here & (tokens >= 0) & (tokens < vocab)
    t = tokens.clamp(0, vocab - 1)[:, None]
    value = x.gather(1, t)
    lp = torch.where(left, value - high - lse, float("-inf"))[:, 0]
    index = torch.arange(vocab, device=x.device)
    rank = ((x > value) | ((x == value) & (index < t))).sum(1)
    out = {"logprob": torch.where(given, lp, 0.0), "entropy": torch.where(here, entropy, 0.0),
           "rank": torch.where(given, rank, -1).int()}
    if k:
        # one key per entry: its value's order, then the lowest index first
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        ids = torch.topk((order << 32) - index, k, dim=1).indices
        best = x.gather(1, ids)
        best = torch.where(left, best - high - lse, float("-inf"))
        out["top_logprob"] = torch.where(here[:, None], best, float("-inf"))
        out["top_ids"] = torch.where(here[:, None], ids, -1).int()
    return out


def _plain_align(s):
    x, rows, tokens = s["x"], s["rows"], s["tokens"].long()
    seqs, most = tokens.shape
    dev = tokens.device
    if rows is not None:
        frames, vocab = rows.shape[1], x.shape[1]
        x = x[rows.clamp(0, x.shape[0] - 1)].float()
        x = torch.where((rows >= 0)[:, :, None], x, float("-inf"))
    else:
        frames, vocab = x.shape[1:]
        x = x.float()
    flen, tlen = s["frame_lens"].long().clamp(0, frames), s["token_lens"].long().clamp(0, most)
    states = 2 * most + 1
    label = torch.full((seqs, states), BLANK, dtype=torch.long, device=dev)
    label[:, 1::2] = tokens
    index = torch.arange(states, device=dev)
    fine = (label >= 0) & (label < vocab) & ((label != BLANK) | (index % 2 == 0)) & (index < 2 * tlen[:, None] + 1)
    label = label.clamp(0, vocab - 1)
    skip = torch.zeros((seqs, states), dtype=torch.bool, device=dev)
    skip[:, 3::2] = tokens[:, 1:] != tokens[:, :-1]
    none = float("-inf")
    emit = torch.where(fine[:, None], x.gather(2, label[:, None].expand(seqs, frames, states)).double(), none)
    best = torch.full((seqs, states + 2), none, dtype=torch.float64, device=dev)     # two states that nothing reaches in front
    best[:, 2] = 0.0                                                                  # before the first frame: in front of blank 0 ...
    summed = best.clone()
    came = torch.zeros((frames, seqs, states), dtype=torch.uint8, device=dev)
    for t in range(frames):
        stay, one, two = best[:, 2:], best[:, 1:-1], torch.where(skip, best[:, :-2], none)
        if t == 0:                                                                    # ... or of token 0
            two = torch.where(index == 1, best[:, 2:3], none)
            one = torch.full_like(one, none)
        m = torch.maximum(torch.maximum(stay, one), two)
        came[t] = torch.where(stay >= m, 0, torch.where(one >= m, 1, 2))
        on = (t < flen)[:, None]
        next_ = m + emit[:, t]
        if s["total"]:
            a, b, c = summed[:, 2:], summed[:, 1:-1], torch.where(skip, summed[:, :-2], none)
            if t == 0:
                c = torch.where(index == 1, summed[:, 2:3], none)
                b = torch.full_like(b, none)
            h = torch.maximum(torch.maximum(a, b), c)
            h0 = torch.where(h > none, h, 0.0)
            more = h0 + torch.log(torch.exp(a - h0) + torch.exp(b - h0) + torch.exp(c - h0)) + emit[:, t]
            summed[:, 2:] = torch.where(on, more, summed[:, 2:])
        best[:, 2:] = torch.where(on, next_, best[:, 2:])
    last = 2 * tlen[:, None]
    at_blank = best.gather(1, last + 2)[:, 0]
    at_token = torch.where(tlen > 0, best.gather(1, last + 1)[:, 0], none)
    at_token = torch.where(flen > 0, at_token, none)
    score = torch.maximum(at_blank, at_token)
    alive = score > none
    state = torch.where(at_token > at_blank, last[:, 0] - 1, last[:, 0])
    path = torch.full((seqs, frames), -1, dtype=torch.long, device=dev)
    for t in range(frames - 1, -1, -1):
        on = alive & (t < flen)
        path[:, t] = torch.where(on, state, -1)
        step = came[t].gather(1, state[:, None])[:, 0].long()
        state = torch.where(on, state - step, state)
        state = state.clamp(min=0)
    labels = torch.where(path >= 0, label.gather(1, path.clamp(min=0)), -1).int()
    # a token's frames: the first and one past the last that its state holds
    frame = torch.arange(frames, device=dev).expand(seqs, frames)
    of = torch.where((path >= 0) & (path % 2 == 1), path // 2, most)      # frames of no token go behind the last
    begin = torch.full((seqs, most + 1), frames, dtype=torch.long, device=dev).scatter_reduce_(1, of, frame, "amin")
    end = torch.zeros((seqs, most + 1), dtype=torch.long, device=dev).scatter_reduce_(1, of, frame + 1, "amax")
    spans = torch.stack([begin, end], -1)[:, :most]
    inside = alive[:, None] & (torch.arange(most, device=dev) < tlen[:, None])
    spans = torch.where(inside[:, :, None], spans, -1).int()
    out = {"score": score.float(), "labels": labels, "spans": spans}
    if s["total"]:
        a = summed.gather(1, last + 2)[:, 0]
        b = torch.where((tlen > 0) & (flen > 0), summed.gather(1, last + 1)[:, 0], none)
        h = torch.maximum(a, b)
        h0 = torch.where(h > none, h, 0.0)
        out["total"] = (h0 + torch.log(torch.exp(a - h0) + torch.exp(b - h0))).float()
    return out


def run(state):
    s = state
    if own:
        from tone_amd import scoring as S

        if s["op"] == "plan":
            slots, status = S.frames_plan(s["table"], s["queue"], s["cursors_in"], s["cursors_out"], s["rows_in"], s["rows_out"], s["first"],
                                          s["length"], s["keep"], s["add"], page_size=s["page"], max_add=s["add_max"])
            return {"table": s["table"], "queue": s["queue"], "cursors": s["cursors_out"], "slots": slots, "status": status}
        if s["op"] == "slots":
            return {"slots": S.frames_slots(s["table"], s["rows"], s["first"], s["begin"], s["count"], page_size=s["page"],
                                            n_pages=s["pages"], max_count=s["most"])}
        if s["op"] == "put":
            S.frames_put(s["src"], s["slots"], s["pool"])
            return {"pool": s["pool"]}
        if s["op"] == "scores":
            r = S.token_scores(s["x"], s["tokens"], k=s["k"], rows=s["rows"])
            out = {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank}
            if s["k"]:
                out |= {"top_logprob": r.top_logprob, "top_ids": r.top_ids}
            return out
        r = S.ctc_align(s["x"], s["tokens"], s["token_lens"], s["frame_lens"], rows=s["rows"], blank=BLANK, total=s["total"])
        out = {"score": r.score, "labels": r.labels, "spans": r.spans}
        if s["total"]:
            out["total"] = r.total
        return out
    return {"plan": _plain_plan, "slots": _plain_slots, "put": _plain_put, "scores": _plain_scores, "align": _plain_align}[s["op"]](s)


# --- work ------------------------------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "plan":
        n, width = c["streams"], -(-c["window"] // c["page"]) + 1
        mean = c["add"] / 2 if c["ragged"] else c["add"]
        pages = n * (max(0, c["window"] - c["add"]) / 2 / c["page"] + mean / c["page"])
        return {"bytes": int(24 * n + 4 * pages + 4 * n * width + 8 * n * c["add"] + 32), "flops": int(n * (width + c["add"]))}
    if c["op"] == "slots":
        n = c["streams"]
        return {"bytes": int(16 * n + 4 * n * (c["count"] / 2 / c["page"] + 1) + 8 * n * c["count"]), "flops": int(n * c["count"])}
    if c["op"] == "put":
        n = c["streams"] * c["add"]
        return {"bytes": int(n * (8 + c["vocab"] * (SIZES[c["src"]] + SIZES[c["pool"]]))), "flops": int(n * c["vocab"])}
    if c["op"] == "scores":
        n = c["rows"]
        return {"bytes": int(n * (c["vocab"] * SIZES[c["dtype"]] + 4 + 12 + 8 * c["k"] + (8 if c["paged"] else 0))),
                "flops": int(6 * n * c["vocab"])}
    phrases, frames = c["seqs"] // c["share"], 0.75 * c["frames"] if c["seqs"] > c["share"] else c["frames"]
    tokens = 0.75 * c["tokens"] if c["seqs"] > c["share"] else c["tokens"]
    paths = c["seqs"] * frames * (2 * tokens + 1)
    return {"bytes": int(phrases * frames * c["vocab"] * SIZES[c["dtype"]] + c["seqs"] * (8 * c["frames"] * (c["paged"] or c["share"] > 1)
                         + 4 * c["frames"] + 12 * c["tokens"] + 16)),
            "flops": int(paths * (13 if c["total"] else 4))}


# --- the definitions, in 64 bits on the CPU ---------------------------------------------------------------------------

def _exact_plan(s):
    page, table, queue = s["page"], s["table"].cpu().numpy().copy(), s["queue"].cpu().numpy().copy()
    head, tail = (int(v) for v in s["cursors_in"].cpu())
    n_pages = len(queue)
    lists = [s[k].cpu().numpy().astype(np.int64) for k in ("rows_in", "rows_out", "first", "length", "keep", "add")]
    slots = np.full((len(lists[0]), s["add_max"]), -1, np.int64)
    head1, tail1 = head, tail
    before = table.copy()
    for b, (ri, ro, first, length, keep, add) in enumerate(zip(*lists)):
        have = {}
        if first < length:
            have = {p: before[ri, p - first // page] for p in range(first // page, (length - 1) // page + 1)}
        kept, end = max(first, keep), length + add
        need = range(kept // page, (end - 1) // page + 1) if kept < end else range(0)
        for p in sorted(have):
            if p not in need:
                queue[tail1 % n_pages] = have[p]
                tail1 += 1
        row = []
        for p in need:
            if p not in have:
                have[p] = queue[head1 % n_pages]
                head1 += 1
            row.append(have[p])
        table[ro] = -1
        table[ro, : len(row)] = row
        f = np.arange(max(length, kept), end)
        slots[b, f - length] = np.asarray(row, np.int64)[f // page - kept // page] * page + f % page if len(f) else 0
    assert head1 <= tail
    return {"table": torch.from_numpy(table), "queue": torch.from_numpy(queue), "cursors": torch.tensor([head1, tail1]),
            "slots": torch.from_numpy(slots), "status": torch.zeros(1, dtype=torch.int32)}


def _exact_slots(s):
    table, page = s["table"].cpu().numpy(), s["page"]
    lists = [s[k].cpu().numpy().astype(np.int64) for k in ("rows", "first", "begin", "count")]
    slots = np.full((len(lists[0]), s["most"]), -1, np.int64)
    for b, (r, first, begin, count) in enumerate(zip(*lists)):
        f = np.arange(begin, begin + count)
        slots[b, :count] = table[r, f // page - first // page].astype(np.int64) * page + f % page
    return {"slots": torch.from_numpy(slots)}


def _exact_put(s):
    pool = s["pool"].cpu().double().numpy().copy()
    slots = s["slots"].cpu().numpy().reshape(-1)
    src = s["src"].cpu().double().numpy().reshape(len(slots), -1)
    pool[slots[slots >= 0]] = src[slots >= 0]
    return {"pool": torch.from_numpy(pool)}


def _exact_scores(s):
    x, k = s["x"].cpu(), s["k"]
    tokens = s["tokens"].cpu().numpy().astype(np.int64)
    rows = np.arange(len(tokens)) if s["rows"] is None else s["rows"].cpu().numpy()
    n, vocab = len(tokens), x.shape[1]
    lp, entropy, rank = np.zeros(n), np.zeros(n), np.full(n, -1, np.int32)
    top, ids = np.full((n, k), -np.inf), np.full((n, k), -1, np.int32)
    for i in range(n):
        if rows[i] < 0:
            continue
        z = x[rows[i]].double().numpy()
        if not np.any(z > -np.inf):
            p, logp = np.zeros(vocab), np.full(vocab, -np.inf)
        else:
            logp = z - z.max()
            logp -= np.log(np.exp(logp).sum())
            p = np.exp(logp)
        entropy[i] = -(p[p > 0] * logp[p > 0]).sum()
        t = tokens[i]
        if 0 <= t < vocab:
            lp[i], rank[i] = logp[t], (z > z[t]).sum() + (z[:t] == z[t]).sum()
        if k:
            floor = np.partition(z, vocab - k)[vocab - k]
            some = np.flatnonzero(z >= floor)
            some = some[np.argsort(-z[some], kind="stable")][:k]
            top[i], ids[i] = logp[some], some
    out = {"logprob": torch.from_numpy(lp), "entropy": torch.from_numpy(entropy), "rank": torch.from_numpy(rank)}
    if k:
        out |= {"top_logprob": torch.from_numpy(top), "top_ids": torch.from_numpy(ids)}
    return out


def _exact_align(s):
    x = s["x"].cpu().double().numpy()
    tokens, T, L = (s[k].cpu().numpy().astype(np.int64) for k in ("tokens", "frame_lens", "token_lens"))
    rows = None if s["rows"] is None else s["rows"].cpu().numpy()
    seqs, most = tokens.shape
    frames = x.shape[1] if rows is None else rows.shape[1]
    each = np.arange(seqs)
    lab = np.full((seqs, 2 * most + 1), BLANK)
    lab[:, 1::2] = np.maximum(tokens, 0)
    closed = np.where(np.arange(2 * most + 1) > 2 * L[:, None], -np.inf, 0.0)      # states behind a sequence's last
    apart = np.full((seqs, 2 * most + 1), -np.inf)
    apart[:, 3::2][lab[:, 3::2] != lab[:, 1:-2:2]] = 0.0                           # a token may follow another one directly
    back = np.zeros((frames, seqs, 2 * most + 1), np.int8)
    best = added = None
    ends = np.full((2, seqs, 2 * most + 1), -np.inf)
    for t in range(frames):
        row = x[:, t] if rows is None else x[rows[:, t]]
        e = np.take_along_axis(row, lab, 1) + closed
        if t == 0:
            best = np.where(np.arange(2 * most + 1) < 2, e, -np.inf)
            added = best.copy()
        else:
            three = np.full((3,) + best.shape, -np.inf)
            three[0], three[1, :, 1:], three[2, :, 2:] = best, best[:, :-1], best[:, :-2] + apart[:, 2:]
            back[t] = np.where(three[0] >= three[1:].max(0), 0, np.where(three[1] >= three[2], 1, 2))
            best = three.max(0) + e
            if s["total"]:
                three[0], three[1, :, 1:], three[2, :, 2:] = added, added[:, :-1], added[:, :-2] + apart[:, 2:]
                h = np.maximum(three.max(0), -1e300)
                with np.errstate(divide="ignore"):
                    added = h + np.log(np.exp(three - h).sum(0)) + e
        if (T == t + 1).any():
            ends[0, T == t + 1], ends[1, T == t + 1] = best[T == t + 1], added[T == t + 1]
    at_blank, at_token = ends[0, each, 2 * L], ends[0, each, 2 * L - 1]
    score = np.maximum(at_blank, at_token)
    total = np.logaddexp(ends[1, each, 2 * L], ends[1, each, 2 * L - 1])
    labels, spans = np.full((seqs, frames), -1, np.int32), np.full((seqs, most, 2), -1, np.int32)
    for b in np.flatnonzero(score > -np.inf):
        at = 2 * L[b] - (at_token[b] > at_blank[b])
        for t in range(T[b] - 1, -1, -1):
            labels[b, t] = lab[b, at]
            if at % 2:
                spans[b, at // 2, 0] = t
                spans[b, at // 2, 1] = max(spans[b, at // 2, 1], t + 1)
            at -= back[t, b, at]
    out = {"score": torch.from_numpy(score), "labels": torch.from_numpy(labels), "spans": torch.from_numpy(spans)}
    if s["total"]:
        out["total"] = torch.from_numpy(total)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "slots": _exact_slots, "put": _exact_put, "scores": _exact_scores, "align": _exact_align}[s["op"]](s)
