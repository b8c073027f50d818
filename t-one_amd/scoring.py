"""The phrase operators: frames held in pages, scores of given tokens, CTC alignment.

The acoustic path answers with a row of log probabilities per 30 ms frame (``ToneSession.run*``).  The operators here work on
those rows where they are, on the device, until the phrase they belong to has ended:

* ``frames_plan`` / ``frames_slots`` -- page tables and slot maps from the streams' frame counts, ``frames_put`` -- a step's
  rows written through such a map; :class:`FrameStore` keeps their buffers and counts;
* ``token_scores`` -- per row the log probability of a given token, its rank, the entropy, the k best tokens;
* ``ctc_align`` -- the best path of given token sequences, each token's frames, the log probability of all paths.

The functions are stateless (``include/tonehip.h`` has the exact definitions): they check types, shapes, strides and devices
here, write new tensors (or the caller's buffers, where they are arguments), do not synchronize, and run on ``stream`` or the
current stream of the tensors' device.  Contents are checked on the device: an index outside its range is left out or counts as
"none", as documented per argument.  Every one can be captured into a graph.  No gradient flows through them.
"""

from __future__ import annotations

import contextlib
from typing import NamedTuple, Optional

import numpy as np

from . import _lib
from . import config as C

MAX_K = 64              # TONE_SCORES_MAX_K
MAX_TOKENS = 1800       # TONE_ALIGN_MAX_TOKENS
MAX_BATCH = 1 << 20     # TONE_FRAMES_MAX_BATCH
STATUS = {1: "out of pages", 2: "a stream's table row is full", 4: "bad request", 8: "bad queue cursors"}   # TONE_FRAMES_*


_types: dict = {}
_mod = None


def _torch():
    global _mod
    if _mod is None:
        import torch
        _mod = torch
    return _mod


def _type(t, name: str) -> int:
    if not _types:
        torch = _torch()
        _types.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})   # TONE_TYPE_*
    try:
        return _types[t.dtype]
    except KeyError:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}") from None


def _vector(t, name: str, dtype, n: int) -> None:
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous ({n},) {dtype} tensor, got {tuple(t.shape)} {t.dtype}")


def _device(first, *others):
    """The common CUDA device of the tensors."""
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")
    if dev.type != "cuda":
        raise ValueError(f"tensors must be on a GPU, got {dev}")
    return dev


class _On:
    """The stream of one call.  Outputs come from the allocator under that stream; where it is not the current one, the
    inputs are marked as in use on it, so that they may be freed at once after the call."""

    __slots__ = ("raw", "_ctx")

    def __init__(self, dev, stream, *inputs):
        torch = _torch()
        self._ctx = None
        if stream is None:
            self.raw = torch._C._cuda_getCurrentRawStream(dev.index)   # current_stream(dev).cuda_stream without the objects
            return
        if stream.device != dev:
            raise ValueError(f"stream on {stream.device}, tensors on {dev}")
        self.raw = stream.cuda_stream
        if stream != torch.cuda.current_stream(dev):
            self._ctx = torch.cuda.stream(stream)
            for t in inputs:
                if t is not None:
                    t.record_stream(stream)

    def __enter__(self):
        if self._ctx is not None:
            self._ctx.__enter__()
        return self.raw

    def __exit__(self, *exc):
        if self._ctx is not None:
            self._ctx.__exit__(*exc)
        return False


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


_INT_MAX = 2 ** 31 - 1


def _too_large(*sizes: int) -> ValueError:
    """For sizes that the library takes as int: ctypes would pass on their low 32 bits."""
    return ValueError(f"sizes past 2^31 - 1 among {sizes}")


# --- pages ------------------------------------------------------------------------------------------------------------

def _check_table(table, page_size: int, n_pages: int) -> None:
    torch = _torch()
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1 \
            or (table.shape[1] > 1 and table.stride(1) != 1) or table.stride(0) < table.shape[1]:
        raise ValueError("table must be a (rows, width) int32 tensor with unit column stride")
    rows, width = table.shape
    if rows > _INT_MAX or width > _INT_MAX or page_size > _INT_MAX or n_pages > _INT_MAX:
        raise _too_large(rows, width, page_size, n_pages)
    if page_size < 1 or n_pages < 1 or width * page_size > _INT_MAX:
        raise ValueError("page_size and n_pages must be positive and width * page_size below 2^31")


def frames_plan(table, queue, cursors_in, cursors_out, rows_in, rows_out, first, length, keep, add, *, page_size: int,
                max_add: int, slots=None, status=None, stream=None):
    """Move streams from the frames [first, length) to [max(first, keep), length + add); returns (slots, status).

    table int32 (rows, width): request b's pages are read from row rows_in[b] and written to row rows_out[b] (all rows
    distinct); queue int32 (n_pages,) of free page ids with int64 (2,) cursors head, tail; the requests int32 (B,).
    slots int64 (B, max_add): where each new frame goes, -1 for none.  status int32 (1,): 0, or a sum of the
    ``STATUS`` bits and then nothing was taken, released or given a slot.  See ``tone_frames_plan`` (include/tonehip.h)."""
    torch = _torch()
    b = int(rows_in.shape[0]) if rows_in.dim() == 1 else -1
    for t, name in ((rows_in, "rows_in"), (rows_out, "rows_out"), (first, "first"), (length, "length"), (keep, "keep"), (add, "add")):
        _vector(t, name, torch.int32, b)
    _vector(queue, "queue", torch.int32, queue.numel())
    _vector(cursors_in, "cursors_in", torch.int64, 2)
    _vector(cursors_out, "cursors_out", torch.int64, 2)
    _check_table(table, page_size, queue.numel())
    if max_add < 0:
        raise ValueError(f"max_add must not be negative, got {max_add}")
    if b > _INT_MAX or max_add > _INT_MAX:
        raise _too_large(b, max_add)
    if b > MAX_BATCH:
        raise ValueError(f"at most {MAX_BATCH} requests in one plan, got {b}")
    if slots is not None and (slots.dtype != torch.int64 or tuple(slots.shape) != (b, max_add) or not slots.is_contiguous()):
        raise ValueError(f"slots must be a contiguous ({b}, {max_add}) int64 tensor")
    if status is not None:
        _vector(status, "status", torch.int32, 1)
    if abs(cursors_in.data_ptr() - cursors_out.data_ptr()) < 16:
        raise ValueError("cursors_out must not alias cursors_in")
    ins = (table, queue, cursors_in, cursors_out, rows_in, rows_out, first, length, keep, add, slots, status)
    dev = _device(*ins)
    lib = _lib.load()
    with _On(dev, stream, *ins) as st:
        if slots is None:
            slots = rows_in.new_empty((b, max_add), dtype=torch.int64)
        if status is None:
            status = rows_in.new_empty(1)
        _lib.check(lib.tone_frames_plan(dev.index, table.data_ptr(), table.stride(0), table.shape[0], table.shape[1],
                                        queue.data_ptr(), queue.numel(), page_size, cursors_in.data_ptr(), cursors_out.data_ptr(),
                                        rows_in.data_ptr(), rows_out.data_ptr(), first.data_ptr(), length.data_ptr(),
                                        keep.data_ptr(), add.data_ptr(), b, slots.data_ptr(), max_add, status.data_ptr(), st),
                   "tone_frames_plan")
    return slots, status


def frames_slots(table, rows, first, begin, count, *, page_size: int, n_pages: int, max_count: int, slots=None, stream=None):
    """Slots int64 (B, max_count) of the frames begin[b] .. begin[b] + count[b] - 1 of the stream that holds frames from
    first[b] on in table row rows[b]; -1 past the count, before ``first`` and where the row has no page."""
    torch = _torch()
    b = int(rows.shape[0]) if rows.dim() == 1 else -1
    for t, name in ((rows, "rows"), (first, "first"), (begin, "begin"), (count, "count")):
        _vector(t, name, torch.int32, b)
    _check_table(table, page_size, n_pages)
    if max_count < 0:
        raise ValueError(f"max_count must not be negative, got {max_count}")
    if b > _INT_MAX or max_count > _INT_MAX:
        raise _too_large(b, max_count)
    if slots is not None and (slots.dtype != torch.int64 or tuple(slots.shape) != (b, max_count) or not slots.is_contiguous()):
        raise ValueError(f"slots must be a contiguous ({b}, {max_count}) int64 tensor")
    ins = (table, rows, first, begin, count, slots)
    dev = _device(*ins)
    lib = _lib.load()
    with _On(dev, stream, *ins) as st:
        if slots is None:
            slots = rows.new_empty((b, max_count), dtype=torch.int64)
        _lib.check(lib.tone_frames_slots(dev.index, table.data_ptr(), table.stride(0), table.shape[0], table.shape[1], n_pages,
                                         page_size, rows.data_ptr(), first.data_ptr(), begin.data_ptr(), count.data_ptr(), b,
                                         slots.data_ptr(), max_count, st), "tone_frames_slots")
    return slots


def _rows_of(t, name: str) -> int:
    """Distance of the rows of a (..., V) tensor, whose leading dimensions must be one run of equally spaced rows."""
    if t.dim() < 2 or t.shape[-1] < 1:
        raise ValueError(f"{name} must be (..., vocab), got {tuple(t.shape)}")
    if t.is_contiguous():
        return t.shape[-1]
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have unit stride along the vocabulary")
    step = run = None
    for d in range(t.dim() - 2, -1, -1):
        if t.shape[d] == 1:
            continue
        if step is None:
            step, run = t.stride(d), t.stride(d) * t.shape[d]
        elif t.stride(d) != run:
            raise ValueError(f"{name}'s leading dimensions must be one run of equally spaced rows")
        else:
            run *= t.shape[d]
    return t.shape[-1] if step is None else step


def _check_put(src, pool) -> tuple[int, int, int, int]:
    """What :func:`frames_put` asks of its rows and its pool: (type of src, type of the pool, distance of src's rows, rows)."""
    stype, ptype = _type(src, "src"), _type(pool, "pool")
    sstride = _rows_of(src, "src")
    vocab = src.shape[-1]
    if pool.dim() != 2 or pool.shape[1] != vocab or (vocab > 1 and pool.stride(1) != 1) or (pool.shape[0] > 1 and pool.stride(0) < vocab):
        raise ValueError(f"pool must be (rows, {vocab}) with unit column stride, got {tuple(pool.shape)}")
    n = src.numel() // vocab
    if vocab > _INT_MAX:
        raise _too_large(vocab)
    if n > 1 and sstride < vocab:
        raise ValueError("src rows must not overlap")
    # (no entry has more than 4 bytes: most calls need no closer look)
    at = src.data_ptr() - pool.data_ptr()
    if -4 * (n * sstride) < at < 4 * (pool.shape[0] * max(pool.stride(0), vocab)) and _meet(src, sstride, n, pool, at):
        raise ValueError("src must not overlap the pool")
    return stype, ptype, sstride, n


def _meet(src, sstride: int, n: int, pool, at: int) -> bool:
    """Whether rows of ``src`` (n, sstride entries apart, the first ``at`` bytes behind the pool's) and the pool share memory;
    columns side by side in rows of the same length do not."""
    vocab, rows = src.shape[-1], pool.shape[0]
    if n == 0 or rows == 0 or src.device != pool.device:
        return False
    each, to = src.element_size(), pool.element_size()
    pitch, pool_pitch = sstride * each, max(pool.stride(0), vocab) * to      # (the stride of a single row says nothing)
    if at >= (rows - 1) * pool_pitch + vocab * to or at + (n - 1) * pitch + vocab * each <= 0:
        return False
    if n == 1:
        pitch = pool_pitch
    elif rows > 1 and pitch != pool_pitch:
        return True
    return not (at % pitch >= vocab * to and at % pitch + vocab * each <= pitch)


def frames_put(src, slots, pool, stream=None) -> None:
    """pool[slots[i]] = row i of ``src`` (..., vocab), rounded once to the pool's type; slots int64 with one entry per row,
    distinct, those outside the pool left out.  pool (n_rows, vocab) float32 / float16 / bfloat16; ``src`` must not lie in it."""
    torch = _torch()
    stype, ptype, sstride, n = _check_put(src, pool)
    if slots.dtype != torch.int64 or slots.numel() != n or not slots.is_contiguous():
        raise ValueError(f"slots must be {n} contiguous int64 entries, got {tuple(slots.shape)} {slots.dtype}")
    dev = _device(src, slots, pool)
    lib = _lib.load()
    with _On(dev, stream, src, slots, pool) as st:
        _lib.check(lib.tone_frames_put(dev.index, src.data_ptr(), stype, sstride, slots.data_ptr(), n, src.shape[-1],
                                       pool.data_ptr(), ptype, max(pool.stride(0), pool.shape[1]), pool.shape[0], st),
                   "tone_frames_put")


# --- scores -----------------------------------------------------------------------------------------------------------

class TokenScores(NamedTuple):
    """Per row, shaped like ``tokens`` / ``rows`` / the leading dimensions of x (top_*: one dimension of k more)."""
    logprob: Optional[object]       # float32; None without tokens
    rank: Optional[object]          # int32; None without tokens
    entropy: object                 # float32, nats
    top_logprob: Optional[object]   # float32; None for k = 0
    top_ids: Optional[object]       # int32; None for k = 0


def token_scores(x, tokens=None, k: int = 0, rows=None, stream=None) -> TokenScores:
    """What rows of logits or log probabilities (..., vocab) say: the log probability and rank of a given token, the entropy,
    the ``k`` best tokens (equal values: lowest id first).

    ``rows`` int64, any shape: row indices into x (n_rows, vocab), e.g. a slot map into a pool; an index outside is no row
    (logprob 0, rank -1, entropy 0, top -inf / -1).  ``tokens`` int32, one per row; an id outside the vocabulary is no token
    (logprob 0, rank -1).  -inf entries have probability 0.  k <= min(vocab, 64)."""
    torch = _torch()
    typ = _type(x, "x")
    vocab = int(x.shape[-1]) if x.dim() >= 2 else 0
    if rows is not None:
        if x.dim() != 2:
            raise ValueError(f"x must be (n_rows, vocab) with rows, got {tuple(x.shape)}")
        if rows.dtype != torch.int64 or not rows.is_contiguous():
            raise ValueError(f"rows must be a contiguous int64 tensor, got {rows.dtype}")
    stride = _rows_of(x, "x")
    shape = rows.shape if rows is not None else x.shape[:-1]
    x_rows = x.numel() // vocab
    n = rows.numel() if rows is not None else x_rows
    if tokens is not None and (tokens.dtype != torch.int32 or tokens.shape != shape or not tokens.is_contiguous()):
        raise ValueError(f"tokens must be a contiguous {tuple(shape)} int32 tensor, got {tuple(tokens.shape)} {tokens.dtype}")
    if vocab > _INT_MAX:
        raise _too_large(vocab)
    k = int(k)
    if not 0 <= k <= min(vocab, MAX_K):
        raise ValueError(f"k must be in 0 .. min(vocab, {MAX_K}), got {k}")
    if x_rows > 1 and stride < vocab:
        raise ValueError("x rows must not overlap")
    dev = _device(x, tokens, rows)
    lib = _lib.load()
    with _On(dev, stream, x, tokens, rows) as st:
        # (new_empty and empty_like take half the time of torch.empty with a shape, dtype and device)
        lp = rank = top = ids = None
        size = tuple(shape)
        entropy = x.new_empty(size, dtype=torch.float32)
        if tokens is not None:
            lp, rank = torch.empty_like(entropy), torch.empty_like(tokens)
        if k:
            size += (k,)
            top, ids = entropy.new_empty(size), entropy.new_empty(size, dtype=torch.int32)
        _lib.check(lib.tone_token_scores(dev.index, x.data_ptr(), typ, stride, x_rows, _ptr(rows), n, vocab, _ptr(tokens), k,
                                         _ptr(lp), entropy.data_ptr(), _ptr(rank), _ptr(top), _ptr(ids), st),
                   "tone_token_scores")
    return TokenScores(lp, rank, entropy, top, ids)


# --- alignment --------------------------------------------------------------------------------------------------------

class CtcAlignment(NamedTuple):
    score: object               # float32 (B,): log probability of the best path
    total: Optional[object]     # float32 (B,): of all paths; None unless asked for
    labels: object              # int32 (B, T): the best path's label per frame, -1 behind the last frame
    spans: object               # int32 (B, L, 2): each token's frames [begin, end), -1 behind the last token


def ctc_align(x, tokens, token_lens, frame_lens, rows=None, blank: int = C.BLANK_ID, total: bool = False,
              stream=None) -> CtcAlignment:
    """Align token sequences with frames of log probabilities.

    x (B, T, vocab), batch and frame strides free (an expanded batch shares its frames), or with ``rows`` int64 (B, T) a pool
    (n_rows, vocab) read through that slot map.  tokens int32 (B, L), token_lens / frame_lens int32 (B,), clamped to L and T.
    A sequence that no path fits has score -inf and labels / spans -1.  See ``tone_ctc_align`` (include/tonehip.h)."""
    torch = _torch()
    typ = _type(x, "x")
    if tokens.dtype != torch.int32 or tokens.dim() != 2 or not tokens.is_contiguous():
        raise ValueError(f"tokens must be a contiguous (B, L) int32 tensor, got {tuple(tokens.shape)} {tokens.dtype}")
    b, most = int(tokens.shape[0]), int(tokens.shape[1])
    if most > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} tokens per sequence, got {most}")
    _vector(token_lens, "token_lens", torch.int32, b)
    _vector(frame_lens, "frame_lens", torch.int32, b)
    if rows is not None:
        if rows.dtype != torch.int64 or rows.dim() != 2 or rows.shape[0] != b or not rows.is_contiguous():
            raise ValueError(f"rows must be a contiguous ({b}, T) int64 tensor, got {tuple(rows.shape)} {rows.dtype}")
        if x.dim() != 2:
            raise ValueError(f"x must be (n_rows, vocab) with rows, got {tuple(x.shape)}")
        frames, x_rows, stride, bstride = int(rows.shape[1]), int(x.shape[0]), x.stride(0), 0
    else:
        if x.dim() != 3 or x.shape[0] != b:
            raise ValueError(f"x must be ({b}, T, vocab), got {tuple(x.shape)}")
        frames, x_rows, stride, bstride = int(x.shape[1]), 0, x.stride(1), x.stride(0)
    vocab = int(x.shape[-1])
    if vocab < 1 or (vocab > 1 and x.stride(-1) != 1):
        raise ValueError("x must have unit stride along a vocabulary of at least one entry")
    if b > _INT_MAX or frames > _INT_MAX or vocab > _INT_MAX:
        raise _too_large(b, frames, vocab)
    if not 0 <= blank < vocab:
        raise ValueError(f"blank {blank} outside the vocabulary of {vocab}")
    dev = _device(x, tokens, token_lens, frame_lens, rows)
    lib = _lib.load()
    need = lib.tone_ctc_align_workspace(b, frames, most)
    if need < 0:
        raise ValueError(f"{frames} frames are too many for one launch")
    with _On(dev, stream, x, tokens, token_lens, frame_lens, rows) as st:
        score = token_lens.new_empty(b, dtype=torch.float32)
        tot = torch.empty_like(score) if total else None
        labels, spans = tokens.new_empty((b, frames)), tokens.new_empty((b, most, 2))
        ws = tokens.new_empty(need, dtype=torch.uint8) if need else None
        _lib.check(lib.tone_ctc_align(dev.index, x.data_ptr(), typ, stride, bstride, x_rows, _ptr(rows), b, frames, vocab, blank,
                                      tokens.data_ptr(), most, token_lens.data_ptr(), frame_lens.data_ptr(), score.data_ptr(),
                                      _ptr(tot), labels.data_ptr(), spans.data_ptr(), _ptr(ws), need, st), "tone_ctc_align")
    return CtcAlignment(score, tot, labels, spans)


# --- a store of frames ------------------------------------------------------------------------------------------------

class FrameStore:
    """The latest rows of many streams, in pages of one pool on the device.

    Stream i holds its frames [first, length), counted from its start.  :meth:`append` adds a step's rows for any subset of
    the streams (:meth:`reserve`: only their slots) and lets go of the frames before ``keep``; :meth:`slots` gives the pool rows
    of a range of frames, for ``token_scores`` / ``ctc_align`` with ``rows=``.  Page tables, slot maps and the free list live on
    the device; the host keeps the counts, so a call that would run out of pages raises before anything has changed.  The
    calls on one store belong on one stream (or ordered by events) and, as the counts are the host's, not into a graph; the
    pool and the tables are the store's own."""

    def __init__(self, n_streams: int, max_frames: int, *, page_size: int = 64, n_pages: Optional[int] = None, vocab: int = C.VOCAB,
                 dtype=None, device: int = 0):
        """``max_frames``: the most a stream holds at once.  ``n_pages``: pages of the pool, by default enough for every
        stream at its most."""
        torch = _torch()
        if n_streams < 1 or max_frames < 1 or page_size < 1 or vocab < 1:
            raise ValueError("n_streams, max_frames, page_size and vocab must be positive")
        dtype = torch.float32 if dtype is None else dtype
        if dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        self.n_streams, self.max_frames, self.page_size = int(n_streams), int(max_frames), int(page_size)
        self.width = -(-self.max_frames // self.page_size) + 1          # a range of frames can begin inside a page
        self.n_pages = int(n_pages) if n_pages is not None else self.n_streams * self.width
        if self.n_pages < 1:
            raise ValueError("n_pages must be positive")
        if not torch.cuda.is_available():
            raise RuntimeError("FrameStore needs a ROCm GPU (torch.cuda.is_available() is False)")
        self.dev = torch.device("cuda", int(device))
        self.pool = torch.zeros((self.n_pages * self.page_size, vocab), dtype=dtype, device=self.dev)
        self._table = torch.full((2 * self.n_streams, self.width), -1, dtype=torch.int32, device=self.dev)
        self._queue = torch.arange(self.n_pages, dtype=torch.int32, device=self.dev)
        self._cursors = torch.tensor([[0, self.n_pages], [0, 0]], dtype=torch.int64, device=self.dev)
        self._home = torch.cuda.current_stream(self.dev)                 # what the allocator knows the buffers by
        self._side = 0                                                   # which cursors are current
        self.first = np.zeros(self.n_streams, np.int64)
        self.length = np.zeros(self.n_streams, np.int64)
        self._parity = np.zeros(self.n_streams, np.int64)
        self.free_pages = self.n_pages
        torch.cuda.current_stream(self.dev).synchronize()                # the buffers are as they should be, for any stream

    @contextlib.contextmanager
    def _use(self, stream):
        """The call's stream as the current one; the buffers are marked as in use on it, so that the store may be dropped while
        its calls are under way."""
        torch = _torch()
        if stream is not None and stream.device != self.dev:
            raise ValueError(f"stream on {stream.device}, the store on {self.dev}")
        with (torch.cuda.stream(stream) if stream is not None else torch.cuda.device(self.dev)):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the calls of a FrameStore cannot be captured into a graph: their counts are the host's")
            now = torch.cuda.current_stream(self.dev)
            if now != self._home:
                for t in (self.pool, self._table, self._queue, self._cursors):
                    t.record_stream(now)
            yield

    def _ids(self, ids) -> np.ndarray:
        ids = np.asarray(ids, np.int64).reshape(-1)
        if ids.size and (ids.min() < 0 or ids.max() >= self.n_streams):
            raise ValueError(f"stream ids must be in [0, {self.n_streams})")
        return ids

    def _upload(self, *columns):
        """int32 columns as one device tensor, through pinned memory that the copy keeps until it is done."""
        torch = _torch()
        n = columns[0].shape[0]
        host = torch.empty((len(columns), n), dtype=torch.int32, pin_memory=True)
        view = host.numpy()
        for row, c in zip(view, columns):
            row[:] = c
        return host.to(self.dev, non_blocking=True)

    def _plan(self, ids, keep, add, max_add):
        if len(set(ids.tolist())) != ids.size:
            raise ValueError("stream ids must be distinct")
        first, length, page = self.first[ids], self.length[ids], self.page_size
        kept, end = np.maximum(first, keep), length + add
        if (keep < 0).any() or (kept > end).any() or (end >= 2 ** 31).any():
            raise ValueError("keep must be in 0 .. length + count, and frame numbers below 2^31")
        if (end - kept > self.max_frames).any():
            raise ValueError(f"a stream would hold more than max_frames = {self.max_frames} frames")
        lo0, lo1 = first // page, kept // page
        hi0, hi1 = np.where(first < length, -(-length // page), lo0), np.where(kept < end, -(-end // page), lo1)
        had, has = first < length, kept < end
        take = int(np.where(has, hi1 - np.where(had, np.maximum(hi0, lo1), lo1), 0).sum())
        drop = int(np.where(had, np.where(has, np.minimum(hi0, lo1), hi0) - lo0, 0).sum())
        if take > self.free_pages:
            raise RuntimeError(f"out of pages: {take} needed, {self.free_pages} of {self.n_pages} free")
        rows = 2 * ids + self._parity[ids]
        req = self._upload(rows, rows ^ 1, first, length, keep, add)
        slots, _ = frames_plan(self._table, self._queue, self._cursors[self._side], self._cursors[1 - self._side], *req.unbind(0),
                               page_size=page, max_add=max_add)
        self._side = 1 - self._side
        self.first[ids], self.length[ids] = kept, end
        self._parity[ids] ^= 1
        self.free_pages += drop - take
        return slots

    @contextlib.contextmanager
    def _undone(self):
        """Takes back what is reserved under it where the block raises.  The host's counts are all there is to take back: a
        plan writes spare table rows, the other cursors and queue entries behind the free ones, and the next one is made from
        the rows and cursors it was made from itself."""
        was = self.first.copy(), self.length.copy(), self._parity.copy(), self._side, self.free_pages
        try:
            yield
        except BaseException:
            self.first, self.length, self._parity, self._side, self.free_pages = was
            raise

    def reserve(self, ids, frames: int, keep=None, counts=None, stream=None):
        """Slots int64 (n, frames) for the next counts[i] (default: ``frames``) frames of the streams ``ids`` (distinct), to be
        written with :func:`frames_put`.  Frames before keep[i] (default: none) are let go; new ones among them get no slot."""
        torch = _torch()
        ids = self._ids(ids)
        add = np.full(ids.size, frames, np.int64) if counts is None else np.asarray(counts, np.int64).reshape(-1)
        keep = self.first[ids] if keep is None else np.asarray(keep, np.int64).reshape(-1)
        if add.shape != ids.shape or keep.shape != ids.shape or (add < 0).any() or (add > frames).any():
            raise ValueError(f"counts must be {ids.size} numbers in 0 .. {frames}, keep {ids.size} frame numbers")
        with self._use(stream):
            return self._plan(ids, keep, add, frames)

    def append(self, rows, ids, keep=None, counts=None, stream=None):
        """Add ``rows`` (n, T, vocab) to the streams ``ids``: :meth:`reserve` and the copy.  Returns the slots (n, T)."""
        torch = _torch()
        ids = self._ids(ids)
        if rows.dim() != 3 or rows.shape[0] != ids.size or rows.shape[2] != self.pool.shape[1]:
            raise ValueError(f"rows must be ({ids.size}, T, {self.pool.shape[1]}), got {tuple(rows.shape)}")
        if rows.device != self.dev:
            raise ValueError(f"rows on {rows.device}, the store on {self.dev}")
        _check_put(rows, self.pool)
        with self._undone():
            slots = self.reserve(ids, int(rows.shape[1]), keep, counts, stream)
            frames_put(rows, slots, self.pool, stream=stream)
        return slots

    def release(self, ids, stream=None) -> None:
        """Let go of all frames of the streams ``ids``; they start again at frame 0."""
        torch = _torch()
        ids = self._ids(ids)
        if ids.size == 0:
            return
        with self._use(stream):
            self._plan(ids, self.length[ids], np.zeros(ids.size, np.int64), 0)
        self.first[ids] = self.length[ids] = 0

    def slots(self, ids, begin, count, stream=None):
        """Pool rows int64 (n, max(count)) of the frames begin[i] .. begin[i] + count[i] - 1 of stream ids[i], -1 behind
        them.  A stream may be named more than once."""
        torch = _torch()
        ids = self._ids(ids)
        begin, count = np.asarray(begin, np.int64).reshape(-1), np.asarray(count, np.int64).reshape(-1)
        if begin.shape != ids.shape or count.shape != ids.shape:
            raise ValueError("ids, begin and count must have one entry per range")
        if (count < 0).any() or (begin < self.first[ids]).any() or (begin + count > self.length[ids]).any():
            raise ValueError("ranges must lie inside the frames their streams hold")
        most = int(count.max()) if ids.size else 0
        with self._use(stream):
            req = self._upload(2 * ids + self._parity[ids], self.first[ids], begin, count)
            return frames_slots(self._table, *req.unbind(0), page_size=self.page_size, n_pages=self.n_pages, max_count=most)
