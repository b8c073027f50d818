"""The phrase operators on the CPU: the oracle against brute force, and every refusal that needs no GPU -- of the Python
functions and of the C entry points, which check their arguments before they touch the device."""

import ctypes

import numpy as np
import pytest

import phrase_oracle as O
from tone_amd import _lib
from tone_amd import scoring as S

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("seed", range(12))
def test_oracle_alignment_is_the_best_and_the_sum_of_all_paths(seed):
    rng = np.random.default_rng(seed)
    f, vocab = int(rng.integers(1, 7)), int(rng.integers(2, 5))
    blank = int(rng.integers(0, vocab))
    tokens = [int(t) for t in rng.integers(0, vocab, int(rng.integers(0, 4))) if t != blank]
    x = np.log(rng.dirichlet(np.ones(vocab), f))
    score, total, labels, spans = O.align(x, tokens, blank)
    want = O.align_by_paths(x, tokens, blank)
    np.testing.assert_allclose([score, total], want, rtol=1e-12)
    if labels is not None:
        assert [c for i, c in enumerate(labels) if c != blank and (i == 0 or labels[i - 1] != c)] == tokens
        np.testing.assert_allclose(sum(x[t, c] for t, c in enumerate(labels)), score, rtol=1e-12)
        for t, (a, b) in zip(tokens, spans):
            assert all(labels[i] == t for i in range(a, b))


def test_oracle_scores_sum_to_one():
    rng = np.random.default_rng(0)
    row = rng.normal(size=35)
    lp, rank, entropy, top, _ = O.scores(row, 7, 35)
    p = np.exp([v for _, v in top])
    np.testing.assert_allclose(p.sum(), 1.0, rtol=1e-12)
    np.testing.assert_allclose(entropy, -(p * np.log(p)).sum(), rtol=1e-12)
    assert top[rank][0] == 7 and top[rank][1] == lp


def test_oracle_plan_keeps_every_page_once():
    rng = np.random.default_rng(3)
    page, n, width, pages = 4, 3, 6, 20
    table, queue, cur = np.full((2 * n, width), -1, np.int32), np.arange(pages, dtype=np.int32), np.array([0, pages])
    first, length, par = np.zeros(n, int), np.zeros(n, int), np.zeros(n, int)
    for _ in range(40):
        add = rng.integers(0, 6, n)
        keep = np.minimum(length + add, np.maximum(first, length - rng.integers(0, 12, n)))
        table, queue, cur, slots = O.plan(table, queue, cur, 2 * np.arange(n) + par, 2 * np.arange(n) + 1 - par, first, length, keep, add, page, 6)
        first, length, par = np.maximum(first, keep), length + add, 1 - par
        held = np.concatenate([table[2 * i + par[i]] for i in range(n)])
        free = [int(queue[i % pages]) for i in range(cur[0], cur[1])]
        assert sorted(list(held[held >= 0]) + free) == list(range(pages))
        got = slots[slots >= 0]
        assert len(set(got)) == len(got)


# --- refusals of the Python functions ---------------------------------------------------------------------------------

def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _plan_args(**change):
    a = dict(table=torch.zeros((4, 3), dtype=torch.int32), queue=torch.arange(8, dtype=torch.int32),
             cursors_in=torch.tensor([0, 8]), cursors_out=torch.zeros(2, dtype=torch.int64), rows_in=_i32(0, 2), rows_out=_i32(1, 3),
             first=_i32(0, 0), length=_i32(0, 0), keep=_i32(0, 0), add=_i32(1, 2), page_size=4, max_add=2)
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    {"table": torch.zeros((4, 3), dtype=torch.int64)}, {"table": torch.zeros((3, 4), dtype=torch.int32).t()},
    {"table": torch.zeros(4, dtype=torch.int32)}, {"queue": torch.arange(8)}, {"queue": torch.empty(0, dtype=torch.int32)},
    {"cursors_in": _i32(0, 8)}, {"cursors_out": torch.zeros(3, dtype=torch.int64)}, {"rows_in": _i32(0)},
    {"rows_out": torch.tensor([1, 3])}, {"first": _i32(0, 0, 0)}, {"add": _i32(0, 1, 2, 3)[::2]}, {"page_size": 0},
    {"max_add": -1}, {"page_size": 2 ** 30}, {"slots": torch.zeros((2, 3), dtype=torch.int64)},
    {"slots": torch.zeros((2, 2), dtype=torch.int32)}, {"status": torch.zeros(2, dtype=torch.int32)}, {},
])
def test_frames_plan_refuses(change):
    """Wrong types, shapes and strides; with nothing changed, tensors that are not on a GPU."""
    with pytest.raises(ValueError):
        S.frames_plan(**_plan_args(**change))


def test_frames_plan_refuses_aliased_cursors():
    a = _plan_args()
    a["cursors_out"] = a["cursors_in"]
    with pytest.raises(ValueError, match="alias"):
        S.frames_plan(**a)


@pytest.mark.parametrize("change", [{"rows": torch.tensor([0])}, {"first": _i32(0, 1)}, {"max_count": -1}, {"n_pages": 0},
                                    {"slots": torch.zeros((1, 3), dtype=torch.int64)}, {}])
def test_frames_slots_refuses(change):
    a = dict(table=torch.zeros((4, 3), dtype=torch.int32), rows=_i32(0), first=_i32(0), begin=_i32(0), count=_i32(1), page_size=4,
             n_pages=3, max_count=2)
    a.update(change)
    with pytest.raises(ValueError):
        S.frames_slots(**a)


@pytest.mark.parametrize("change", [
    {"src": torch.zeros((2, 5), dtype=torch.float64)}, {"src": torch.zeros((2, 4))}, {"src": torch.zeros((5, 2)).t()},
    {"slots": torch.zeros(3, dtype=torch.int64)}, {"slots": torch.zeros(2, dtype=torch.int32)}, {"pool": torch.zeros((9, 5), dtype=torch.int8)},
    {"pool": torch.zeros((3, 3, 5))}, {"pool": torch.zeros((1, 5)).expand(9, 5)}, {"src": torch.zeros((1, 5)).expand(2, 5)}, {},
])
def test_frames_put_refuses(change):
    a = dict(src=torch.zeros((2, 5)), slots=torch.zeros(2, dtype=torch.int64), pool=torch.zeros((9, 5)))
    a.update(change)
    with pytest.raises(ValueError):
        S.frames_put(**a)


def test_rows_of_any_leading_shape():
    x = torch.zeros((6, 10, 8))
    assert S._rows_of(x, "x") == 8 and S._rows_of(x[:, :, :5], "x") == 8 and S._rows_of(x[:, :1], "x") == 80
    assert S._rows_of(x[::2, :1, :3], "x") == 160 and S._rows_of(x[:1, ::2], "x") == 16 and S._rows_of(x[:1, :1, :3], "x") == 3
    assert S._rows_of(torch.zeros((1, 8)).expand(4, 8), "x") == 0 and S._rows_of(torch.zeros((0, 8)), "x") == 8
    for bad in (x[:, :7], x.transpose(0, 1), x[:, :, ::2]):
        with pytest.raises(ValueError):
            S._rows_of(bad, "x")


@pytest.mark.parametrize("change", [
    {"x": torch.zeros((2, 5), dtype=torch.int32)}, {"x": torch.zeros(5)}, {"x": torch.zeros((2, 0))}, {"x": torch.zeros((5, 2)).t()},
    {"tokens": torch.zeros(2, dtype=torch.int64)}, {"tokens": torch.zeros(3, dtype=torch.int32)}, {"k": 6}, {"k": -1},
    {"x": torch.zeros((2, 100)), "k": 65}, {"rows": torch.zeros(2, dtype=torch.int32)},
    {"x": torch.zeros((1, 2, 5)), "rows": torch.zeros(2, dtype=torch.int64)}, {"rows": torch.zeros(3, dtype=torch.int64)},
    {"x": torch.zeros((1, 5)).expand(2, 5)}, {},
])
def test_token_scores_refuses(change):
    a = dict(x=torch.zeros((2, 5)), tokens=torch.zeros(2, dtype=torch.int32), k=2)
    a.update(change)
    with pytest.raises(ValueError):
        S.token_scores(**a)


@pytest.mark.parametrize("change", [
    {"x": torch.zeros((2, 6, 5), dtype=torch.float64)}, {"x": torch.zeros((3, 6, 5))}, {"x": torch.zeros((6, 5))},
    {"x": torch.zeros((2, 5, 6)).transpose(1, 2)}, {"tokens": torch.zeros((2, 3), dtype=torch.int64)},
    {"tokens": torch.zeros(2, dtype=torch.int32)}, {"tokens": torch.zeros((2, S.MAX_TOKENS + 1), dtype=torch.int32)},
    {"token_lens": _i32(1)}, {"frame_lens": torch.tensor([1, 1])}, {"blank": 5}, {"blank": -1},
    {"rows": torch.zeros((2, 6), dtype=torch.int64)}, {"x": torch.zeros((9, 5)), "rows": torch.zeros((3, 6), dtype=torch.int64)},
    {"x": torch.zeros((9, 5)), "rows": torch.zeros((2, 6), dtype=torch.int32)}, {},
])
def test_ctc_align_refuses(change):
    a = dict(x=torch.zeros((2, 6, 5)), tokens=torch.zeros((2, 3), dtype=torch.int32), token_lens=_i32(3, 2), frame_lens=_i32(6, 6), blank=4)
    a.update(change)
    with pytest.raises(ValueError):
        S.ctc_align(**a)


# --- refusals of the C entry points: before any device call, so the pointers here are never followed --------------------

P = ctypes.c_void_p(4096)      # not null
Q = ctypes.c_void_p(8192)


def _refused(rc, *words):
    msg = _lib.load().tone_last_error().decode()
    assert rc == -1 and all(w in msg for w in words), (rc, msg)


def test_c_frames_plan_refuses():
    def call(table=P, stride=3, n_rows=4, width=3, queue=P, n_pages=8, page=4, cin=P, cout=Q, req=P, batch=2, slots=P, max_add=2, status=P):
        return _lib.load().tone_frames_plan(0, table, stride, n_rows, width, queue, n_pages, page, cin, cout, req, P, P, P, P, P, batch,
                                            slots, max_add, status, None)
    _refused(call(table=None), "tone_frames_plan", "null")
    _refused(call(queue=None), "null")
    _refused(call(status=None), "null")
    _refused(call(req=None), "null")
    _refused(call(slots=None), "null")
    _refused(call(cout=P), "cursors_out")
    _refused(call(stride=2), "table_stride")
    _refused(call(page=0), "positive")
    _refused(call(n_pages=0), "positive")
    _refused(call(batch=-1), "negative")
    _refused(call(page=1 << 30), "2^31")


def test_c_frames_plan_refuses_overlapping_cursors():
    at = [ctypes.c_void_p(4096 + 8 * i) for i in range(5)]
    for i, j in ((2, 1), (2, 2), (2, 3)):
        _refused(_lib.load().tone_frames_plan(0, P, 3, 4, 3, P, 8, 4, at[i], at[j], P, P, P, P, P, P, 2, P, 2, P, None), "cursors_out")


def test_c_frames_slots_and_put_refuse():
    lib = _lib.load()
    _refused(lib.tone_frames_slots(0, P, 3, 4, 3, 8, 4, None, P, P, P, 1, P, 2, None), "null")
    _refused(lib.tone_frames_slots(0, P, 2, 4, 3, 8, 4, P, P, P, P, 1, P, 2, None), "table_stride")
    _refused(lib.tone_frames_slots(0, P, 3, 4, 3, 8, 4, P, P, P, P, -1, P, 2, None), "negative")
    _refused(lib.tone_frames_slots(0, P, 3, 4, 3, 8, 4, P, P, P, P, 1 << 30, P, 1 << 20, None), "one launch")
    _refused(lib.tone_frames_put(0, P, 7, 5, P, 2, 5, P, 0, 5, 9, None), "type")
    _refused(lib.tone_frames_put(0, P, 0, 4, P, 2, 5, P, 0, 5, 9, None), "stride")
    _refused(lib.tone_frames_put(0, P, 0, 5, None, 2, 5, P, 0, 5, 9, None), "null")
    _refused(lib.tone_frames_put(0, P, 0, 5, P, -2, 5, P, 0, 5, 9, None), "range")


def test_c_token_scores_refuses():
    lib = _lib.load()

    def call(x=P, typ=0, stride=5, x_rows=2, rows=None, n=2, vocab=5, tokens=P, k=2, lp=P, ent=P, top=P):
        return lib.tone_token_scores(0, x, typ, stride, x_rows, rows, n, vocab, tokens, k, lp, ent, P, top, P, None)
    _refused(call(x=None), "null")
    _refused(call(ent=None), "null")
    _refused(call(top=None), "null")
    _refused(call(lp=None), "logprob")
    _refused(call(k=6), "k must")
    _refused(call(vocab=100, stride=100, k=65), "k must")
    _refused(call(typ=3), "type")
    _refused(call(x_rows=1), "fewer rows")
    _refused(call(stride=4), "stride")
    _refused(call(n=-1), "range")
    _refused(call(n=1 << 32, x_rows=1 << 32), "one launch")
    _refused(call(x=ctypes.c_void_p(4098)), "aligned")
    _refused(call(x=ctypes.c_void_p(4097), typ=2), "aligned")


def test_c_ctc_align_refuses():
    lib = _lib.load()
    need = lib.tone_ctc_align_workspace(2, 6, 3)

    def call(x=P, typ=0, batch=2, frames=6, vocab=5, blank=4, tokens=P, most=3, lens=P, score=P, labels=P, spans=P, ws=P, wb=need):
        return lib.tone_ctc_align(0, x, typ, 5, 30, 0, None, batch, frames, vocab, blank, tokens, most, lens, P, score, None, labels, spans,
                                  ws, wb, None)
    _refused(call(x=None), "null")
    _refused(call(tokens=None), "null")
    _refused(call(lens=None), "null")
    _refused(call(score=None), "null")
    _refused(call(labels=None), "null")
    _refused(call(spans=None), "null")
    _refused(call(typ=-1), "type")
    _refused(call(blank=5), "blank")
    _refused(call(most=S.MAX_TOKENS + 1), "max_tokens")
    _refused(call(frames=-1), "range")
    _refused(call(ws=None), "workspace")
    _refused(call(wb=need - 1), "workspace")
    assert lib.tone_ctc_align_workspace(2, 6, S.MAX_TOKENS + 1) == -1


def test_c_sizes_past_one_launch_are_refused():
    """Sizes whose counts of threads pass 32 bits, or whose frame loops pass 31."""
    lib = _lib.load()
    big = 1 << 30
    _refused(lib.tone_frames_plan(0, P, 3, 4, 3, P, 8, 4, P, Q, P, P, P, P, P, P, 2, P, big, P, None), "one launch")
    _refused(lib.tone_frames_plan(0, P, 3, 4, 3, P, 8, 4, P, Q, P, P, P, P, P, P, 1 << 26, P, 2, P, None), "one launch")
    _refused(lib.tone_frames_slots(0, P, 3, 4, 3, 8, 4, P, P, P, P, 1, P, big, None), "one launch")
    _refused(lib.tone_frames_slots(0, P, 3, 4, 3, 8, 4, P, P, P, P, 1 << 24, P, 1, None), "one launch")
    _refused(lib.tone_frames_put(0, P, 0, 64, P, 1 << 29, 64, P, 0, 64, 9, None), "one launch")
    for vocab, n in ((35, 1 << 29), (64, 1 << 29), (65, 1 << 26)):
        _refused(lib.tone_token_scores(0, P, 0, vocab, n, None, n, vocab, None, 0, None, P, None, None, None, None), "one launch")
    for batch, frames in ((1, big), (1 << 22, 4)):
        _refused(lib.tone_ctc_align(0, P, 0, 5, 30, 0, None, batch, frames, 5, 4, P, 3, P, P, P, None, P, P, P, 1 << 60, None), "one launch")
    assert lib.tone_ctc_align_workspace(1, big, 3) == -1 < lib.tone_ctc_align_workspace(1, 1 << 29, 3)


def test_c_empty_calls_do_nothing():
    lib = _lib.load()
    assert lib.tone_frames_slots(0, None, 3, 4, 3, 8, 4, None, None, None, None, 0, None, 2, None) == 0
    assert lib.tone_frames_put(0, None, 0, 5, None, 0, 5, None, 0, 5, 9, None) == 0
    assert lib.tone_token_scores(0, None, 0, 5, 0, None, 0, 5, None, 0, None, None, None, None, None, None) == 0
    assert lib.tone_ctc_align(0, None, 0, 5, 0, 0, None, 0, 6, 5, 4, None, 3, None, None, None, None, None, None, None, 0, None) == 0


def _overlaps():
    """Rows and a pool in one buffer of (12, 16) entries: (src, pool, whether they share memory)."""
    b = torch.zeros((12, 16))
    h = torch.zeros((12, 32), dtype=torch.float16)
    flat = b.view(-1)
    return [
        (b[2:5, :5], b[:, :5], True), (b[:4, :5], b[4:, :5], False), (b[4:, :5], b[:4, :5], False), (b[:5, :5], b[4:, :5], True),
        (b[:, :5], b[:, 5:10], False), (b[:, 5:10], b[:, :5], False), (b[:, 4:9], b[:, :5], True), (b[:, 11:], b[:, :5], False),
        (b[3:4, 5:10], b[:, :5], False), (b[3:4, 4:9], b[:, :5], True), (b[3:4, 12:], b[:, :4], False), (b[::2, :5], b[:, 8:13], True),
        (flat[30:35].view(1, 5), b[:, :5], True), (b[:, :5], flat[21:26].view(1, 5), False), (b[:, :5], flat[18:23].view(1, 5), True),
        (b[:, :5], b[:0, :5], False), (b[:0, :5], b[:, :5], False), (b, b, True), (b[:3], b[3:], False), (h[:, :8], h[:, 8:16], False),
        (h[:, :8], h[:, 7:15], True), (h.view(torch.float32)[:, :8], h[:, 16:24], False), (h.view(torch.float32)[:, :8], h[:, 15:23], True),
        (h[:, :8], h.view(torch.float32)[:, 4:12], False), (h[:, 16:24], h.view(torch.float32)[:, :8], False), (h[:, 15:23], h.view(torch.float32)[:, :8], True),
    ]


@pytest.mark.parametrize("i", range(26))
def test_frames_put_refuses_rows_of_the_pool(i):
    """Rows in the memory of the pool would be read and written in no order; what lies beside them may be copied."""
    src, pool, meets = _overlaps()[i]
    mine = {a + j for r in range(src.shape[0]) for a in [src[r].data_ptr()] for j in range(src.shape[1] * src.element_size())}
    theirs = {a + j for r in range(pool.shape[0]) for a in [pool[r].data_ptr()] for j in range(pool.shape[1] * pool.element_size())}
    assert meets >= bool(mine & theirs)
    n = src.shape[0]
    with pytest.raises(ValueError, match="overlap" if meets else "on a GPU"):
        S.frames_put(src, torch.arange(n), pool)
    if not meets:
        return
    _refused(_lib.load().tone_frames_put(0, src.data_ptr(), S._type(src, ""), src.stride(0), P, n, src.shape[1], pool.data_ptr(),
                                         S._type(pool, ""), pool.stride(0), pool.shape[0], None), "overlaps")


def test_sizes_past_31_bits_are_refused():
    """The library takes them as int, and ctypes would pass on their low 32 bits: 2^32 + 35 entries as 35."""
    big = 2 ** 32 + 5
    meta = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    i32, i64 = (lambda *s: meta(*s, dtype=torch.int32)), (lambda *s: meta(*s, dtype=torch.int64))  # noqa: E731
    calls = [
        lambda: S.token_scores(meta(1, big)),
        lambda: S.frames_put(meta(1, big), i64(1), meta(1, big)),
        lambda: S.ctc_align(meta(1, big, 5), i32(1, 2), i32(1), i32(1), blank=4),
        lambda: S.ctc_align(meta(1, 6, big), i32(1, 2), i32(1), i32(1), blank=4),
        lambda: S.ctc_align(meta(9, 5), i32(1, 2), i32(1), i32(1), rows=i64(1, big), blank=4),
        lambda: S.ctc_align(meta(big, 6, 5), i32(big, 2), i32(big), i32(big), blank=4),
        lambda: S.frames_plan(**_plan_args(max_add=big)),
        lambda: S.frames_plan(**_plan_args(queue=i32(big))),
        lambda: S.frames_plan(**_plan_args(table=i32(big, 3))),
        lambda: S.frames_plan(**_plan_args(**{n: i32(big) for n in ("rows_in", "rows_out", "first", "length", "keep", "add")})),
        lambda: S.frames_slots(i32(4, 3), i32(2), i32(2), i32(2), i32(2), page_size=4, n_pages=big, max_count=2),
        lambda: S.frames_slots(i32(4, 3), i32(2), i32(2), i32(2), i32(2), page_size=big, n_pages=4, max_count=2),
        lambda: S.frames_slots(i32(4, 3), i32(2), i32(2), i32(2), i32(2), page_size=4, n_pages=4, max_count=big),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match=r"2\^31 - 1"):
            call()
            pytest.fail(f"call {i}")


def test_plans_of_too_many_requests_are_refused():
    """Every workgroup reads all requests, so the time grows with their square: the last sizes below 2^25 would take minutes."""
    n = S.MAX_BATCH + 1
    ids = torch.zeros(n, dtype=torch.int32)
    with pytest.raises(ValueError, match="requests"):
        S.frames_plan(**_plan_args(**{k: ids for k in ("rows_in", "rows_out", "first", "length", "keep", "add")}))
    lib = _lib.load()
    _refused(lib.tone_frames_plan(0, P, 3, 4, 3, P, 8, 4, P, Q, P, P, P, P, P, P, n, P, 2, P, None), "one launch")


def test_frames_put_of_a_pool_of_one_row():
    """Whose stride says nothing."""
    b = torch.zeros(20)
    one, zero = torch.zeros(1, dtype=torch.int64), b.as_strided((1, 5), (0, 1))
    for src, meets in ((b[5:10].view(1, 5), False), (b[4:9].view(1, 5), True), (b[2:7].as_strided((1, 5), (0, 1)), True), (b[5:10].as_strided((1, 5), (0, 1)), False), (b[6:16].view(2, 5), False)):
        with pytest.raises(ValueError, match="overlap" if meets else "on a GPU"):
            S.frames_put(src, one.repeat(src.shape[0]), zero)
    with pytest.raises(ValueError, match="overlap"):
        S.frames_put(b[:10].view(2, 5), one.repeat(2), zero)
