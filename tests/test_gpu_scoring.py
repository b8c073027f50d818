"""The phrase operators on a real MI355X against their 64-bit restatements (oracle/phrase_oracle.py): page plans and slot maps,
row puts, token scores, CTC alignment; odd sizes, masks, strides, streams, graphs, and the phrase path as a server runs it.

Tolerances.  EPS = 2^-24 is half a step of fp32.  A sum of n positive terms added one after another is off by at most n EPS of its
value; a term e^z (z <= 0) by 2 |z| EPS for the rounding of z and its product with log2 e, and 4 EPS for the exponential.
With s = sum e^z and mean = sum p |z|, ln s and the logprob are off by (n + 2 mean + 4) EPS plus their own last roundings, the
entropy's sum u / s by the same factor twice of its value (mean) and 2 mean for the rounded products.  n counts the longest chain
of additions that any split of the row over 64 lanes can have, V / 64 + 16.  One frame of the log-sum-exp over paths
adds at most 3 terms in 32 bits: an exponential of at most 4 EPS each, a sum of at most 3 and a logarithm of at most 1.1, so
4 + 2 + 2 + 4 EPS and in all below 16 EPS per frame; all else of it is 64 bits wide.  Best paths are 64 bits throughout and must agree exactly."""

import numpy as np
import pytest

import phrase_oracle as O

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


def S():
    from tone_amd import scoring
    return scoring


def _dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype))).cuda()


# --- pages ------------------------------------------------------------------------------------------------------------

class Pool:
    """Streams that hold frames, as a server's buffers have them: rows of the table in ping-pong, the free queue."""

    def __init__(self, rng, n, page, width, pages, head=0):
        self.page, self.width, self.n = page, width, n
        self.table = np.full((2 * n, width), -1, np.int32)
        self.queue = np.full(pages, -1, np.int32)
        self.queue[(head + np.arange(pages)) % pages] = rng.permutation(pages)
        self.cursors = np.array([head, head + pages], np.int64)
        self.first, self.length, self.par = np.zeros(n, np.int64), np.zeros(n, np.int64), np.zeros(n, np.int64)
        self.dev = [_dev(self.table), _dev(self.queue), _dev(self.cursors), torch.zeros(2, dtype=torch.int64, device="cuda")]

    def step(self, ids, keep, add, max_add, **kw):
        ids = np.asarray(ids)
        rows = 2 * ids + self.par[ids], 2 * ids + 1 - self.par[ids]
        first, length = self.first[ids], self.length[ids]
        t, q, cin, cout = self.dev
        slots, status = S().frames_plan(t, q, cin, cout, *(_dev(v, np.int32) for v in (*rows, first, length, keep, add)),
                                        page_size=self.page, max_add=max_add, **kw)
        assert int(status) == 0
        self.table, self.queue, self.cursors, want = O.plan(self.table, self.queue, self.cursors, *rows, first, length, keep, add, self.page, max_add)
        self.first[ids], self.length[ids], self.par[ids] = np.maximum(first, keep), length + add, 1 - self.par[ids]
        self.dev[2], self.dev[3] = cout, cin
        np.testing.assert_array_equal(slots.cpu().numpy(), want)
        np.testing.assert_array_equal(t.cpu().numpy(), self.table)
        np.testing.assert_array_equal(q.cpu().numpy(), self.queue)
        np.testing.assert_array_equal(cout.cpu().numpy(), self.cursors)
        return slots


@pytest.mark.parametrize("n,page,max_add,steps", [(1, 4, 3, 25), (1, 1, 10, 8), (7, 5, 10, 20), (70, 16, 13, 12), (300, 64, 10, 10),
                                                  (700, 7, 3, 6), (3, 48, 2000, 4), (9000, 64, 10, 2)])
def test_plan_over_steps(n, page, max_add, steps):
    """Random subsets of streams over many steps: ragged adds (zero among them), frames let go, streams closed, the queue wrapping."""
    rng = np.random.default_rng(n + page)
    window = 4 * max(page, max_add)
    width = -(-window // page) + 2
    p = Pool(rng, n, page, width, n * (width + -(-max_add // page) + 1) + 3, head=int(rng.integers(0, 1000)))
    for _ in range(steps):
        ids = rng.permutation(n)[: rng.integers(1, n + 1)]
        first, length = p.first[ids], p.length[ids]
        add = rng.integers(0, max_add + 1, len(ids))
        low = np.maximum(first, length + add - window)
        keep = np.where(rng.random(len(ids)) < 0.3, rng.integers(low, length + add + 1), low)
        p.step(ids, keep, add, max_add)


@pytest.mark.parametrize("n", [512, 513, 2048, 2049])
def test_plan_of_whole_batches(n):
    """Either side of the sizes at which the launch changes its shape; every stream in a call, then every other one."""
    rng = np.random.default_rng(n)
    p = Pool(rng, n, 6, 8, n * 9)
    p.step(rng.permutation(n), np.zeros(n, int), rng.integers(0, 12, n), 11)
    ids = np.arange(0, n, 2)
    p.step(ids, p.length[ids] // 2, rng.integers(0, 12, len(ids)), 11)
    p.step(np.arange(n), p.length - np.minimum(p.length - p.first, 3), np.full(n, 2), 2)


def test_plan_of_no_requests_and_no_frames():
    p = Pool(np.random.default_rng(0), 3, 4, 5, 20)
    slots = p.step(np.array([], int), np.array([], int), np.array([], int), 6)
    assert tuple(slots.shape) == (0, 6)
    p.step([0, 1], [0, 0], [6, 3], 6)
    p.step([0, 1, 2], [6, 2, 0], [0, 0, 0], 0)          # nothing new: one stream closed, one shortened


@pytest.mark.parametrize("what,bit", [("pages", 1), ("row", 2), ("first", 4), ("keep", 4), ("add", 4), ("row_id", 4), ("same_row", 4),
                                      ("cursors", 8), ("queue_short", 8)])
def test_plan_refused_on_the_device_changes_nothing(what, bit):
    """Every status bit: no page is taken or released, the rows keep their pages, every slot is -1."""
    p = Pool(np.random.default_rng(1), 4, 4, 5, 40, head=33)
    p.step([0, 1, 2, 3], [0, 0, 0, 0], [6, 9, 1, 4], 12)
    rows_in, rows_out = 2 * np.arange(4) + p.par, 2 * np.arange(4) + 1 - p.par
    first, length, keep, add = p.first.copy(), p.length.copy(), p.first.copy(), np.array([4, 4, 4, 4])
    t, q, cin, cout = p.dev
    if what == "pages":
        cin = _dev(np.array([p.cursors[1] - 2, p.cursors[1]]))
        add = np.array([6, 6, 6, 6])
    elif what == "row":
        add = np.array([4, 12, 4, 4])
    elif what == "first":
        first = first + np.array([0, 0, 30, 0])
    elif what == "keep":
        keep = keep + np.array([0, 0, 0, 30])
    elif what == "add":
        add = np.array([4, 4, 4, 13])
    elif what == "row_id":
        rows_out = rows_out + np.array([0, 0, 0, 100])
    elif what == "same_row":
        rows_out = np.where(np.arange(4) == 2, rows_in, rows_out)
    elif what == "cursors":
        cin = _dev(np.array([9, 3]))
    else:
        cin = _dev(np.array([5, 46]))
    before = t.clone(), q.clone()
    slots, status = S().frames_plan(t, q, cin, cout, *(_dev(v, np.int32) for v in (rows_in, rows_out, first, length, keep, add)),
                                    page_size=4, max_add=12)
    assert int(status) & bit and bool((slots == -1).all())
    assert torch.equal(cout, cin) and torch.equal(q, before[1])
    for b in range(4):
        assert torch.equal(t[int(rows_in[b])], before[0][int(rows_in[b])])
        if rows_out[b] < 8:
            assert torch.equal(t[int(rows_out[b])], before[0][int(rows_in[b])])


@pytest.mark.parametrize("cursors", [(0, 2 ** 63 - 1), (2 ** 62, 2 ** 63 - 1), (3, 2 ** 63 - 2), (-1, 5), (-2 ** 63, 2 ** 63 - 1), (0, 41)])
def test_plan_of_cursors_of_any_size(cursors):
    """Cursors that describe no queue, their difference plus the released pages beyond 63 bits among them."""
    p = Pool(np.random.default_rng(2), 4, 4, 5, 40)
    p.step([0, 1, 2, 3], [0, 0, 0, 0], [6, 9, 1, 4], 12)
    t, q, _, cout = p.dev
    cin = _dev(np.array(cursors))
    queue = q.clone()
    rows = (2 * np.arange(4) + p.par, 2 * np.arange(4) + 1 - p.par)
    slots, status = S().frames_plan(t, q, cin, cout, *(_dev(v, np.int32) for v in (*rows, p.first, p.length, p.length, np.zeros(4))),
                                    page_size=4, max_add=12)
    assert int(status) == 8 and bool((slots == -1).all())
    assert torch.equal(cout, cin) and torch.equal(q, queue)


def test_plan_near_the_largest_frame_numbers():
    """Frame numbers up to 2^31 - 1 (a stream that never closes) do not wrap."""
    p = Pool(np.random.default_rng(2), 2, 64, 6, 30)
    p.first[:] = p.length[:] = 2 ** 31 - 120
    p.step([0, 1], [0, 0], [100, 119], 119)
    p.step([1, 0], [0, 2 ** 31 - 100], [0, 10], 119)


@pytest.mark.parametrize("page", [1, 7, 64])
def test_slots_read_what_was_planned(page):
    rng = np.random.default_rng(page)
    n = 40
    width = 300 // page + 3
    p = Pool(rng, n, page, width, n * (width + 60 // page + 2))
    for _ in range(5):
        p.step(np.arange(n), np.maximum(p.first, p.length - 200), rng.integers(0, 60, n), 60)
    ids = rng.integers(0, n, 50)                        # the same stream may be read twice
    first = p.first[ids]
    begin = first + rng.integers(-3, 40, 50)
    count = rng.integers(0, 260, 50)
    rows = 2 * ids + p.par[ids]
    rows[:2] = (-1, 2 * n)                              # no such row
    got = S().frames_slots(p.dev[0], *(_dev(v, np.int32) for v in (rows, first, begin, count)), page_size=page,
                           n_pages=len(p.queue), max_count=250)
    want = O.slots(p.table, rows, first, begin, count, page, len(p.queue), 250)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    bad = p.dev[0].clone()
    bad[:, 1] = len(p.queue)                            # a page outside the pool, another below it
    bad[:, 0] = -5
    got = S().frames_slots(bad, *(_dev(v, np.int32) for v in (rows, first, begin, count)), page_size=page, n_pages=len(p.queue), max_count=250)
    np.testing.assert_array_equal(got.cpu().numpy(), O.slots(bad.cpu().numpy(), rows, first, begin, count, page, len(p.queue), 250))


@pytest.mark.parametrize("src", sorted(TYPES))
@pytest.mark.parametrize("pool", sorted(TYPES))
@pytest.mark.parametrize("n,vocab,pad", [(1, 35, 0), (10, 35, 0), (1000, 35, 3), (333, 1, 0), (257, 64, 0), (77, 1000, 5), (20, 8, 8), (3, 20000, 0)])
def test_put(src, pool, n, vocab, pad):
    g = torch.Generator(device="cuda").manual_seed(n + vocab)
    x = torch.randn((n, vocab + pad), device="cuda", generator=g).mul_(30).to(TYPES[src])[:, :vocab]
    x[0, 0] = float("nan")
    x[-1, vocab - 1] = float("-inf")
    wide = torch.full((2 * n + 3, vocab + pad), 7.0, dtype=TYPES[pool], device="cuda")
    slots = torch.randperm(2 * n + 3, device="cuda", generator=g)[:n].contiguous()
    slots[n // 2] = -1 if n > 2 else slots[n // 2]
    if n > 3:
        slots[1], slots[3] = 2 * n + 3, -(2 ** 40)      # outside: left out
    want = wide.clone()
    ok = (slots >= 0) & (slots < 2 * n + 3)
    want[slots[ok], :vocab] = x[ok].to(TYPES[pool])
    S().frames_put(x, slots, wide[:, :vocab])
    assert torch.equal(wide.nan_to_num(1e4), want.nan_to_num(1e4)) and torch.equal(wide.isnan(), want.isnan())


# --- scores -----------------------------------------------------------------------------------------------------------

def _check_scores(x, tokens, k, rows=None, **kw):
    """x: a device tensor (n, V); every output of every row."""
    r = S().token_scores(x, None if tokens is None else _dev(tokens, np.int32), k=k, rows=None if rows is None else _dev(rows, np.int64), **kw)
    v = x.shape[-1]
    data = x.float().cpu().numpy().astype(np.float64)
    n = len(rows) if rows is not None else data.shape[0]
    got = [None if t is None else t.cpu().numpy() for t in r]
    for i in range(n):
        at = i if rows is None else int(rows[i])
        tok = -1 if tokens is None else int(tokens[i])
        if not 0 <= at < data.shape[0]:
            want = (0.0, -1, 0.0, [(-1, -np.inf)] * k, 0.0)
        else:
            want = O.scores(data[at], tok, k)
        lp, rank, entropy, top, mean = want
        tol = (v / 64 + 16 + 2 * mean + 4) * EPS
        where = f"row {i}"
        if tokens is not None:
            _close(got[0][i], lp, tol + 4 * EPS * (abs(lp) if np.isfinite(lp) else 0), where)
            assert got[1][i] == rank, where
        _close(got[2][i], entropy, tol + mean * (2 * tol + 2 * EPS) + 4 * EPS * (1 + entropy), where)
        if k:
            assert got[4][i].tolist() == [t for t, _ in top], where
            for a, (_, b) in zip(got[3][i], top):
                _close(a, b, tol + 4 * EPS * (abs(b) if np.isfinite(b) else 0), where)
    return r


def _close(a, b, tol, where):
    # a difference of two fp32 values can lie outside fp32 (lowest - highest = -2 x the largest): rounded to the nearest
    # fp32 value that is an infinity, from (2 - 2^-24) 2^127 on
    if abs(b) >= (2 - 2.0 ** -24) * 2.0 ** 127:
        b = np.sign(b) * np.inf
    if not np.isfinite(b):
        assert a == b, (where, a, b)
    else:
        assert abs(float(a) - b) <= tol, (where, float(a), b, tol)


def _rows(n, v, dtype, seed, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((n, v), device="cuda", generator=g).mul_(scale).to(TYPES[dtype])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (1, 2, 0), (3, 35, 35), (10, 35, 8), (130, 35, 1), (65, 34, 5), (5, 63, 63), (5, 64, 64),
                                   (5, 65, 64), (7, 127, 16), (9, 512, 20), (6, 513, 9), (4, 1023, 64), (3, 2049, 10), (2, 5000, 33),
                                   (1, 20011, 50)])
def test_scores(dtype, n, v, k):
    rng = np.random.default_rng(n * v)
    x = _rows(n, v, dtype, n * v)
    _check_scores(x, rng.integers(-1, v + 1, n), k)


@pytest.mark.parametrize("n", [4097, 20000])
def test_scores_of_many_short_rows(n):
    """The forms for many rows: every whole output against float64 on the device's host copy, and a sample in full."""
    x = _rows(n, 35, "fp32", n)
    tokens = np.random.default_rng(n).integers(-1, 36, n)
    r = S().token_scores(x, _dev(tokens, np.int32), k=8)
    d = x.cpu().double()
    lp = torch.log_softmax(d, -1).numpy()
    given = (tokens >= 0) & (tokens < 35)
    want = np.where(given, lp[np.arange(n), tokens.clip(0, 34)], 0.0)
    assert np.abs(r.logprob.cpu().numpy() - want).max() <= 64 * EPS * (1 + np.abs(want).max())
    order = np.argsort(-d.numpy(), axis=1, kind="stable")
    np.testing.assert_array_equal(r.top_ids.cpu().numpy(), order[:, :8])
    rank = np.where(given, (order == tokens[:, None].clip(0, 34)).argmax(1), -1)
    np.testing.assert_array_equal(r.rank.cpu().numpy(), rank)
    np.testing.assert_allclose(r.top_logprob.cpu().numpy(), np.take_along_axis(lp, order[:, :8], 1), rtol=1e-6, atol=64 * EPS)
    entropy = -(np.exp(lp) * lp).sum(1)
    assert np.abs(r.entropy.cpu().numpy() - entropy).max() <= 200 * EPS
    sample = slice(0, 50)
    _check_scores(x[sample], tokens[sample], 8)


@pytest.mark.parametrize("v", [35, 64, 300, 4096, 9001])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_scores_of_equal_values(v, dtype):
    """Ties everywhere: the lowest index first, the rank counts lower indices; -0 and +0 are one value."""
    x = torch.randint(0, 3, (6, v), device="cuda", generator=torch.Generator(device="cuda").manual_seed(v)).to(TYPES[dtype])
    x[0] = 1.5
    x[1] = torch.where(torch.arange(v, device="cuda") % 2 == 0, -0.0, 0.0).to(TYPES[dtype])
    x[2] = torch.arange(v, device="cuda").div(v, rounding_mode="floor").to(TYPES[dtype])
    x[3] = (torch.arange(v, device="cuda") // 5).to(TYPES[dtype])          # ascending
    x[4] = -(torch.arange(v, device="cuda") // 5).to(TYPES[dtype])         # descending
    _check_scores(x, [v - 1, v // 2, 0, v // 3, 1, v - 1], min(v, 40))


@pytest.mark.parametrize("v", [5, 35, 64, 200, 3000, 9001])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_scores_of_masked_rows(v, dtype):
    """-inf entries, rows of nothing else, rows of the type's lowest value, one entry left, huge values."""
    low, high = torch.finfo(TYPES[dtype]).min, torch.finfo(TYPES[dtype]).max
    x = _rows(9, v, dtype, v)
    x[0] = float("-inf")
    x[1] = low
    x[2, : v - 1] = float("-inf")
    x[3, 1:] = low
    x[4, ::2] = float("-inf")
    x[5, : v // 2] = low
    x[6] = float("-inf")
    x[6, v // 2] = low                       # all of the probability on the lowest value
    x[7, 0] = high
    x[8, -1] = high
    x[8, 0] = low
    _check_scores(x, [0, v - 1, v - 1, 1, 0, 2, v // 2, 1, 0], min(v, 12))
    _check_scores(x, [v - 1, 0, 0, 0, 1, v - 1, 0, 0, v - 1], min(v, 64))


@pytest.mark.parametrize("v", [35, 64, 300, 9001])
def test_scores_of_rows_with_nan_or_infinity(v):
    """They make their own row NaN and no other, and the ids stay in range."""
    x = _rows(5, v, "fp32", v)
    clean = x.clone()
    x[1, v // 2] = float("nan")
    x[3, 0] = float("inf")
    r = S().token_scores(x, torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device="cuda"), k=4)
    for i in (1, 3):
        assert bool(r.entropy[i].isnan()) and bool(r.logprob[i].isnan())
    assert int(r.top_ids.min()) >= 0 and int(r.top_ids.max()) < v and int(r.rank.min()) >= 0 and int(r.rank.max()) < v
    want = S().token_scores(clean, torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device="cuda"), k=4)
    for a, b in zip(r, want):
        assert torch.equal(a[[0, 2, 4]], b[[0, 2, 4]])


@pytest.mark.parametrize("v", [35, 130, 2500])
def test_scores_through_a_slot_map(v):
    """Rows in any order, twice, none at all; x with spare columns; shapes kept."""
    rng = np.random.default_rng(v)
    x = _rows(50, v + 3, "fp32", v)[:, :v]
    rows = rng.integers(0, 50, 60)
    rows[[0, 7, 59]] = (-1, 50, 2 ** 40)
    _check_scores(x, rng.integers(0, v, 60), 6, rows)
    r = S().token_scores(x, _dev(rng.integers(0, v, (4, 15)), np.int32), k=6, rows=_dev(rows.reshape(4, 15), np.int64))
    assert tuple(r.logprob.shape) == (4, 15) and tuple(r.top_ids.shape) == (4, 15, 6)
    flat = S().token_scores(x, None, k=6, rows=_dev(rows, np.int64))
    assert torch.equal(flat.top_ids, r.top_ids.view(60, 6)) and flat.logprob is None and flat.rank is None
    assert torch.equal(flat.entropy, r.entropy.view(-1))


@pytest.mark.parametrize("v", [7, 35, 64, 65, 700])
def test_scores_of_nan_of_any_bits(v):
    """NaN with every bit set, of both signs, more than once in a row: ids stay distinct and in range, ranks in range."""
    bits = np.random.default_rng(v).standard_normal((40, v)).astype(np.float32).view(np.uint32)
    for i in range(40):
        at = np.random.default_rng(i).permutation(v)[: 1 + i % min(v, 9)]
        bits[i, at] = [0x7FFFFFFF, 0xFFFFFFFF, 0x7F800001, 0x7FC00000][i % 4]
    x = _dev(bits.view(np.int32), np.int32).view(torch.float32)
    tokens = _dev(np.arange(40) % v, np.int32)
    r = S().token_scores(x, tokens, k=min(v, 64))
    ids, rank = r.top_ids.cpu().numpy(), r.rank.cpu().numpy()
    assert ((ids >= 0) & (ids < v)).all() and all(len(set(row)) == len(row) for row in ids.tolist())
    assert ((rank >= 0) & (rank < v)).all()


def test_scores_of_no_rows():
    r = S().token_scores(torch.empty((0, 35), device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), k=3)
    assert tuple(r.top_ids.shape) == (0, 3) and r.entropy.numel() == 0
    r = S().token_scores(torch.empty((0, 35), device="cuda"), None, k=3, rows=torch.tensor([0, -1], device="cuda"))
    assert r.top_ids.tolist() == [[-1] * 3] * 2
    S().frames_put(torch.zeros((2, 35), device="cuda"), torch.tensor([0, 1], device="cuda"), torch.empty((0, 35), device="cuda"))
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    r = S().ctc_align(torch.empty((0, 35), device="cuda"), one.view(1, 1), one, one, rows=torch.zeros((1, 1), dtype=torch.int64, device="cuda"))
    assert r.score.item() == -np.inf and r.labels.tolist() == [[-1]]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n,v,k", [(40, 35, 8), (4, 700, 10), (1, 65537, 20), (3, 131072, 5)])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_scores_of_unaligned_rows(dtype, n, v, k, offset):
    """Rows that begin at any element: the same values as an aligned copy gives."""
    flat = _rows(1, n * (v + 1) + 8, dtype, v).view(-1)
    x = flat[offset : offset + n * (v + 1)].view(n, v + 1)[:, :v]
    tokens = torch.arange(n, dtype=torch.int32, device="cuda") * 7 % v
    a, b = S().token_scores(x, tokens, k=k), S().token_scores(x.contiguous(), tokens, k=k)
    assert torch.equal(a.top_ids, b.top_ids) and torch.equal(a.rank, b.rank)
    for u, w in ((a.logprob, b.logprob), (a.entropy, b.entropy), (a.top_logprob, b.top_logprob)):
        # both are within the tolerance of the exact value, whatever chains of additions they take
        assert float((u - w).abs().max()) <= 2 * (v / 64 + 40) * EPS * (1 + float(w.abs().max()))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("v", [40000, 65537, 131072])
def test_scores_of_one_wide_row(dtype, v):
    """A single row over a wide vocabulary, random and in ascending order."""
    x = _rows(2, v, dtype, v)
    x[1] = x[1].float().sort().values.to(TYPES[dtype])
    for i in range(2):
        _check_scores(x[i : i + 1], [v // 3], 32)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("v,k", [(2500, 1), (9001, 10), (9001, 64), (40000, 20)])
def test_scores_of_ordered_rows(v, k, dtype):
    """Rows that ascend, descend, ascend from the middle on, ascend lane by lane, and ascend with NaN-free masks in between."""
    x = _rows(5, v, dtype, v + k).float().sort(-1)[0]
    x[1] = x[1].flip(0)
    x[2] = x[2].roll(v // 2)
    x[3] = x[3][torch.arange(v, device="cuda").mul(97).remainder(v).argsort()]
    x[4, ::3] = float("-inf")
    _check_scores(x.to(TYPES[dtype]), [v - 1, 0, v // 2, v // 3, v - 2], k)


def test_scores_are_the_same_every_time():
    x = _rows(3, 131072, "bf16", 1)
    tokens = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")
    a = S().token_scores(x, tokens, k=20)
    for _ in range(5):
        assert all(torch.equal(u, w) for u, w in zip(a, S().token_scores(x, tokens, k=20)))


# --- alignment --------------------------------------------------------------------------------------------------------

def _ctc(rng, b, f, most, vocab, blank, peaked=True):
    """Log probabilities (b, f, vocab), tokens (b, most) with repeats, lengths (one at full size)."""
    tlen = rng.integers(0, most + 1, b)
    flen = rng.integers(0, f + 1, b)
    tlen[0], flen[0] = most, f
    tokens = rng.integers(0, vocab, (b, most))
    tokens = np.where(tokens == blank, (tokens + 1) % vocab, tokens)
    rep = rng.random((b, most)) < 0.2
    for i in range(1, most):
        tokens[:, i] = np.where(rep[:, i], tokens[:, i - 1], tokens[:, i])
    x = rng.normal(0, 1.5, (b, f, vocab))
    if peaked:
        for i in range(b):
            for j in range(tlen[i]):
                if flen[i]:
                    x[i, int((j + 0.5) * flen[i] / tlen[i]), tokens[i, j]] += 5
    x = x - np.log(np.exp(x).sum(-1, keepdims=True))
    return x, tokens.astype(np.int32), tlen.astype(np.int32), flen.astype(np.int32)


def _check_align(x, tokens, tlen, flen, blank, total, data=None, **kw):
    r = S().ctc_align(x, _dev(tokens), _dev(tlen), _dev(flen), blank=blank, total=total, **kw)
    data = x.float().cpu().numpy().astype(np.float64) if data is None else data
    score, labels, spans = r.score.cpu().numpy(), r.labels.cpu().numpy(), r.spans.cpu().numpy()
    b, most = tokens.shape
    for i in range(b):
        n, f = int(np.clip(tlen[i], 0, most)), int(np.clip(flen[i], 0, labels.shape[1]))
        w_score, w_total, w_labels, w_spans = O.align(data[i, :f], tokens[i, :n].tolist(), blank)
        assert score[i] == np.float32(w_score), (i, score[i], w_score)
        alive = w_labels is not None
        assert labels[i].tolist() == (w_labels if alive else [-1] * f) + [-1] * (labels.shape[1] - f), i
        assert spans[i].tolist() == (w_spans if alive else [[-1, -1]] * n) + [[-1, -1]] * (most - n), i
        if total:
            _close(r.total[i].item(), w_total, (f + 1) * 16 * EPS + EPS * abs(w_total) if np.isfinite(w_total) else 0, f"sequence {i}")
    return r


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("total", [False, True])
@pytest.mark.parametrize("b,f,most,vocab", [(1, 1, 1, 2), (3, 1, 2, 5), (4, 2, 1, 35), (5, 7, 3, 35), (6, 33, 9, 35), (3, 64, 31, 35), (3, 65, 32, 35),
                                            (2, 130, 33, 100), (2, 70, 63, 35), (2, 129, 64, 36), (2, 200, 100, 40), (1, 300, 127, 35)])
def test_align(dtype, total, b, f, most, vocab):
    rng = np.random.default_rng(b * f + most)
    blank = vocab - 1 if most % 2 else 0
    x, tokens, tlen, flen = _ctc(rng, b, f, most, vocab, blank)
    _check_align(_dev(x).to(TYPES[dtype]), tokens, tlen, flen, blank, total)


@pytest.mark.parametrize("f,most", [(700, 300), (520, 255), (300, 256), (2100, 700), (64, 700), (1400, 640), (2100, 1000)])
def test_align_long(f, most):
    """Long sequences; too few frames for the tokens among them."""
    rng = np.random.default_rng(f)
    x, tokens, _, _ = _ctc(rng, 2, f, most, 35, 34)
    lens = np.array([[most, f], [most // 2, f - f // 3]], np.int32)
    _align_by_rows(rng, x, tokens, lens)


@pytest.mark.parametrize("most", [63, 64, 159, 160, 415, 416, 799, 800, 1183, 1184])
def test_align_either_side_of_a_shape(most):
    """Token counts around those at which the launch takes more waves or more states per lane."""
    rng = np.random.default_rng(most)
    f = most + most // 4 + 40
    x, tokens, _, _ = _ctc(rng, 2, f, most, 35, 34)
    _align_by_rows(rng, x, tokens, np.array([[most, f], [most - 1, f - 1]], np.int32))


def _align_by_rows(rng, x, tokens, lens):
    """Against the definition evaluated a frame at a time over all states (the oracle's loops are too slow here)."""
    b, f, vocab = x.shape
    x32 = x.astype(np.float32).astype(np.float64)
    r = S().ctc_align(_dev(x, np.float32), _dev(tokens), _dev(lens[:, 0].copy()), _dev(lens[:, 1].copy()), blank=34, total=True)
    for i in range(b):
        n, fr = int(lens[i, 0]), int(lens[i, 1])
        lab = np.full(2 * n + 1, 34)
        lab[1::2] = tokens[i, :n]
        jump = np.zeros(2 * n + 1, bool)
        jump[3::2] = lab[3::2] != lab[1:-2:2]
        v = np.where(np.arange(2 * n + 1) < 2, x32[i, 0, lab], -np.inf)
        w = v.copy()
        back = np.zeros((fr, 2 * n + 1), int)
        for t in range(1, fr):
            for a in (0, 1):
                src = w if a else v
                c = np.full((3, 2 * n + 1), -np.inf)
                c[0], c[1, 1:], c[2, 2:] = src, src[:-1], np.where(jump[2:], src[:-2], -np.inf)
                if a:
                    h = np.maximum(c.max(0), -1e300)
                    with np.errstate(divide="ignore"):
                        w = h + np.log(np.exp(c - h).sum(0)) + x32[i, t, lab]
                else:
                    back[t] = c.argmax(0)
                    v = c.max(0) + x32[i, t, lab]
        s = 2 * n - 1 if v[2 * n - 1] > v[2 * n] else 2 * n
        assert r.score[i].item() == np.float32(v[s])
        if v[s] == -np.inf:
            assert bool((r.labels[i] == -1).all()) and bool((r.spans[i] == -1).all()) and r.total[i].item() == -np.inf
            continue
        want = np.full(f, -1)
        for t in range(fr - 1, -1, -1):
            want[t] = lab[s]
            s -= back[t, s]
        np.testing.assert_array_equal(r.labels[i].cpu().numpy(), want)
        tot = np.logaddexp(w[2 * n], w[2 * n - 1])
        _close(r.total[i].item(), tot, (fr + 1) * 16 * EPS + EPS * abs(tot), f"sequence {i}")


def test_align_edges():
    """No frames, no tokens, more tokens than frames, repeats that need a blank, a token outside, the blank as a token."""
    rng = np.random.default_rng(0)
    x, _, _, _ = _ctc(rng, 9, 6, 4, 5, 4, peaked=False)
    tokens = np.array([[0, 1, 2, 3], [0, 0, 0, 0], [1, 1, 1, 1], [0, 1, 2, 3], [0, 9, 1, 1], [0, 4, 1, 1], [0, -1, 1, 1], [2, 2, 2, 0], [3, 3, 1, 1]], np.int32)
    tlen = np.array([4, 0, 4, 0, 2, 2, 2, 9, 2], np.int32)      # 9: clamped to 4
    flen = np.array([0, 0, 6, 3, 6, 6, 6, 99, 3], np.int32)     # 99: clamped to 6
    _check_align(_dev(x, np.float32), tokens, tlen, flen, 4, True)
    tlen[0], flen[0] = -3, -1
    _check_align(_dev(x, np.float32), tokens, tlen, flen, 4, False)


def test_align_of_equal_scores_prefers_to_stay():
    """Constant rows: every path has the same score, and the tie rule alone decides."""
    for f, tokens in ((5, [0, 1]), (7, [0, 0]), (9, [0, 1, 1, 2]), (4, [0]), (40, [0, 1, 0, 2, 2, 1])):
        x = np.full((1, f, 4), -2.0)
        _check_align(_dev(x, np.float32), np.array([tokens], np.int32), np.array([len(tokens)], np.int32), np.array([f], np.int32), 3, True)


def test_align_with_nan_and_infinity():
    """NaN, +inf and -inf entries all close their label in that frame."""
    rng = np.random.default_rng(4)
    x, tokens, tlen, flen = _ctc(rng, 6, 30, 6, 8, 7)
    x[1, 3, :] = np.nan
    x[2, rng.random((30, 8)) < 0.2] = -np.inf
    x[3, rng.random((30, 8)) < 0.2] = np.inf
    x[4, rng.random((30, 8)) < 0.2] = np.nan
    x[5] = -np.inf
    tlen[:], flen[:] = 4, 30
    _check_align(_dev(x, np.float32), tokens, tlen, flen, 7, True)


@pytest.mark.parametrize("most", [2, 60, 300])
def test_align_of_entries_that_are_no_log_probabilities(most):
    """Large positive entries: the score is their sum, the total ends at 2^29 ln 2 instead of wrapping around."""
    frames = 40000
    x = torch.full((1, 1, 9), 5.9e4, device="cuda").expand(1, frames, 9)
    tokens = _dev((np.arange(most) % 8)[None], np.int32)
    r = S().ctc_align(x, tokens, _dev([most], np.int32), _dev([frames], np.int32), blank=8, total=True)
    assert float(r.score) == np.float32(5.9e4 * frames)
    assert 3.7e8 < float(r.total) < 3.8e8
    r = S().ctc_align(x[:, :1000], tokens, _dev([most], np.int32), _dev([1000], np.int32), blank=8, total=True)
    assert 5.9e7 <= float(r.total) <= 5.9e7 + 1000 * np.log(3) + 5.9e7 * 2 * EPS


def test_align_reads_any_strides_and_slot_maps():
    rng = np.random.default_rng(5)
    x, tokens, tlen, flen = _ctc(rng, 5, 50, 12, 35, 34)
    base = _check_align(_dev(x, np.float32), tokens, tlen, flen, 34, True)
    x32 = x.astype(np.float32)
    wide = torch.full((50, 5, 40), float("nan"), device="cuda")
    wide[:, :, :35] = _dev(x32.transpose(1, 0, 2))
    again = S().ctc_align(wide.transpose(0, 1)[:, :, :35], _dev(tokens), _dev(tlen), _dev(flen), total=True)
    assert all(torch.equal(a, b) for a, b in zip(base, again))
    pool = torch.full((700, 37), float("nan"), device="cuda")
    rows = rng.permutation(700)[:250].reshape(5, 50)
    pool[_dev(rows), :35] = _dev(x32)
    rows_d = torch.where(torch.arange(50, device="cuda") < _dev(flen)[:, None], _dev(rows), -1)
    again = S().ctc_align(pool[:, :35], _dev(tokens), _dev(tlen), _dev(flen), rows=rows_d, total=True)
    assert all(torch.equal(a, b) for a, b in zip(base, again))
    # one phrase's frames under five texts: an expanded batch
    same = S().ctc_align(_dev(x32[:1]).expand(5, 50, 35), _dev(tokens), _dev(tlen), _dev(np.full(5, 50, np.int32)), total=True)
    _check_align(_dev(np.repeat(x32[:1], 5, 0)), tokens, tlen, np.full(5, 50, np.int32), 34, True)
    full = S().ctc_align(_dev(np.repeat(x32[:1], 5, 0)), _dev(tokens), _dev(tlen), _dev(np.full(5, 50, np.int32)), total=True)
    assert all(torch.equal(a, b) for a, b in zip(same, full))
    # frames without a row are closed: no path crosses them
    rows_d[0, 10] = 700
    lost = S().ctc_align(pool[:, :35], _dev(tokens), _dev(tlen), _dev(flen), rows=rows_d, total=True)
    assert lost.score[0].item() == -np.inf and lost.total[0].item() == -np.inf and torch.equal(lost.score[1:], base.score[1:])


def test_align_of_an_empty_batch_and_no_frames():
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    r = S().ctc_align(torch.empty((0, 5, 35), device="cuda"), z(0, 3), z(0), z(0), total=True)
    assert r.score.numel() == 0 and tuple(r.spans.shape) == (0, 3, 2)
    r = S().ctc_align(torch.empty((2, 0, 35), device="cuda"), z(2, 3), _dev(np.array([0, 2], np.int32)), z(2), total=True)
    assert r.score.tolist() == [0.0, -np.inf] and r.total.tolist() == [0.0, -np.inf] and bool((r.spans == -1).all())
    r = S().ctc_align(_rows(8, 35, "fp32", 1).view(2, 4, 35).log_softmax(-1), z(2, 0), z(2), _dev(np.array([4, 0], np.int32)))
    assert r.labels.tolist() == [[34] * 4, [-1] * 4] and r.score[1].item() == 0.0


# --- streams, graphs, far offsets -------------------------------------------------------------------------------------

def _small_calls():
    """One call of each operator on fixed inputs: name -> (function of a stream, inputs that a replay may change)."""
    rng = np.random.default_rng(9)
    x, tokens, tlen, flen = _ctc(rng, 4, 60, 14, 35, 34)
    xd, td, ld, fd = _dev(x, np.float32), _dev(tokens), _dev(tlen), _dev(flen)
    wide = _rows(2, 70001, "bf16", 3)
    wt = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    flat = torch.randint(0, 35, (4, 60), dtype=torch.int32, device="cuda")
    pool = torch.zeros((300, 35), device="cuda")
    slots = torch.randperm(300, device="cuda")[:240].view(4, 60).contiguous()
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(8, 5).contiguous()
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    queue, cin, cout = torch.arange(100, 160, dtype=torch.int32, device="cuda") % 60, torch.tensor([7, 30], device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    req = [i(0, 2, 4, 6), i(1, 3, 5, 7), i(0, 3, 9, 0), i(0, 8, 20, 40), i(0, 5, 9, 40), i(9, 3, 0, 0)]
    return {
        "plan": (lambda st: S().frames_plan(table, queue, cin, cout, *req, page_size=16, max_add=10, stream=st) + (table, queue, cout), []),
        "slots": (lambda st: (S().frames_slots(table, req[0], req[2], req[2], req[3], page_size=16, n_pages=60, max_count=50, stream=st),), []),
        "put": (lambda st: (S().frames_put(xd, slots, pool, stream=st), pool)[1:], [xd]),
        "scores": (lambda st: S().token_scores(xd, flat, k=5, stream=st), [xd]),
        "scores-wide": (lambda st: S().token_scores(wide, wt, k=20, stream=st), [wide]),
        "align": (lambda st: S().ctc_align(xd, td, ld, fd, total=True, stream=st), [xd]),
    }


@pytest.mark.parametrize("name", ["plan", "slots", "put", "scores", "scores-wide", "align"])
def test_on_another_stream(name):
    fn, _ = _small_calls()[name]
    want = [t.clone() for t in fn(None)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = fn(s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("name", ["plan", "slots", "put", "scores", "scores-wide", "align"])
def test_captured_and_replayed(name):
    """Two graphs of one call, replayed in turn with changed inputs and eager calls between: each agrees with the eager result."""
    fn, inputs = _small_calls()[name]
    fn(None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = fn(None)
        graphs.append((g, out))
    torch.cuda.synchronize()
    for step in range(4):
        for t in inputs:
            t.add_(torch.randn_like(t, dtype=torch.float32).mul_(0.1).to(t.dtype))
        want = [t.clone() for t in fn(None)]
        torch.cuda.synchronize()
        for g, out in (graphs if step % 2 else graphs[::-1]):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, out)), f"replay {step}"


def test_two_calls_at_once():
    """Calls on two streams with their own outputs do not touch each other."""
    calls = _small_calls()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for name in ("scores-wide", "align"):
        fn = calls[name][0]
        want = [t.clone() for t in fn(None)]
        torch.cuda.synchronize()
        got = [fn(s) for _ in range(8) for s in (s1, s2)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for out in got for a, b in zip(want, out))


def test_rows_past_32_bit_offsets():
    """A pool of more than 2^31 entries: rows written and read at its end (and none at the offsets' low 32 bits)."""
    n = 2 ** 31 // 35 + 1000
    pool = torch.zeros((n, 35), dtype=torch.bfloat16, device="cuda")
    x = _rows(40, 35, "bf16", 8).float().log_softmax(-1).to(torch.bfloat16)
    rows = torch.arange(n - 40, n, device="cuda")
    S().frames_put(x, rows, pool)
    assert torch.equal(pool[n - 40 :], x) and not bool(pool[:2000].any())
    tokens = torch.arange(40, dtype=torch.int32, device="cuda") % 34
    a, b = S().token_scores(pool, tokens, k=5, rows=rows), S().token_scores(x, tokens, k=5)
    assert all(torch.equal(u, w) for u, w in zip(a, b))
    one = torch.tensor([6], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40], dtype=torch.int32, device="cuda")
    text = tokens[None, :6].contiguous()
    a = S().ctc_align(pool, text, one, lens, rows=rows[None].contiguous(), total=True)
    b = S().ctc_align(x[None], text, one, lens, total=True)
    assert all(torch.equal(u, w) for u, w in zip(a, b))
    far = torch.zeros((2, n * 35), dtype=torch.bfloat16, device="cuda")[:, -35:]      # two rows 2^31 entries apart
    far[1] = x[3]
    r = S().token_scores(far, torch.tensor([1, 2], dtype=torch.int32, device="cuda"), k=5)
    assert torch.equal(r.top_ids[1], S().token_scores(x[3:4], None, k=5).top_ids[0])


def test_the_phrase_path():
    """The operators as a server runs them: frames put page by page over many steps, a phrase read back, aligned and scored."""
    rng = np.random.default_rng(6)
    n, page, steps = 5, 16, 12
    p = Pool(rng, n, page, 12, 60, head=11)
    x, tokens, tlen, _ = _ctc(rng, n, 10 * steps, 20, 35, 34)
    x32 = _dev(x, np.float32)
    pool = torch.full((60 * page, 35), float("nan"), device="cuda")
    for t in range(steps):
        slots = p.step(np.arange(n), p.first, np.full(n, 10), 10)
        S().frames_put(x32[:, 10 * t : 10 * t + 10].contiguous(), slots, pool)
    begin, count = np.array([0, 5, 17, 100, 60]), np.array([120, 90, 64, 20, 1])
    rows = S().frames_slots(p.dev[0], *(_dev(v, np.int32) for v in (2 * np.arange(n) + p.par, p.first, begin, count)), page_size=page, n_pages=60,
                            max_count=120)
    data = np.zeros((n, 120, 35))
    for i in range(n):
        data[i, : count[i]] = x[i, begin[i] : begin[i] + count[i]].astype(np.float32)
    a = _check_align(pool, tokens, tlen, count.astype(np.int32), 34, True, data=data, rows=rows)
    r = S().token_scores(pool, a.labels, k=3, rows=rows)
    labels = a.labels.cpu().numpy()
    for i in range(n):
        for t in range(120):
            if labels[i, t] < 0:
                assert r.logprob[i, t].item() == 0.0
            else:
                assert abs(r.logprob[i, t].item() - data[i, t, labels[i, t]]) <= 1e-5


# --- the store and the pipeline ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("page,dtype", [(64, "fp32"), (7, "fp16"), (1, "bf16")])
def test_store_against_a_list_of_rows(page, dtype):
    """Random appends, ranges read, streams released: every frame a stream holds reads back as it was put."""
    rng = np.random.default_rng(page)
    n, t, most = 9, 13, 90
    store = S().FrameStore(n, most, page_size=page, n_pages=n * (-(-most // page) + 1) - 3, vocab=6, dtype=TYPES[dtype])
    held = [np.zeros((0, 6)) for _ in range(n)]
    first = np.zeros(n, int)
    for step in range(40):
        ids = rng.permutation(n)[: rng.integers(1, n + 1)]
        rows = _rows(len(ids) * t, 6, dtype, step).view(len(ids), t, 6)
        counts = rng.integers(0, t + 1, len(ids)) if step % 2 else None
        end = first[ids] + [len(held[i]) for i in ids] + (t if counts is None else counts)
        keep = np.maximum(first[ids], end - rng.integers(0, most + 1, len(ids)))
        store.append(rows, ids, keep=keep, counts=counts)
        for j, i in enumerate(ids):
            new = rows[j, : (t if counts is None else counts[j])].float().cpu().numpy()
            held[i] = np.concatenate([held[i], new])[keep[j] - first[i] :]
            first[i] = keep[j]
        if step % 7 == 3:
            gone = rng.permutation(n)[:2]
            store.release(gone)
            for i in gone:
                held[i], first[i] = held[i][:0], 0
        pages = sum(-(-(first[i] + len(held[i])) // page) - first[i] // page for i in range(n) if len(held[i]))
        assert store.free_pages == store.n_pages - pages
        ids = rng.integers(0, n, 5)
        count = np.array([rng.integers(0, len(held[i]) + 1) for i in ids])
        begin = np.array([first[i] + rng.integers(0, len(held[i]) - c + 1) for i, c in zip(ids, count)])
        slots = store.slots(ids, begin, count)
        assert slots.shape == (5, count.max())
        for j, (i, b, c) in enumerate(zip(ids, begin, count)):
            assert bool((slots[j, c:] == -1).all())
            np.testing.assert_array_equal(store.pool[slots[j, :c]].float().cpu().numpy(), held[i][b - first[i] : b - first[i] + c])


def test_store_refuses_and_stays_as_it_was():
    store = S().FrameStore(3, 32, page_size=8, n_pages=6, vocab=5)
    rows = _rows(30, 5, "fp32", 1).view(3, 10, 5)
    slots = store.append(rows, [2, 0, 1])                # 2 pages each: all of them
    before = store.pool.clone(), store._table.clone(), store._queue.clone(), store._cursors.clone(), store.first.copy(), store.length.copy()
    with pytest.raises(RuntimeError, match="out of pages"):
        store.append(rows, [0, 1, 2])
    for bad in (dict(ids=[0, 0, 1]), dict(ids=[0, 1, 3]), dict(ids=[0, 1]), dict(ids=[0, 1, 2], keep=[0, 0, 21]),
                dict(ids=[0, 1, 2], keep=[-1, 0, 0]), dict(ids=[0, 1, 2], counts=[11, 0, 0]), dict(ids=[0, 1, 2], counts=[1, 1])):
        with pytest.raises(ValueError):
            store.append(rows, **bad)
    with pytest.raises(ValueError):
        store.append(_rows(90, 5, "fp32", 1).view(3, 30, 5), [0, 1, 2])       # more than a stream holds
    with pytest.raises(ValueError):
        store.append(rows.cpu(), [0, 1, 2])
    with pytest.raises(ValueError):
        store.slots([0], [5], [6])
    now = store.pool, store._table, store._queue, store._cursors
    assert all(torch.equal(a, b) for a, b in zip(before, now)) and (store.first == before[4]).all() and (store.length == before[5]).all()
    with pytest.raises(RuntimeError, match="out of pages"):                  # pages let go by a call are free from the next on
        store.append(rows[:2], [0, 1], keep=[16, 20])
    store.append(rows[1:2], [1], keep=[10], counts=[0])   # none of stream 1
    assert store.free_pages == 2
    store.append(rows[:1], [0], keep=[16])                # frames 16 .. 19 of stream 0
    assert store.free_pages == 3 and torch.equal(store.pool[store.slots([0], [16], [4])[0]], rows[0, 6:])
    assert torch.equal(store.pool[slots[0]], rows[0])     # stream 2 as it was
    for bad in (dict(n_streams=0, max_frames=8), dict(n_streams=1, max_frames=0), dict(n_streams=1, max_frames=8, page_size=0),
                dict(n_streams=1, max_frames=8, n_pages=0), dict(n_streams=1, max_frames=8, dtype=torch.int8)):
        with pytest.raises(ValueError):
            S().FrameStore(**bad)


def test_store_refuses_capture_and_stays_as_it_was():
    store = S().FrameStore(2, 20, page_size=4, vocab=5)
    rows = _rows(2, 15, "fp32", 3).view(2, 3, 5)
    store.append(rows, [0, 1])
    out = torch.zeros(4, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out += 1
        for call in (lambda: store.append(rows, [0, 1]), lambda: store.release([0]), lambda: store.slots([0], [0], [3])):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    g.replay()
    assert list(store.length) == [3, 3] and store.free_pages == store.n_pages - 2
    slots = store.slots([0, 1], [0, 0], [3, 3])
    assert torch.equal(store.pool[slots], rows)


def test_store_dropped_while_its_calls_are_under_way():
    """Its buffers go back to the allocator only when the stream of its calls has passed them."""
    s = torch.cuda.Stream()
    rows = _rows(8, 35 * 400, "fp32", 1).view(8, 400, 35)
    torch.cuda.synchronize()
    store = S().FrameStore(8, 400, vocab=35)
    size = store.pool.shape
    big = torch.zeros(64 << 20, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            big += 1                          # holds the store's work back
    store.append(rows, list(range(8)), stream=s)
    del store
    taken = [torch.zeros(size, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    assert all(not bool(t.any()) for t in taken)


def test_store_on_a_stream_of_its_own():
    store, want = S().FrameStore(2, 64, page_size=8, vocab=5), S().FrameStore(2, 64, page_size=8, vocab=5)
    side = torch.cuda.Stream()
    rows = _rows(40, 5, "fp32", 1).view(2, 20, 5)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        store.append(rows, [1, 0], stream=side)
        want.append(rows, [1, 0])
    slots = store.slots([0, 1], [3, 0], [50, 60], stream=side)
    side.synchronize()
    assert torch.equal(slots, want.slots([0, 1], [3, 0], [50, 60])) and torch.equal(store.pool, want.pool)


@pytest.fixture(scope="module")
def session():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    from tone_amd.model import ToneSession
    from tone_amd.weights import synthetic_weights
    s = ToneSession(synthetic_weights(0), device=0, precision="fp32", max_batch=2)
    yield s
    s.close()


def _speech(seed, chunks):
    """Noise with pauses, so that phrases end inside the audio."""
    rng = np.random.default_rng(seed)
    x = np.clip(rng.normal(0, 2500, (chunks, 2400)), -32768, 32767).astype(np.int32)
    x[chunks // 3 : chunks // 3 + 4] = 0
    return x


class _Fixed:
    """A host decoder that answers one text whatever it hears."""

    def __init__(self, text):
        self.text = text

    def forward(self, logprobs):
        assert logprobs.dtype == np.float32 and logprobs.shape[1] == 35
        return self.text


@pytest.mark.parametrize("text", [None, "да нет", "", "\u0434\u0430!", "\u0430" * 300])
def test_pipeline_scores_its_phrases(session, text, monkeypatch):
    """StreamingGreedyPipeline(scores=...): the phrases of the plain pipeline, with the scores that the oracle gives for their
    text on the same frames; more streams than a device batch, closed at different times."""
    from tone_amd import pipeline as P
    decoder = lambda: None if text is None else _Fixed(text)  # noqa: E731
    chunks = {0: _speech(1, 14), 1: _speech(2, 9), 2: _speech(3, 14)}
    plain, scored = P.StreamingGreedyPipeline(session, 3, decoder()), P.StreamingGreedyPipeline(session, 3, decoder(), scores=4)
    # the rows as the pipeline puts them (a step's last bits depend on its batch size, so no replay of one stream gives them)
    kept, put = [], S().frames_put
    monkeypatch.setattr(S(), "frames_put", lambda x, slots, pool, stream=None: (kept.append(x.cpu().numpy()), put(x, slots, pool, stream))[1])
    found, rows_of = {}, {i: [] for i in chunks}
    for name, pipe in (("plain", plain), ("scored", scored)):
        slots = {i: pipe.open_stream() for i in chunks}
        got = {i: [] for i in chunks}
        for step in range(14):
            on = [i for i in chunks if step < len(chunks[i])]
            kept.clear()
            out = pipe.forward(np.stack([chunks[i][step] for i in on]), [slots[i] for i in on], [step == len(chunks[i]) - 1 for i in on])
            for j, (i, phrases) in enumerate(zip(on, out)):
                got[i] += phrases
                if name == "scored":
                    rows_of[i].append(np.concatenate(kept)[j])
            for i in on:
                if step == len(chunks[i]) - 1:
                    pipe.close_stream(slots[i])
        found[name] = got
    assert scored._store.free_pages == scored._store.n_pages
    assert sum(len(p) for p in found["plain"].values()) > 2
    for i, audio in chunks.items():
        rows = np.concatenate(rows_of[i]).astype(np.float64)
        shift = 0.33 + 2400 / 8000
        assert [(p.text, p.start_time, p.end_time) for p in found["scored"][i]] == [(p.text, p.start_time, p.end_time) for p in found["plain"][i]]
        # the phrases' frames, from the splitter run on the same rows
        st, spans = P.FrameSplitterState(), []
        speech = np.exp(rows[:, 33]) + np.exp(rows[:, 34]) <= 0.9
        for k in range(len(audio)):
            before = st.offset
            out, st = P.split_frames(np.arange(10 * k, 10 * k + 10), speech[10 * k : 10 * k + 10], st, is_last=k == len(audio) - 1)
            spans += [(max(before, s - 3), len(t)) for t, s, _ in out]
        assert len(spans) == len(found["scored"][i])
        for p, (begin, count) in zip(found["scored"][i], spans):
            ids = P.text_tokens(p.text)
            if ids is None:
                assert p.score is None and p.tokens == []
                continue
            score, total, labels, tok = O.align(rows[begin : begin + count], ids, 34)
            if labels is None:
                assert p.score is None and p.total is None and p.tokens == []
                continue
            assert p.score == float(np.float32(score)) and abs(p.total - total) <= (count + 1) * 16 * EPS + EPS * abs(total)
            assert [t.text for t in p.tokens] == list(p.text)
            for t, (a, b) in zip(p.tokens, tok):
                assert t.start_time == max(0, round((begin + a) * 0.03 - shift, 2)) and t.end_time == max(0, round((begin + b) * 0.03 - shift, 2))
                lp = rows[begin + a : begin + b, P.LABELS.index(t.text)]
                assert abs(t.logprob - lp.mean()) <= 1e-5
                best = rows[begin + a + int(np.argmax(lp))]
                order = np.argsort(-best, kind="stable")[:4]
                assert [v for v, _ in t.alternatives] == [P.LABELS[o] if o < 34 else "" for o in order]
                assert np.abs(np.array([v for _, v in t.alternatives]) - best[order]).max() <= 1e-5
                assert abs(t.entropy + (np.exp(best) * best).sum()) <= 1e-4


def test_pipeline_out_of_pages_leaves_its_streams_as_they_were(session):
    from tone_amd import pipeline as P
    pipe = P.StreamingGreedyPipeline(session, 2, scores=0, score_pages=1)
    a, b = pipe.open_stream(), pipe.open_stream()
    chunk = _speech(1, 2)
    pipe.forward(chunk[:1], [a])
    state = pipe.state_of(b).clone()
    with pytest.raises(RuntimeError, match="out of pages"):
        pipe.forward(chunk[1:], [b])
    assert torch.equal(pipe.state_of(b), state) and pipe._open[b].offset == 0
    with pytest.raises(ValueError):
        P.StreamingGreedyPipeline(session, 2, scores=36)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,v", [(5, 65), (5, 128), (5, 256), (5, 512), (5, 1024), (5, 4096), (5, 65536), (5, 65537), (5, 131072), (300, 5000),
                                 (1600, 16384)])
def test_scores_of_rows_of_nan(n, v, dtype):
    """Rows of nothing but NaN, of either sign, and of NaN but for a few entries: ids distinct and in range, ranks in range, floating
    outputs NaN; the other rows as they are without them."""
    x = _rows(n, v, dtype, v)
    clean = x.clone()
    nan = torch.tensor([0x7FC00000, -0x400000], dtype=torch.int32, device="cuda").view(torch.float32).to(TYPES[dtype])
    x[0] = nan[0]
    x[1] = nan[1]
    x[2, : v - 1] = nan[0]
    x[3, : v // 2] = nan[1]
    x[3, v // 2 + 3 :] = nan[0]
    tokens = torch.arange(n, dtype=torch.int32, device="cuda") * 31 % v
    for k in (1, 10, 64):
        r, want = S().token_scores(x, tokens, k=k), S().token_scores(clean, tokens, k=k)
        ids, rank = r.top_ids.cpu().numpy(), r.rank.cpu().numpy()
        assert ids.min() >= 0 and ids.max() < v and rank.min() >= 0 and rank.max() < v, k
        assert all(len(set(row)) == k for row in ids.tolist())
        assert all(bool(t[:4].isnan().all()) for t in (r.logprob, r.entropy, r.top_logprob))
        assert all(torch.equal(a[4:], b[4:]) for a, b in zip(r, want))


def test_pipeline_steps_without_the_splitter(session):
    """step_frames by itself answers with the frame info for as long as a caller likes, scores or not, and holds no rows back:
    what the splitter does not see is of no phrase."""
    from tone_amd import pipeline as P
    pipe, plain = P.StreamingGreedyPipeline(session, 1, scores=2, score_pages=40), P.StreamingGreedyPipeline(session, 1)
    a, b = pipe.open_stream(), plain.open_stream()
    audio = _speech(3, 12)
    for step in range(230):
        np.testing.assert_array_equal(pipe.step_frames(audio[step % 12][None], [a]), plain.step_frames(audio[step % 12][None], [b]))
    assert pipe._store.free_pages == pipe._store.n_pages and pipe._store.length[a] == 0
    with pytest.raises(ValueError):
        pipe.step_frames(audio[:1, :100], [a])
    got = [p for i in range(12) for p in pipe.forward(audio[i][None], [a], [i == 11])[0]]
    want = [p for i in range(12) for p in plain.forward(audio[i][None], [b], [i == 11])[0]]
    assert len(got) > 0 and [(p.text, p.start_time, p.end_time) for p in got] == [(p.text, p.start_time, p.end_time) for p in want]
    assert all(len(p.tokens) == len(p.text) and p.score is not None for p in got)




class _Flags:
    """Speech flags and tokens in the place of the model's (synthetic weights hear speech everywhere): pauses of 25 frames."""

    def __init__(self, monkeypatch, pauses, steps):
        from tone_amd import pipeline as P
        self.tokens = np.random.default_rng(len(pauses)).integers(0, 34, (len(pauses), 10 * steps)).astype(np.int32)
        self.tokens[:, ::3] = 34
        self.speech = np.ones((len(pauses), 10 * steps), bool)
        for i, begins in enumerate(pauses):
            for b in begins:
                self.speech[i, b : b + 25] = False
        monkeypatch.setattr(P, "decode_frame_info", lambda info: next(self.left))

    def at(self, step):
        now = slice(10 * step, 10 * step + 10)
        self.left = iter([(t[now], s[now]) for t, s in zip(self.tokens, self.speech)])


@pytest.mark.parametrize("scores", [None, 3])
def test_pipeline_after_a_decoder_that_raised(session, monkeypatch, scores):
    """A decoder that raises loses the phrases of its step alone: every stream's later phrases and scores are as undisturbed."""
    from tone_amd import pipeline as P

    class Once(P.GreedyLogprobDecoder):
        broken = False

        def forward(self, logprobs):
            if self.broken:
                self.broken = False
                raise RuntimeError("on purpose")
            return super().forward(logprobs)
    chunks = np.stack([_speech(4, 14), _speech(5, 14)])
    flags = _Flags(monkeypatch, [[30, 100], [60]], 14)            # stream 0 pauses in step 3, stream 1 in step 6
    runs = []
    for broken in (False, True):
        dec = Once()
        pipe = P.StreamingGreedyPipeline(session, 2, dec, scores=scores)
        slots = [pipe.open_stream(), pipe.open_stream()]
        steps, raised = [], None
        for step in range(14):
            dec.broken = broken and raised is None and step >= 3
            flags.at(step)
            try:
                steps.append(pipe.forward(chunks[:, step], slots, [step == 13] * 2))
            except RuntimeError:
                raised = step
                steps.append(None)
        runs.append(steps)
        assert (raised is not None) == broken
        if scores is not None:
            assert all(pipe._store.length[s] == pipe._open[s].offset + pipe._open[s].speech.size for s in slots)
    assert [len(p) for p in runs[0][raised]] == [1, 0] and sum(len(p) for s in runs[0][raised + 1 :] for p in s) == 4
    for want, got in zip(*runs):
        assert got is None or got == want


def _run(pipe, chunks, flags, at=None, fail=None):
    """All phrases per step and stream; in step ``at`` the call raises once under ``fail`` and is made again."""
    slots = [pipe.open_stream() for _ in chunks]
    got = []
    for step in range(chunks.shape[1]):
        last = [step == chunks.shape[1] - 1] * len(slots)
        if step == at:
            flags.at(step)
            with fail(), pytest.raises(RuntimeError, match="on purpose"):
                pipe.forward(chunks[:, step], slots, last)
        flags.at(step)
        got.append(pipe.forward(chunks[:, step], slots, last))
    return slots, got


@pytest.mark.parametrize("resident", [True, False])
@pytest.mark.parametrize("where", ["run", "put", "split"])
@pytest.mark.parametrize("at", [0, 7])
def test_pipeline_scores_after_a_step_that_raised(session, monkeypatch, resident, where, at):
    """A step that raises leaves the store with the splitter: made again, the phrases and scores are those of an undisturbed run."""
    from tone_amd import pipeline as P
    chunks = np.stack([_speech(4, 14), _speech(5, 14)])

    def raising(*a, **k):
        raise RuntimeError("on purpose")

    def fail():
        m = pytest.MonkeyPatch()
        if where == "run":
            m.setattr(session, "run_ring" if resident else "run_rows", raising)
        elif where == "put":
            m.setattr(S(), "frames_put", raising)
        else:
            m.setattr(P, "split_frames", raising)
        return _undone(m)
    flags = _Flags(monkeypatch, [[30, 100], [60]], 14)
    want, pipe = (P.StreamingGreedyPipeline(session, 2, scores=3, resident=resident) for _ in range(2))
    _, a = _run(want, chunks, flags)
    if where != "run":
        # the model has stepped: its state is put back as a caller would, so that the same step can be made again
        kept = {}
        monkeypatch.setattr(pipe, "forward", _run_of(pipe, kept))
    slots, b = _run(pipe, chunks, flags, at, fail)
    assert sum(len(p) for step in a for p in step) == 5 and a == b
    assert all(pipe._store.length[s] == pipe._open[s].offset + pipe._open[s].speech.size for s in slots)


def _undone(m):
    import contextlib

    @contextlib.contextmanager
    def block():
        try:
            yield
        finally:
            m.undo()
    return block()


def _run_of(pipe, kept):
    """pipe.forward that puts the model's state back where the call raises."""
    forward = pipe.forward

    def call(*args):
        kept.update(slab=pipe._slab.clone(), parity=pipe._parity.copy(), rings=None if pipe._rings is None else pipe._rings.clone())
        try:
            return forward(*args)
        except RuntimeError:
            torch.cuda.synchronize()
            pipe._slab.copy_(kept["slab"])
            pipe._parity[:] = kept["parity"]
            if pipe._rings is not None:
                pipe._rings.copy_(kept["rings"])
            raise
    return call


def test_pipeline_refuses_too_few_is_last(session):
    """Before the step: the streams are as they were."""
    from tone_amd import pipeline as P
    pipe = P.StreamingGreedyPipeline(session, 2, scores=0)
    a, b = pipe.open_stream(), pipe.open_stream()
    state = pipe.state_of(a).clone()
    with pytest.raises(ValueError, match="is_last"):
        pipe.forward(np.stack([_speech(1, 1)[0], _speech(2, 1)[0]]), [a, b], [False])
    assert torch.equal(pipe.state_of(a), state) and list(pipe._store.length) == [0, 0]


def test_store_refuses_rows_that_cannot_be_put_and_stays_as_it_was():
    """Rows that are one row repeated: refused before any frame is reserved."""
    store = S().FrameStore(2, 32, page_size=8, vocab=5)
    store.append(_rows(20, 5, "fp32", 1).view(2, 10, 5), [0, 1])
    now = lambda: (store.pool, store._table, store._queue, store._cursors)  # noqa: E731
    before, first, length, free = [t.clone() for t in now()], store.first.copy(), store.length.copy(), store.free_pages
    for rows in (_rows(1, 5, "fp32", 2).view(1, 1, 5).expand(2, 10, 5), _rows(2, 5, "fp32", 2).view(2, 1, 5).expand(2, 10, 5)):
        with pytest.raises(ValueError):
            store.append(rows, [0, 1])
    assert all(torch.equal(a, b) for a, b in zip(before, now()))
    assert (store.first == first).all() and (store.length == length).all() and store.free_pages == free


def test_store_takes_a_reservation_back_where_the_copy_raises(monkeypatch):
    store = S().FrameStore(2, 32, page_size=8, n_pages=6, vocab=5)
    rows = _rows(60, 5, "fp32", 1).view(2, 30, 5)
    store.append(rows[:, :10].contiguous(), [0, 1])

    def raising(*a, **k):
        raise RuntimeError("on purpose")
    with monkeypatch.context() as m:
        m.setattr(S(), "frames_put", raising)
        for _ in range(3):
            with pytest.raises(RuntimeError, match="on purpose"):
                store.append(rows[:, 10:16].contiguous(), [1, 0], keep=[9, 9])
    assert list(store.first) == [0, 0] and list(store.length) == [10, 10] and store.free_pages == 2
    store.append(rows[:, 10:16].contiguous(), [0, 1])
    assert torch.equal(store.pool[store.slots([0, 1], [0, 0], [16, 16])], rows[:, :16])


@pytest.mark.parametrize("src,pool", [((slice(None), slice(35)), (slice(None), slice(35, 70))), ((slice(None), slice(35, 70)), (slice(None), slice(35))),
                                      ((slice(0, 20), slice(35)), (slice(20, None), slice(35))), ((slice(7, 8), slice(36, 71)), (slice(None), slice(1, 36)))])
def test_put_beside_the_rows_it_reads(src, pool):
    """Rows and a pool in one buffer that share no entry."""
    b = _rows(60, 71, "fp32", 4)
    want = b.clone()
    n = b[src].shape[0]
    slots = torch.randperm(b[pool].shape[0], device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))[:n].contiguous()
    want[pool][slots] = b[src]
    S().frames_put(b[src], slots, b[pool])
    assert torch.equal(b, want)
    with pytest.raises(ValueError, match="overlap"):
        S().frames_put(b[src], slots, b[:, src[1]])


def test_align_of_too_many_frames_is_refused():
    """Before anything is allocated: one frame repeated 2^29 + 1 times."""
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="frames"):
        S().ctc_align(torch.zeros((1, 1, 5), device="cuda").expand(1, 2 ** 29 + 1, 5), one.view(1, 1), one, one, blank=4)


@pytest.mark.parametrize("most", [2, 60, 300, 700, 900, 1300])
def test_align_of_large_entries_and_a_closed_frame(most):
    """Large entries of either sign make no path out of none: a closed frame or label and too few frames leave both outputs
    -inf, and an unlikely path that is open is not lost among likely ones that are closed."""
    frames = 2700
    tokens = _dev(np.stack([np.arange(most) % 8, np.zeros(most)]), np.int32)
    lens = _dev([most, most], np.int32)
    for size in (5.9e4, 40.0, -5.9e4):
        x = torch.full((2, frames, 9), size, device="cuda")
        x[0, frames // 3] = float("-inf")              # no way through this frame
        short = torch.tensor([frames, min(frames, 2 * most - 2)], dtype=torch.int32, device="cuda")      # repeats need a blank between
        r = S().ctc_align(x, tokens, lens, short, blank=8, total=True)
        assert r.score.tolist() == [-np.inf] * 2 and r.total.tolist() == [-np.inf] * 2 and bool((r.labels == -1).all())
    # the blank unlikely and open in every frame, the tokens likely and each closed in its turn: blanks alone are left
    x = torch.full((1, 1000, 9), 5.9e4, device="cuda")
    x[:, :, 8] = -5.9e4
    x[:, 500, :8] = float("-inf")
    r = S().ctc_align(x, tokens[:1], _dev([0], np.int32), _dev([1000], np.int32), blank=8, total=True)
    assert float(r.score) == -5.9e7 and abs(float(r.total) + 5.9e7) <= 5.9e7 * 8 * EPS
    # one token: it lies on either side of the closed frame, the rest are unlikely blanks
    x[:, :, :8] = -5.9e4
    x[:, 500, :8] = float("-inf")
    r = S().ctc_align(x, _dev([[3]], np.int32), _dev([1], np.int32), _dev([1000], np.int32), blank=8, total=True)
    paths = np.log(500 * 501 / 2 + 499 * 500 / 2)
    assert float(r.score) == -5.9e7 and abs(float(r.total) + 5.9e7 - paths) <= 5.9e7 * 8 * EPS


def _sums(x, tokens, blank):
    """(score, total) of one sequence: x float64 (F, V), all states of a frame at once, in 64 bits."""
    lab = np.full(2 * len(tokens) + 1, blank)
    lab[1::2] = tokens
    jump = np.zeros(len(lab), bool)
    jump[3::2] = lab[3::2] != lab[1:-2:2]
    v = w = np.where(np.arange(len(lab)) < 2, x[0, lab], -np.inf)
    for row in x[1:]:
        c = np.full((2, 3, len(lab)), -np.inf)
        for at, src in ((0, v), (1, w)):
            c[at, 0], c[at, 1, 1:], c[at, 2, 2:] = src, src[:-1], np.where(jump[2:], src[:-2], -np.inf)
        h = np.maximum(c[1].max(0), -1e300)
        with np.errstate(divide="ignore"):
            w = h + np.log(np.exp(c[1] - h).sum(0)) + row[lab]
        v = c[0].max(0) + row[lab]
    return max(v[-1], v[-2]), np.logaddexp(w[-1], w[-2])


@pytest.mark.parametrize("f,most,vocab", [(1, 1, 35), (40, 9, 35), (187, 43, 35), (500, 120, 35), (500, 120, 300), (2000, 300, 35), (2000, 700, 35),
                                          (2300, 1000, 35)])
@pytest.mark.parametrize("sure", [0.5, 1e-2, 1e-5, 1e-7, 1e-9])
def test_align_of_confident_rows(f, most, vocab, sure):
    """Rows that leave about ``sure`` to all but the label said: the total lies close to 0 and has to be right in proportion.

    Each entry's factor e^v is held as 1 + d and a power of 2, d in 32 bits.  With |v| <= ln 2 / 2 the power is 1 and d is off by
    2 EPS of itself (its last rounding, and four roundings of the rest of its series, which is at most a fifth of it), so the
    factor's logarithm by 2 EPS |d| / (1 + d) <= 2.4 EPS |v|.  Beyond, two roundings of the reduced argument (EPS / 4 each) and
    2 EPS of |d| <= 0.42, divided by 1 + d >= 0.7, are below 2 EPS, which is below 6 EPS |v|.  The total is a mean over the paths,
    weighted by their probability, so it is off by at most 6 EPS of that mean of sum |v|: minus the derivative of the total by a
    common factor of all entries.  The states are 64 bits wide: at most 8 roundings a frame of the kernel, and as many of the
    definition evaluated here.  Then one rounding to 32 bits."""
    rng = np.random.default_rng(f)
    tokens = rng.integers(0, vocab - 1, most)
    tokens[tokens >= 34] += 1 if vocab > 35 else 0
    said = np.full(f, 34)
    said[((np.arange(most) + 0.5) * f / most).astype(int)] = tokens
    left = sure * rng.random(f) + 1e-30
    x = np.log(left)[:, None] + np.log(rng.dirichlet(np.ones(vocab), f) + 1e-30)
    x[np.arange(f), said] = np.log1p(-left)
    x = x.astype(np.float32)
    r = S().ctc_align(_dev(x[None]), _dev(tokens[None], np.int32), _dev([most], np.int32), _dev([f], np.int32), blank=34, total=True)
    x = x.astype(np.float64)
    score, total = _sums(x, tokens, 34)
    assert r.score.item() == np.float32(score)
    size = (_sums(x * (1 - 1e-4), tokens, 34)[1] - total) / 1e-4
    tol = 6 * EPS * size * 1.01 + 16 * f * 2.0 ** -53 + EPS * abs(total)
    assert abs(r.total.item() - total) <= tol, (r.total.item(), total, tol)


@pytest.mark.parametrize("most,f", [(170, 230), (700, 760)])
def test_long_alignment_captured_and_replayed(most, f):
    """Shapes whose stages need more LDS than a launch has by default, in two graphs with eager calls between."""
    rng = np.random.default_rng(most)
    x, tokens, _, _ = _ctc(rng, 2, f, most, 900, 34)
    xd, td = _dev(x, np.float32), _dev(tokens)
    lens = _dev([most, most - 7], np.int32), _dev([f, f - 3], np.int32)
    fn = lambda: S().ctc_align(xd, td, *lens, total=True)  # noqa: E731
    fn()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = fn()
        graphs.append((g, out))
    torch.cuda.synchronize()
    for step in range(3):
        xd.add_(torch.randn_like(xd).mul_(0.1))
        want = [t.clone() for t in fn()]
        torch.cuda.synchronize()
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, out)), f"replay {step}"


def test_store_calls_of_no_streams():
    store = S().FrameStore(2, 32, page_size=8, vocab=5)
    assert tuple(store.reserve([], 4).shape) == (0, 4) and tuple(store.append(torch.empty((0, 3, 5), device="cuda"), []).shape) == (0, 3)
    assert tuple(store.append(torch.empty((2, 0, 5), device="cuda"), [0, 1]).shape) == (2, 0)
    store.release([])
    assert tuple(store.slots([], [], []).shape) == (0, 0) and tuple(store.slots([1], [0], [0]).shape) == (1, 0)
    rows = _rows(6, 5, "fp32", 1).view(2, 3, 5)
    assert torch.equal(store.pool[store.append(rows, [0, 1])], rows) and store.free_pages == store.n_pages - 2


@pytest.mark.parametrize("f,most", [(8192, 20), (8193, 30), (20000, 40), (9000, 200)])
def test_align_of_many_frames(f, most):
    """Paths of more legs than are traced between two barriers (256 of 32 frames)."""
    rng = np.random.default_rng(f)
    x, tokens, _, _ = _ctc(rng, 1, f, most, 35, 34)
    _align_by_rows(rng, x, tokens, np.array([[most, f]], np.int32))


def test_plan_of_very_many_streams():
    rng = np.random.default_rng(5)
    n = 70001
    p = Pool(rng, n, 4, 4, 3 * n, head=12345)
    p.step(rng.permutation(n), np.zeros(n, int), rng.integers(0, 6, n), 5)
    ids = rng.permutation(n)[: n // 2]
    p.step(ids, p.length[ids] // 2, rng.integers(0, 6, len(ids)), 5)
