"""Attention over a paged cache with a sliding window and first tokens that
stay visible, against float64 from the definition: windows and sinks around the
tiles' sizes, every kernel and split, pages that are no longer there, values
that a row may not see."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from dpuf_amd import abi

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip(eng):
    h = R.Hip()
    yield h
    h.free_all()


def say(*a):
    print(*a, flush=True)


def sees(p, t, window, sink):
    return (t <= p) & ((t > p - window) | (t < sink))


def windowed(cache, q, scale, nq, window, sink):
    """As paged_ref.attention, of the keys that a row's window leaves."""
    G, n = nq // cache.nkv, cache.n_rows
    out, A = np.zeros((n, nq, cache.hd)), np.zeros((n, nq, cache.hd))
    lse, S, vmax = np.full((n, nq), -np.inf), np.zeros((n, nq)), np.zeros((n, nq))
    for s, (r, c) in enumerate(zip(cache.rows, cache.ctx)):
        there = cache.present(s)
        for h in range(cache.nkv):
            k, v = cache.gather(cache.k, s, h), cache.gather(cache.v, s, h)
            for i in range(r):
                see = np.where(there & sees(c - r + i, np.arange(c), window, sink))[0]
                if len(see) == 0:
                    continue
                row = cache.starts[s] + i
                for j in range(h * G, (h + 1) * G):
                    x = k[see] @ q[row, j] * scale
                    m = x.max()
                    e = np.exp(x - m)
                    lse[row, j] = m + np.log(e.sum())
                    p = e / e.sum()
                    out[row, j] = p @ v[see]
                    A[row, j] = p @ np.abs(v[see])
                    S[row, j] = (np.abs(k[see]) @ np.abs(q[row, j])).max() * scale
                    vmax[row, j] = np.abs(v[see]).max()
    return out, lse, A, S, vmax


def call(eng, hip, cache, nq, q, scale, window, sink, out_t=None, max_ctx=None, extra=0, stream=None):
    """Outputs and lse of one call; `extra` rows behind the last sequence's."""
    out_t = cache.t if out_t is None else out_t
    n = cache.n_rows + extra
    dq = hip.put(np.concatenate([q, np.zeros((extra,) + q.shape[1:], q.dtype)]))
    do = hip.put(R.to_type(np.full((n, nq, cache.hd), 7.5, np.float32), out_t))
    dl = hip.put(np.full((n, nq), 7.5, np.float32))
    b, p = cache.batch(max_ctx, n), cache.pages(w=False)
    ws = int(eng.dpuf_amd_paged_attn_window_workspace(C.byref(b), C.byref(p), nq, window, sink))
    dws = hip.put(np.full(max(ws, 16), 0xFF, np.uint8))        # NaN: nothing may rely on a cleared workspace
    rc = eng.dpuf_amd_paged_attn_window(C.byref(b), C.byref(p), nq, dq.p, scale, window, sink, out_t, do.p, dl.p,
                                        dws.p if ws else None, ws, stream)
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    return R.from_type(do.get(), out_t), dl.get(), ws


def bound_of(t, out_t, out, A, S, vmax, hd, ctx):
    """paged_ref.attention_bound's, and as much again for the probabilities'
    rounding: o is divided by their sum as they were rounded, so that an error e
    of a probability counts as e (v - o), at most |e| (|v| + |o|), and sum |e| |o|
    is at most half a step of A."""
    more = A * R.HALF_STEP[t] * 1.01 + (ctx * 2.0 ** -25 * vmax[..., None] if t == R.F16 else 0.0)
    return R.attention_bound(t, out_t, out, A, S, vmax, hd, ctx) + more


def check(cache, nq, q, scale, out, lse, out_t, window, sink):
    n = cache.n_rows
    ref, rl, A, S, vmax = windowed(cache, R.from_type(q, cache.t), scale, nq, window, sink)
    bound = bound_of(cache.t, out_t, ref, A, S, vmax, cache.hd, min(max(cache.ctx), window + sink))
    err = np.abs(out[:n] - ref)
    say(f"  worst error {float((err / bound).max()) if err.size else 0.0:.3f} of the bound")
    assert np.all(err <= bound)
    empty = np.isneginf(rl)
    assert np.array_equal(np.isneginf(lse[:n]), empty)
    assert np.all(out[:n][empty] == 0.0)
    dl = np.abs(lse[:n][~empty] - rl[~empty])
    assert np.all(dl <= R.score_error(S, cache.hd)[~empty] + np.abs(rl[~empty]) * 2.0 ** -22 + 2.0 ** -20)
    assert np.all(out[n:] == 7.5) and np.all(lse[n:] == 7.5)


# rows, contexts: a first token, lengths around 16, 32, 64 and 128, an empty sequence, one without new rows, one with
# more new rows than cached ones, chunks of longer contexts
RAGGED = ([1, 1, 0, 3, 1, 40, 2, 1, 0, 5, 70], [1, 17, 0, 3, 130, 95, 64, 33, 50, 3, 301])


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("nq,nkv,hd,page", [(4, 1, 64, 16), (4, 4, 128, 32), (10, 2, 128, 16), (8, 1, 256, 64),
                                            (32, 1, 128, 16), (21, 7, 256, 16)])
@pytest.mark.parametrize("window,sink", [(1, 0), (1, 1), (7, 0), (16, 4), (33, 16), (64, 1), (100, 40), (20, 70),
                                         (300, 2), (1 << 30, 0), (5, 1 << 30), (1 << 30, 1 << 30)])
def test_ragged(eng, hip, nq, nkv, hd, page, t, window, sink):
    rng = np.random.default_rng(nq * 1000 + hd + t)
    cache = R.Cache(hip, rng, t, *RAGGED, nkv, hd, page, slots_first=bool(nq & 2))
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)) * 1.5, t)
    scale = float(np.float32(1 / np.sqrt(hd)))
    say(f"ragged: {nq}/{nkv} heads of {hd}, pages of {page}, type {t}, window {window}, sink {sink}")
    out, lse, _ = call(eng, hip, cache, nq, q, scale, window, sink, extra=3)
    check(cache, nq, q, scale, out, lse, t, window, sink)


# Every kernel and split of the keys: (rows, contexts, max_ctx given, window, sink)
MODES = {
    "few": ([0, 1, 3, 1, 0], [40, 1300, 700, 90, 0], None, 100, 4),
    "few, split": ([0, 5, 0, 1, 0, 0], [40, 1300, 1, 2700, 0, 9], None, 1000, 70),
    "few, one row": ([1], [2111], None, 700, 4),
    "few, shorter than its window": ([1, 1], [2111, 33], None, 5000, 4),
    "many": ([40], [395], None, 90, 33),
    "many, split": ([33], [3500], None, 1500, 0),
    "wide, short keys": ([150], [333], 5000, 2500, 3),
    "wide, split": ([97], [4300], None, 2300, 129),
    "wide, few rows of them": ([0], [50], 4096, 2200, 1),
    "mixed": ([1, 70, 1, 30], [900, 400, 33, 30], None, 50, 5),
    "mixed, split": ([1, 70, 2, 0, 1, 30], [1900, 3400, 600, 7, 33, 30], None, 1300, 20),
}


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("mode", MODES)
def test_kernels_and_splits(eng, hip, mode, hd):
    """... and device row counts below n_rows: the rows behind stay."""
    rows, ctx, max_ctx, window, sink = MODES[mode]
    rng = np.random.default_rng(len(mode) + hd)
    t = R.F16 if hd == 64 else R.BF16
    cache = R.Cache(hip, rng, t, rows, ctx, 2, hd, 32, slots_first=hd == 128, table_extra=160)
    q = R.to_type(rng.standard_normal((cache.n_rows, 8, hd)) * 1.5, t)
    extra = 100 if mode == "wide, few rows of them" else 0
    say(f"{mode}: hd {hd}, window {window}, sink {sink}")
    out, lse, ws = call(eng, hip, cache, 8, q, 0.1, window, sink, max_ctx=max_ctx, extra=extra,
                        out_t=R.F32 if hd == 256 else None)
    check(cache, 8, q, 0.1, out, lse, R.F32 if hd == 256 else t, window, sink)


@pytest.mark.parametrize("max_ctx", [1, 600, 100000])
@pytest.mark.parametrize("mode", ["few, split", "many, split", "wide, split", "mixed", "mixed, split"])
def test_estimates_of_the_longest_context(eng, hip, mode, max_ctx):
    """Keys are split by what the windows leave, whatever the caller's estimate
    of the longest context is."""
    rows, ctx, _, window, sink = MODES[mode]
    rng = np.random.default_rng(len(mode) + max_ctx)
    cache = R.Cache(hip, rng, R.BF16, rows, ctx, 2, 64, 16, table_extra=6000)
    q = R.to_type(rng.standard_normal((cache.n_rows, 8, 64)) * 1.5, R.BF16)
    say(f"estimates: {mode}, max_ctx {max_ctx}")
    out, lse, _ = call(eng, hip, cache, 8, q, 0.1, window, sink, max_ctx=max_ctx, extra=2)
    check(cache, 8, q, 0.1, out, lse, R.BF16, window, sink)


@pytest.mark.parametrize("rows,ctx", [([50], [9000]), ([1, 60, 1, 45], [300, 9000, 4000, 45]), ([30, 20], [8200, 30])])
@pytest.mark.parametrize("window", [8191, 8200, 9007, 9008, 1 << 30])
def test_long_windows_of_chunks(eng, hip, rows, ctx, window):
    """Many ranges of keys, and windows a key less than what the table holds
    (9 008 rows), as much, and more."""
    rng = np.random.default_rng(window + len(rows))
    cache = R.Cache(hip, rng, R.BF16, rows, ctx, 1, 64, 16)
    q = R.to_type(rng.standard_normal((cache.n_rows, 4, 64)) * 1.5, R.BF16)
    say(f"long windows: rows {rows} over {ctx}, window {window}, table {cache.table.shape}")
    out, lse, _ = call(eng, hip, cache, 4, q, 0.125, window, 3, extra=1)
    check(cache, 4, q, 0.125, out, lse, R.BF16, window, 3)


@pytest.mark.parametrize("rows", [1, 3])
def test_hundreds_of_sequences(eng, hip, rows):
    rng = np.random.default_rng(rows)
    n = 300
    ctx = [int(c) for c in rng.integers(rows, 90, n)]
    cache = R.Cache(hip, rng, R.BF16, [rows if i % 7 else 0 for i in range(n)], ctx, 1, 64, 16)
    q = R.to_type(rng.standard_normal((cache.n_rows, 4, 64)) * 1.5, R.BF16)
    say(f"{n} sequences of {rows} rows")
    out, lse, _ = call(eng, hip, cache, 4, q, 0.125, 20, 3, extra=5)
    check(cache, 4, q, 0.125, out, lse, R.BF16, 20, 3)


@pytest.mark.parametrize("mode", MODES)
def test_pages_outside_every_window_may_be_anything(eng, hip, mode):
    """Tables whose other entries are gone, another sequence's or no page at
    all, and pools of NaN there: the same bits."""
    rows, ctx, max_ctx, window, sink = MODES[mode]
    rng = np.random.default_rng(len(mode))
    cache = R.Cache(hip, rng, R.BF16, rows, ctx, 2, 64, 16, table_extra=300)
    q = R.to_type(rng.standard_normal((cache.n_rows, 8, 64)) * 1.5, R.BF16)
    say(f"pages gone, {mode}")
    want = call(eng, hip, cache, 8, q, 0.1, window, sink, max_ctx=max_ctx)
    table, gone = cache.table.copy(), 0
    for s, (r, c) in enumerate(zip(rows, ctx)):
        lo = max(0, c - r - window + 1) if r else c
        for j in range(table.shape[1]):
            if j * 16 >= c or ((j + 1) * 16 <= lo and (j * 16 >= sink or r == 0)):
                table[s, j] = rng.choice([-1, cache.n, 2 ** 31 - 1, -2 ** 31])
                gone += j * 16 < c
                if j * 16 < c:
                    cache.k[cache.table[s, j]] = R.to_type([np.nan], R.BF16)[0]
                    cache.v[cache.table[s, j]] = R.to_type([np.nan], R.BF16)[0]
    cache.d_table.set(table)
    cache.dk.set(cache.k)
    cache.dv.set(cache.v)
    got = call(eng, hip, cache, 8, q, 0.1, window, sink, max_ctx=max_ctx)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    assert gone > 0 or window >= max(ctx) or max(ctx) < 64


@pytest.mark.parametrize("rows,ctx", [([1, 2, 60], [90, 140, 180]), ([600], [700])])
def test_absent_pages_within_a_window(eng, hip, rows, ctx):
    """Rows whose whole window lies on absent pages are empty."""
    rng = np.random.default_rng(5)
    bad = [(0, 0), (0, 4), (0, 5)] + ([(1, 0), (1, 7), (1, 8), (2, 3), (2, 9)] if len(ctx) > 1 else [(0, 40), (0, 43)])
    cache = R.Cache(hip, rng, R.F16, rows, ctx, 2, 64, 16, bad=bad)
    q = R.to_type(rng.standard_normal((cache.n_rows, 4, 64)), R.F16)
    for window, sink in ((9, 0), (9, 16), (40, 3), (16, 20)):
        say(f"absent pages: rows {rows}, window {window}, sink {sink}")
        out, lse, _ = call(eng, hip, cache, 4, q, 0.125, window, sink, extra=1)
        check(cache, 4, q, 0.125, out, lse, R.F16, window, sink)
        if (window, sink) == (9, 0):
            assert np.isneginf(lse[:cache.n_rows]).any()


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("mode", MODES)
def test_a_row_that_sees_itself_alone(eng, hip, mode, hd, t):
    """A window of one: the outputs are the values, bit for bit, and with a
    first key of weight 0 beside it they are too."""
    rows, ctx, max_ctx, _, _ = MODES[mode]
    rng = np.random.default_rng(hd + t)
    cache = R.Cache(hip, rng, t, rows, ctx, 2, hd, 16, table_extra=300)
    q = R.to_type(rng.standard_normal((cache.n_rows, 8, hd)) * 1.5, t)
    want = np.zeros((cache.n_rows, 8, hd))
    for s, (r, c) in enumerate(zip(rows, ctx)):
        for i in range(r):
            p = c - r + i
            if p >= 0:
                v = R.from_type(cache.row(cache.v, cache.table[s, p // 16], p % 16), t)
                want[cache.starts[s] + i] = np.repeat(v, 4, 0)
    say(f"itself alone, {mode}: hd {hd}, type {t}")
    out, lse, _ = call(eng, hip, cache, 8, q, 0.1, 1, 0, max_ctx=max_ctx)
    assert np.array_equal(out, want)


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("mode", MODES)
def test_infinities_and_nan_outside_a_window(eng, hip, mode, hd, t):
    """Values of infinities and NaN, and a key of NaN, spread over the cache:
    rows get what the definition gives for the keys that they see."""
    rows, ctx, max_ctx, window, sink = MODES[mode]
    rng = np.random.default_rng(2 * len(mode) + hd)
    nq, page = 8, 16
    cache = R.Cache(hip, rng, t, rows, ctx, 2, hd, page, table_extra=320)
    for s, (n, c) in enumerate(zip(rows, ctx)):
        first = max(0, c - n - window + 1)
        # before the first row's window, in it as later rows leave it, and new rows' own
        at = [i for i in (sink, first - 1, first - 40, first + n // 2, first + n - 2, c - 1) if 0 <= i < c and n]
        for i in at:
            pg, r = cache.table[s, i // page], i % page
            for h in range(2):
                cols = rng.integers(0, hd, 3)
                cache.v[pg, h, r, cols] = R.to_type([np.inf, -np.inf, np.nan], t)[rng.integers(0, 3, 3)]
        if n > 1 and first > sink:
            cache.k[cache.table[s, first // page], 1, first % page, 3] = R.to_type([np.nan], t)[0]
    cache.dv.set(cache.v)
    cache.dk.set(cache.k)
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)), t)
    say(f"odd values, {mode}: hd {hd}, type {t}, window {window}, sink {sink}")
    out, lse, _ = call(eng, hip, cache, nq, q, 0.1, window, sink, max_ctx=max_ctx)
    with np.errstate(all="ignore"):
        ref, rl, A, S, _ = windowed(cache, R.from_type(q, t), 0.1, nq, window, sink)
        # the values themselves are below 10 (standard normal)
        bound = bound_of(t, t, ref, A, S, np.full(S.shape, 10.0), hd, max(ctx))
        assert np.array_equal(np.isnan(out), np.isnan(ref))
        assert np.array_equal(np.isposinf(out), np.isposinf(ref)) and np.array_equal(np.isneginf(out), np.isneginf(ref))
        ok = np.isfinite(ref)
        assert ok.any() or not cache.n_rows
        assert np.all(np.abs(out[ok] - ref[ok]) <= bound[ok])
        assert np.array_equal(np.isnan(lse), np.isnan(rl)) and np.array_equal(np.isneginf(lse), np.isneginf(rl))


def test_scores_far_apart(eng, hip):
    """Scores of a few hundred: the running maximum moves, what it left is 0."""
    rng = np.random.default_rng(8)
    for rows, ctx in (([1, 3], [300, 77]), ([90], [333])):
        for t in (R.BF16, R.F16):
            cache = R.Cache(hip, rng, t, rows, ctx, 2, 128, 16, kscale=9.0)
            q = R.to_type(rng.standard_normal((cache.n_rows, 8, 128)) * 9.0, t)
            say(f"far scores: rows {rows}, type {t}")
            out, lse, _ = call(eng, hip, cache, 8, q, 0.088, 150, 3)
            check(cache, 8, q, 0.088, out, lse, t, 150, 3)


@pytest.mark.parametrize("rows,page", [(1, 1024), (3, 1024), (200, 1024), (7, 16)])
def test_places_near_the_table_s_end(eng, hip, rows, page):
    """A context of about 2^30 rows (2^26 in pages of 16) whose pages are gone
    but for the first and the last few."""
    rng = np.random.default_rng(rows)
    hd, nq, nkv, window, sink = 64, 4, 2, 300, 20
    entries = (1 << 20) if page == 1024 else 1 << 22
    ctx = entries * page - 3
    n = 40
    table = np.full((1, entries), -1, np.int32)
    ids = rng.permutation(n).astype(np.int32)
    held = sorted({i // page for i in list(range(sink)) + list(range(ctx - rows - window + 1, ctx))})
    table[0, held] = ids[:len(held)]
    k, v = (R.to_type(rng.standard_normal((n, nkv, page, hd)), R.BF16) for _ in range(2))
    q = R.to_type(rng.standard_normal((rows, nq, hd)), R.BF16)
    dk, dv, dq, dt = hip.put(k), hip.put(v), hip.put(q), hip.put(table)
    starts, lens = hip.put(np.array([0, rows], np.int32)), hip.put(np.array([ctx], np.int32))
    p = abi.DpufAmdPages(type=R.BF16, n_pages=n, page_size=page, n_kv_heads=nkv, head_dim=hd,
                         page_stride=nkv * page * hd, head_stride=page * hd, row_stride=hd, k=dk.p, v=dv.p, w=None)
    b = abi.DpufAmdBatch(n_seqs=1, n_rows=rows, table_stride=entries, max_ctx=ctx, row_start=starts.p, ctx_len=lens.p,
                         page_table=dt.p)
    ws = int(eng.dpuf_amd_paged_attn_window_workspace(C.byref(b), C.byref(p), nq, window, sink))
    dws, do = hip.put(np.zeros(max(16, ws), np.uint8)), hip.put(np.zeros((rows, nq, hd), np.float32))
    dl = hip.put(np.zeros((rows, nq), np.float32))
    say(f"{rows} rows at place {ctx}")
    rc = eng.dpuf_amd_paged_attn_window(C.byref(b), C.byref(p), nq, dq.p, 0.125, window, sink, R.F32, do.p, dl.p, dws.p,
                                        ws, None)
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    out, k64, v64, q64 = do.get(), R.from_type(k, R.BF16), R.from_type(v, R.BF16), R.from_type(q, R.BF16)
    at = np.array(sorted(set(range(sink)) | set(range(ctx - rows - window + 1, ctx))))
    for i in range(rows):
        see = at[sees(ctx - rows + i, at, window, sink)]
        assert len(see) == window + sink
        pg = table[0, see // page]
        for j in range(nq):
            kk, vv = k64[pg, j // 2, see % page], v64[pg, j // 2, see % page]
            x = kk @ q64[i, j] * 0.125
            e = np.exp(x - x.max())
            pr = e / e.sum()
            S = (np.abs(kk) @ np.abs(q64[i, j])).max() * 0.125
            A = pr @ np.abs(vv)
            ref = pr @ vv
            bound = bound_of(R.BF16, R.F32, ref[None], A[None], np.array([S]), np.abs(vv).max()[None], hd, 400)[0]
            assert np.all(np.abs(out[i, j] - ref) <= bound), (i, j)


def test_two_streams_and_a_graph(eng, hip):
    """Two calls at once on streams of their own with workspaces of their own;
    then a captured call replayed over new lengths and values between eager
    calls gives what the eager call gives."""
    rng = np.random.default_rng(11)
    nq, hd, window, sink = 8, 128, 700, 4
    caches = [R.Cache(hip, rng, R.BF16, rows, ctx, 2, hd, 32) for rows, ctx in
              (([1, 1, 1], [900, 1500, 3]), ([200, 1], [1800, 700]))]
    work = []
    for cache in caches:
        q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)) * 1.5, R.BF16)
        b, p = cache.batch(), cache.pages(w=False)
        n = int(eng.dpuf_amd_paged_attn_window_workspace(C.byref(b), C.byref(p), nq, window, sink))
        work.append((cache, q, hip.put(q), hip.put(np.zeros((cache.n_rows, nq, hd), np.uint16)),
                     hip.put(np.zeros((cache.n_rows, nq), np.float32)), hip.put(np.zeros(max(16, n), np.uint8)), n, b,
                     p, hip.stream()))

    def launch(wk, s):
        cache, q, dq, do, dl, ws, n, b, p, _ = wk
        assert eng.dpuf_amd_paged_attn_window(C.byref(b), C.byref(p), nq, dq.p, 0.09, window, sink, R.BF16, do.p, dl.p,
                                              ws.p, n, s) == 0

    say("two streams")
    for _ in range(3):
        for wk in work:
            launch(wk, wk[-1])
    for wk in work:
        assert hip.lib.hipStreamSynchronize(wk[-1]) == 0
        check(wk[0], nq, wk[1], 0.09, R.from_type(wk[3].get(), R.BF16), wk[4].get(), R.BF16, window, sink)
    say("graph")
    wk = work[0]
    cache, q, dq, do, dl, *_, s = wk
    graph, ge = C.c_void_p(), C.c_void_p()
    assert hip.lib.hipStreamBeginCapture(s, 1) == 0
    launch(wk, s)
    assert hip.lib.hipStreamEndCapture(s, C.byref(graph)) == 0
    assert hip.lib.hipGraphInstantiate(C.byref(ge), graph, None, None, 0) == 0
    for ctx in ([900, 1500, 3], [10, 1480, 3], [33, 0, 1], [899, 1499, 2]):
        cache.d_ctx.set(np.array(ctx, np.int32))
        cache.ctx = ctx
        do.set(np.full((3, nq, hd), 0x7FC0, np.uint16))
        assert hip.lib.hipGraphLaunch(ge, s) == 0
        assert hip.lib.hipStreamSynchronize(s) == 0
        got, gl = do.get(), dl.get()
        check(cache, nq, q, 0.09, R.from_type(got, R.BF16), gl, R.BF16, window, sink)
        launch(wk, s)
        assert hip.lib.hipStreamSynchronize(s) == 0
        assert np.array_equal(do.get(), got) and np.array_equal(dl.get().view(np.uint32), gl.view(np.uint32))
    hip.lib.hipGraphExecDestroy(ge)
    hip.lib.hipGraphDestroy(graph)
    for wk in work:
        hip.lib.hipStreamDestroy(wk[-1])


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,ctx,window,sink", [
    ([70], [70], 100, 0), ([1], [95], 200, 3), ([1, 40, 0, 3], [90, 55, 3, 88], 128, 2), ([33], [3500], 4000, 0),
    ([140], [2200], 3000, 1), ([1, 1, 1], [20, 1300, 600], 1500, 4), ([70, 2], [70, 90], 3, 150)])
def test_windows_that_reach_everything_at_any_width_of_the_table(eng, hip, rows, ctx, window, sink, hd, t):
    """A window or first tokens as long as every sequence: the same bits with a
    table that holds fewer rows than those, as many or more, and a row that
    sees itself alone has its v."""
    got = []
    reach = max(window, sink)
    for extra in (0, -(-reach // 16) - -(-max(ctx) // 16), 1 << 12):
        rng = np.random.default_rng(hd + t)
        cache = R.Cache(hip, rng, t, rows, ctx, 2, hd, 16, table_extra=extra)
        q = R.to_type(rng.standard_normal((cache.n_rows, 8, hd)) * 1.5, t)
        say(f"whole windows: {rows} rows over {ctx}, hd {hd}, type {t}, a table of {cache.table.shape[1]} pages")
        assert (16 * cache.table.shape[1] < reach) == (extra == 0)
        out, lse, _ = call(eng, hip, cache, 8, q, 0.1, window, sink)
        check(cache, 8, q, 0.1, out, lse, t, window, sink)
        for s, (r, c) in enumerate(zip(rows, ctx)):
            if r == c:
                v = R.from_type(cache.row(cache.v, cache.table[s, 0], 0), t)
                assert np.array_equal(out[cache.starts[s]], np.repeat(v, 4, 0))
        got.append((out, lse))
        hip.free_all()
    assert all(np.array_equal(g[0], got[0][0]) and np.array_equal(g[1], got[0][1]) for g in got[1:])


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("mode", MODES)
def test_pages_outside_every_window_may_be_others(eng, hip, mode, t):
    """Entries behind a window that still are pages of the pool, as a program
    leaves them that gives pages back: pages of NaN by now, other sequences'
    pages, and pages that the row sees at another place: the same bits."""
    rows, ctx, max_ctx, window, sink = MODES[mode]
    rng = np.random.default_rng(len(mode) + t)
    cache = R.Cache(hip, rng, t, rows, ctx, 2, 64, 16, table_extra=300)
    q = R.to_type(rng.standard_normal((cache.n_rows, 8, 64)) * 1.5, t)
    say(f"pages of others, {mode}, type {t}")
    want = call(eng, hip, cache, 8, q, 0.1, window, sink, max_ctx=max_ctx)
    seen, gone = [], []
    for s, (r, c) in enumerate(zip(rows, ctx)):
        lo = max(0, c - r - window + 1) if r else c
        for j in range(cache.table.shape[1]):
            out = j * 16 >= c or ((j + 1) * 16 <= lo and (j * 16 >= sink or r == 0))
            (gone if out else seen).append((s, j))
    own = cache.table.copy()
    live = np.array([own[at] for at in seen])
    nan = np.setdiff1d(np.arange(cache.n), live).astype(np.int32)
    for pool in (cache.k, cache.v):
        pool[nan] = R.to_type([np.nan], t)[0]
    cache.dk.set(cache.k)
    cache.dv.set(cache.v)
    for what in ("their own, of NaN", "seen ones", "any"):
        table = own.copy()
        for s, j in gone:
            if what == "seen ones":
                table[s, j] = rng.choice(live)
            elif what == "any":
                table[s, j] = rng.integers(0, cache.n)
            elif table[s, j] < 0:
                table[s, j] = rng.choice(nan)
        assert table.min() >= 0 and table.max() < cache.n
        cache.d_table.set(table)
        got = call(eng, hip, cache, 8, q, 0.1, window, sink, max_ctx=max_ctx)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), what
        out, lse, _ = got
        cache.table = own
        check(cache, 8, q, 0.1, out, lse, t, window, sink)


@pytest.mark.parametrize("t", [R.BF16, R.F16])
def test_a_full_call_of_32_heads(eng, hip, t):
    """512 rows of 32 heads, 8 kv heads of 128, in fp32 as an engine takes them."""
    rng = np.random.default_rng(31 + t)
    cache = R.Cache(hip, rng, t, [512], [1907], 8, 128, 64)
    q = R.to_type(rng.standard_normal((512, 32, 128)) * 1.5, t)
    scale = float(np.float32(1 / np.sqrt(128)))
    say(f"512 rows of 32 heads, type {t}")
    out, lse, _ = call(eng, hip, cache, 32, q, scale, 300, 5, out_t=R.F32)
    check(cache, 32, q, scale, out, lse, R.F32, 300, 5)
