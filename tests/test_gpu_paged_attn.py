"""Attention of new tokens over a paged cache, and the attention weights of
cached rows, against float64 from the definition: ragged batches, odd lengths,
every head dim and grouping the kernels are built for, rows nobody may see."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip(eng):
    h = R.Hip()
    yield h
    h.free_all()


def say(*a):
    print(*a, flush=True)


def call(eng, hip, cache, nq, q, scale, out_t=None, max_ctx=None, extra=0, stream=None, lse=True):
    """Outputs and lse of one call; `extra` rows behind the last sequence's."""
    out_t = cache.t if out_t is None else out_t
    n = cache.n_rows + extra
    qs = np.concatenate([q, np.zeros((extra,) + q.shape[1:], q.dtype)])
    dq = hip.put(qs)
    fill = R.to_type(np.full((n, nq, cache.hd), 7.5, np.float32), out_t)
    do, dl = hip.put(fill), hip.put(np.full((n, nq), 7.5, np.float32))
    b, p = cache.batch(max_ctx, n), cache.pages(w=False)
    ws = int(eng.dpuf_amd_paged_attn_workspace(C.byref(b), C.byref(p), nq))
    dws = hip.put(np.full(max(ws, 16), 0xFF, np.uint8))        # NaN: nothing may rely on a cleared workspace
    rc = eng.dpuf_amd_paged_attn(C.byref(b), C.byref(p), nq, dq.p, scale, out_t, do.p, dl.p if lse else None,
                                 dws.p if ws else None, ws, stream)
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    return R.from_type(do.get(), out_t), dl.get(), dq, dl, ws


def check(cache, nq, q, scale, out, lse, out_t):
    n = cache.n_rows
    ref, rl, A, S, vmax, _ = R.attention(cache, R.from_type(q, cache.t), scale, nq)
    bound = R.attention_bound(cache.t, out_t, ref, A, S, vmax, cache.hd, max(cache.ctx))
    err = np.abs(out[:n] - ref)
    worst = float((err / bound).max()) if err.size else 0.0
    say(f"  worst error {worst:.3f} of the bound")
    assert np.all(err <= bound)
    empty = np.isneginf(rl)
    assert np.array_equal(np.isneginf(lse[:n]), empty)
    assert np.all(out[:n][empty] == 0.0)
    dl = np.abs(lse[:n][~empty] - rl[~empty])
    assert np.all(dl <= R.score_error(S, cache.hd)[~empty] + np.abs(rl[~empty]) * 2.0 ** -22 + 2.0 ** -20)
    assert np.all(out[n:] == 7.5) and np.all(lse[n:] == 7.5)


# rows, contexts: a first token, lengths around 16, 32, 64 and 128, an empty sequence, one without new rows, one with
# more new rows than cached ones, a chunk of a longer context
RAGGED = ([1, 1, 0, 3, 1, 40, 2, 1, 0, 5], [1, 17, 0, 3, 130, 95, 64, 33, 50, 3])


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("nq,nkv,hd,page", [(4, 1, 64, 16), (4, 4, 128, 32), (10, 2, 128, 16), (8, 1, 256, 64),
                                            (16, 2, 64, 128), (32, 1, 128, 16), (14, 2, 64, 1024), (21, 7, 256, 16)])
def test_ragged(eng, hip, nq, nkv, hd, page, t):
    rng = np.random.default_rng(nq * 1000 + hd + t)
    cache = R.Cache(hip, rng, t, *RAGGED, nkv, hd, page, slots_first=bool(nq & 2))
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)) * 1.5, t)
    scale = float(np.float32(1 / np.sqrt(hd)))
    say(f"ragged: {nq}/{nkv} heads of {hd}, pages of {page}, type {t}")
    out, lse, *_ = call(eng, hip, cache, nq, q, scale, extra=3)
    check(cache, nq, q, scale, out, lse, t)


@pytest.mark.parametrize("max_ctx", [1, 700, 100000])
@pytest.mark.parametrize("hd,rows,ctx", [(128, [1, 1, 2], [1300, 5, 2111]), (64, [150], [1999]), (256, [70, 1], [1100, 900])])
def test_split_over_the_keys(eng, hip, hd, rows, ctx, max_ctx):
    """Long contexts of few rows go over several workgroups, whatever the
    caller's estimate of the longest context is."""
    rng = np.random.default_rng(hd + max_ctx)
    cache = R.Cache(hip, rng, R.BF16, rows, ctx, 2, hd, 32, table_extra=3100)
    q = R.to_type(rng.standard_normal((cache.n_rows, 6, hd)) * 1.5, R.BF16)
    say(f"split: hd {hd}, rows {rows}, contexts {ctx}, max_ctx {max_ctx}")
    out, lse, *_, ws = call(eng, hip, cache, 6, q, 0.11, out_t=R.F32, max_ctx=max_ctx)
    assert (ws > 0) == (max_ctx > 512)
    check(cache, 6, q, 0.11, out, lse, R.F32)


@pytest.mark.parametrize("rows,ctx", [([1, 2, 60], [90, 140, 180]), ([600], [700])])
def test_pages_outside_the_pool_are_absent(eng, hip, rows, ctx):
    rng = np.random.default_rng(5)
    bad = [(0, 1), (0, 4), (0, 5)] + ([(1, 0), (2, 3), (2, 7)] if len(ctx) > 1 else [(0, 0), (0, 43)])
    cache = R.Cache(hip, rng, R.F16, rows, ctx, 2, 64, 16, bad=bad)
    q = R.to_type(rng.standard_normal((cache.n_rows, 4, 64)), R.F16)
    say(f"bad pages: rows {rows}")
    out, lse, *_ = call(eng, hip, cache, 4, q, 0.125, extra=1)
    check(cache, 4, q, 0.125, out, lse, R.F16)


def test_lengths_beyond_the_table(eng, hip):
    """Lengths are clamped to the page table: a context of more rows than the
    table's pages hold reads those."""
    rng = np.random.default_rng(6)
    cache = R.Cache(hip, rng, R.BF16, [1, 4], [32, 32], 1, 64, 16, table_extra=0)
    q = R.to_type(rng.standard_normal((5, 2, 64)), R.BF16)
    say("lengths beyond the table")
    cache.d_ctx.set(np.array([2 ** 31 - 1, 40], np.int32))
    out, lse, *_ = call(eng, hip, cache, 2, q, 0.125)
    check(cache, 2, q, 0.125, out, lse, R.BF16)


def test_scores_far_apart(eng, hip):
    """Scores of a few hundred: the running maximum moves, what it left is 0."""
    rng = np.random.default_rng(8)
    for rows, ctx in (([1, 3], [300, 77]), ([90], [333])):
        cache = R.Cache(hip, rng, R.BF16, rows, ctx, 2, 128, 16, kscale=9.0)
        q = R.to_type(rng.standard_normal((cache.n_rows, 8, 128)) * 9.0, R.BF16)
        say(f"far scores: rows {rows}")
        out, lse, *_ = call(eng, hip, cache, 8, q, 0.088)
        check(cache, 8, q, 0.088, out, lse, R.BF16)


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("nq,nkv,hd,page", [(4, 1, 64, 16), (10, 2, 128, 32), (8, 1, 256, 64), (32, 1, 128, 16)])
def test_weights(eng, hip, nq, nkv, hd, page, t):
    rng = np.random.default_rng(nq + hd)
    bad = [(4, 3), (5, 0)] if page == 16 else []
    cache = R.Cache(hip, rng, t, *RAGGED, nkv, hd, page, slots_first=t == R.F16, bad=bad)
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)) * 1.5, t)
    scale, decay = 1 / np.sqrt(hd), 0.75
    say(f"weights: {nq}/{nkv} heads of {hd}, pages of {page}, type {t}")
    _, lse, dq, dl, _ = call(eng, hip, cache, nq, q, scale)
    _, rl, _, S, _, fresh = R.attention(cache, R.from_type(q, t), float(np.float32(scale)), nq)
    outs = []
    for w_in in (cache.dw, cache.dw, None):
        dst = hip.put(np.full_like(cache.w, -3.0))
        b, p = cache.batch(max_ctx=60), cache.pages(dw=dst)
        rc = eng.dpuf_amd_paged_attn_weights(C.byref(b), C.byref(p), nq, dq.p, scale, dl.p, decay,
                                             w_in.p if w_in else None, None)
        assert rc == 0, (rc, eng.dpuf_amd_last_error())
        outs.append(dst.get())
    assert np.array_equal(outs[0].view(np.uint32), outs[1].view(np.uint32))
    # exp(score - lse): two score errors, the lse's own rounding; sums of every row's share in fp32
    rel = 2 * R.score_error(S.max(initial=0), hd) + np.abs(rl[np.isfinite(rl)]).max() * 2.0 ** -22 + 2.0 ** -20
    rel += (max(cache.rows) * nq // nkv + 40) * 2.0 ** -24
    for out, d in ((outs[0], decay), (outs[2], 0.0)):
        left = np.ones_like(out, bool)
        for s, c in enumerate(cache.ctx):
            for i in range(c):
                if not cache.ok(s, i):
                    continue
                pg, r = cache.table[s, i // page], i % page
                left[pg, :, r] = False
                old = cache.w[pg, :, r].astype(np.float64) * d
                want = old + fresh[s][:, i]
                assert np.all(np.abs(out[pg, :, r] - want) <= rel * fresh[s][:, i] + 2.0 ** -22 * np.abs(old) + 1e-30), \
                    (s, i)
        assert np.all(out[left] == -3.0)
    # in place, and without new rows: the decay alone
    b, p = cache.batch(n_rows=0), cache.pages()
    assert eng.dpuf_amd_paged_attn_weights(C.byref(b), C.byref(p), nq, None, scale, None, decay, cache.dw.p, None) == 0
    got = cache.dw.get()
    for s, c in enumerate(cache.ctx):
        for i in range(c):
            if cache.ok(s, i):
                pg, r = cache.table[s, i // page], i % page
                assert np.array_equal(got[pg, :, r], cache.w[pg, :, r] * np.float32(decay))


# Every kernel and split of the keys: (rows, contexts, max_ctx given).  No more rows than sequences, with a sequence
# that has most of them; one sequence with fewer and more than 384 packed rows (4 heads a kv head), short and long;
# chunks beside decoding sequences.
MODES = {
    "few, split": ([0, 5, 0, 1, 0, 0], [40, 1300, 1, 700, 0, 9], None),
    "few, one row": ([1], [2111], None),
    "many": ([40], [95], None),
    "many, split": ([33], [1500], None),
    "wide, short keys": ([150], [333], 5000),
    "wide, split": ([97], [2300], None),
    "wide, few rows of them": ([0], [50], 4096),
    "mixed, split": ([1, 70, 2, 0, 1, 30], [1900, 1400, 600, 7, 33, 30], None),
}


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("mode", MODES)
def test_kernels_and_splits(eng, hip, mode, hd):
    """... and device row counts below n_rows: the rows behind stay."""
    rows, ctx, max_ctx = MODES[mode]
    rng = np.random.default_rng(len(mode) + hd)
    t = R.F16 if hd == 64 else R.BF16
    cache = R.Cache(hip, rng, t, rows, ctx, 2, hd, 32, slots_first=hd == 128, table_extra=160)
    q = R.to_type(rng.standard_normal((cache.n_rows, 8, hd)) * 1.5, t)
    extra = 100 if mode == "wide, few rows of them" else 0
    say(f"{mode}: hd {hd}")
    out, lse, *_ = call(eng, hip, cache, 8, q, 0.1, max_ctx=max_ctx, extra=extra)
    check(cache, 8, q, 0.1, out, lse, t)


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("mode", [m for m in MODES if m not in ("few, one row", "wide, few rows of them")])
def test_infinities_and_nan_that_a_row_does_not_see(eng, hip, mode, hd, t):
    """K and V rows of new tokens hold infinities and NaN: the rows before
    them, which do not see them, keep their values; those that do see them get
    what the definition gives."""
    rows, ctx, max_ctx = MODES[mode]
    rng = np.random.default_rng(2 * len(mode) + hd)
    nq, page = 8, 16
    cache = R.Cache(hip, rng, t, rows, ctx, 2, hd, page, table_extra=320)
    for s, (n, c) in enumerate(zip(rows, ctx)):
        for i in range(max(1, c - n + 1), c):
            pg, r = cache.table[s, i // page], i % page
            for h in range(2):
                at = rng.integers(0, hd, 3)
                cache.v[pg, h, r, at] = R.to_type([np.inf, -np.inf, np.nan], t)[rng.integers(0, 3, 3)]
        if n > 1:       # the last token's key: only the last row sees it
            cache.k[cache.table[s, (c - 1) // page], 1, (c - 1) % page, 3] = R.to_type([np.nan], t)[0]
    cache.dv.set(cache.v)
    cache.dk.set(cache.k)
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)), t)
    say(f"odd values, {mode}: hd {hd}, type {t}")
    out, lse, *_ = call(eng, hip, cache, nq, q, 0.1, max_ctx=max_ctx)
    with np.errstate(all="ignore"):
        ref, rl, A, S, _, _ = R.attention(cache, R.from_type(q, t), 0.1, nq)
        # the values themselves are below 10 (standard normal)
        bound = R.attention_bound(t, t, ref, A, S, np.full(S.shape, 10.0), hd, max(ctx))
        assert np.array_equal(np.isnan(out), np.isnan(ref))
        assert np.array_equal(np.isposinf(out), np.isposinf(ref)) and np.array_equal(np.isneginf(out), np.isneginf(ref))
        ok = np.isfinite(ref)
        assert ok.any() and not ok.all()
        assert np.all(np.abs(out[ok] - ref[ok]) <= bound[ok])
        assert np.array_equal(np.isnan(lse), np.isnan(rl)) and np.array_equal(np.isneginf(lse), np.isneginf(rl))


@pytest.mark.parametrize("max_ctx", [60, 6000, 20000])
@pytest.mark.parametrize("nq,hd,rows,ctx", [(6, 64, [71], [300]), (2, 128, [200, 0, 1], [260, 40, 90]),
                                            (16, 128, [50], [50]), (10, 256, [40], [333])])
def test_weights_of_chunks(eng, hip, nq, hd, rows, ctx, max_ctx):
    """Chunks of a prompt, over every split of the keys among workgroups."""
    rng = np.random.default_rng(nq + hd)
    t = R.F16 if nq == 6 else R.BF16
    cache = R.Cache(hip, rng, t, rows, ctx, 2, hd, 16, table_extra=1300, bad=[(0, 1)])
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)) * 1.5, t)
    say(f"weights of chunks: hd {hd}, rows {rows}, contexts {ctx}, max_ctx {max_ctx}")
    _, lse, dq, dl, _ = call(eng, hip, cache, nq, q, 0.1)
    _, rl, _, S, _, fresh = R.attention(cache, R.from_type(q, t), float(np.float32(0.1)), nq)
    dst = hip.put(np.full_like(cache.w, -3.0))
    b, p = cache.batch(max_ctx=max_ctx), cache.pages(dw=dst)
    rc = eng.dpuf_amd_paged_attn_weights(C.byref(b), C.byref(p), nq, dq.p, 0.1, dl.p, 0.5, cache.dw.p, None)
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    out = dst.get()
    # as for test_weights
    rel = 2 * R.score_error(S.max(initial=0), hd) + np.abs(rl[np.isfinite(rl)]).max() * 2.0 ** -22 + 2.0 ** -20
    rel += (max(rows) * nq // 2 + 40) * 2.0 ** -24
    for s, c in enumerate(ctx):
        for i in range(c):
            if not cache.ok(s, i):
                continue
            pg, r = cache.table[s, i // 16], i % 16
            old = cache.w[pg, :, r].astype(np.float64) * 0.5
            assert np.all(np.abs(out[pg, :, r] - old - fresh[s][:, i]) <=
                          rel * fresh[s][:, i] + 2.0 ** -22 * np.abs(old) + 1e-30), (s, i)
            out[pg, :, r] = -3.0
    assert np.all(out == -3.0)


def test_two_streams_and_a_graph(eng, hip):
    """Two calls at once on streams of their own with workspaces of their own;
    then a captured call replayed over new lengths and values between eager
    calls gives what the eager call gives."""
    rng = np.random.default_rng(11)
    nq, hd = 8, 128
    caches = [R.Cache(hip, rng, R.BF16, rows, ctx, 2, hd, 32) for rows, ctx in
              (([1, 1, 1], [900, 1500, 3]), ([200, 1], [800, 700]))]
    work = []
    for cache in caches:
        q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)) * 1.5, R.BF16)
        b, p = cache.batch(), cache.pages(w=False)
        n = int(eng.dpuf_amd_paged_attn_workspace(C.byref(b), C.byref(p), nq))
        work.append((cache, q, hip.put(q), hip.put(np.zeros((cache.n_rows, nq, hd), np.uint16)),
                     hip.put(np.zeros((cache.n_rows, nq), np.float32)), hip.put(np.zeros(max(16, n), np.uint8)), n, b,
                     p, hip.stream()))

    def launch(wk, s):
        cache, q, dq, do, dl, ws, n, b, p, _ = wk
        assert eng.dpuf_amd_paged_attn(C.byref(b), C.byref(p), nq, dq.p, 0.09, R.BF16, do.p, dl.p, ws.p, n, s) == 0

    say("two streams")
    for _ in range(3):
        for wk in work:
            launch(wk, wk[-1])
    for wk in work:
        assert hip.lib.hipStreamSynchronize(wk[-1]) == 0
        check(wk[0], nq, wk[1], 0.09, R.from_type(wk[3].get(), R.BF16), wk[4].get(), R.BF16)
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
        check(cache, nq, q, 0.09, R.from_type(got, R.BF16), gl, R.BF16)
        launch(wk, s)
        assert hip.lib.hipStreamSynchronize(s) == 0
        assert np.array_equal(do.get(), got) and np.array_equal(dl.get().view(np.uint32), gl.view(np.uint32))
    hip.lib.hipGraphExecDestroy(ge)
    hip.lib.hipGraphDestroy(graph)
    for wk in work:
        hip.lib.hipStreamDestroy(wk[-1])


def test_host_memory_is_refused(eng, hip):
    rng = np.random.default_rng(12)
    cache = R.Cache(hip, rng, R.BF16, [1], [20], 1, 64, 16)
    q = hip.put(np.zeros((1, 1, 64), np.uint16))
    out = hip.put(np.zeros((1, 1, 64), np.uint16))
    host = np.zeros(4096, np.int32)
    b, p = cache.batch(), cache.pages(w=False)
    ok = lambda: eng.dpuf_amd_paged_attn(C.byref(b), C.byref(p), 1, q.p, 1.0, R.BF16, out.p, None, None, 0, None)
    assert ok() == 0
    for name in ("row_start", "ctx_len", "page_table"):
        keep = getattr(b, name)
        setattr(b, name, host.ctypes.data)
        assert ok() == -1, name
        setattr(b, name, keep)
    p.k = host.ctypes.data & ~15
    assert ok() == -1
    hip.sync()


def weights_of(eng, hip, cache, nq, q, scale, max_ctx=None):
    """pages->w of one call from nothing, [page][kv head][row]."""
    _, lse, dq, dl, _ = call(eng, hip, cache, nq, q, scale)
    dst = hip.put(np.full_like(cache.w, -3.0))
    b, p = cache.batch(max_ctx=max_ctx), cache.pages(dw=dst)
    assert eng.dpuf_amd_paged_attn_weights(C.byref(b), C.byref(p), nq, dq.p, scale, dl.p, 1.0, None, None) == 0
    return dst.get()


# batches for the few-row kernel, the other, and both, and max_ctx for its tiles of 128, 64 and 32 keys
ODD = [([1, 3, 1], [200, 90, 40], None), ([70], [300], 30000), ([70], [300], 6000), ([70], [300], 300),
       ([90, 1, 1, 1], [333, 250, 40, 33], 100000)]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,ctx,max_ctx", ODD)
def test_weights_of_keys_that_score_minus_infinity(eng, hip, rows, ctx, max_ctx, hd):
    """An infinite element of a key that every query has with the other sign:
    each row gives that key nothing, and the others what they get without it."""
    rng = np.random.default_rng(hd + len(rows))
    nq = 10
    cache = R.Cache(hip, rng, R.BF16, rows, ctx, 2, hd, 16, table_extra=6300)
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)), R.BF16)
    q[..., 5] = R.to_type(-0.5, R.BF16)
    for s, i in ((0, 0), (0, 17), (0, ctx[0] - rows[0] - 1)):
        cache.k[cache.table[s, i // 16], :, i % 16, 5] = R.to_type([np.inf], R.BF16)[0]
    cache.dk.set(cache.k)
    say(f"scores of -infinity: rows {rows}, contexts {ctx}, max_ctx {max_ctx}, hd {hd}")
    got = weights_of(eng, hip, cache, nq, q, 0.1, max_ctx)
    with np.errstate(all="ignore"):
        _, rl, _, _, _, fresh = R.attention(cache, R.from_type(q, R.BF16), float(np.float32(0.1)), nq)
    # |q| and |k| below 6 (standard normal): as the weights' own tests
    rel = 2 * R.score_error(36.0 * hd * 0.1, hd) + np.abs(rl[np.isfinite(rl)]).max() * 2.0 ** -22 + 2.0 ** -20
    rel += (max(rows) * nq // 2 + 40) * 2.0 ** -24
    for s, c in enumerate(ctx):
        for i in range(c):
            w = got[cache.table[s, i // 16], :, i % 16]
            assert np.all(np.abs(w - fresh[s][:, i]) <= rel * fresh[s][:, i] + 1e-30), (s, i, w, fresh[s][:, i])


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,ctx,max_ctx", ODD)
def test_weights_of_keys_behind_a_row_without_a_number(eng, hip, rows, ctx, max_ctx, hd):
    """A query with NaN gives NaN to the keys that its row sees, and to no
    others: those keep the bits that they have with another query there."""
    rng = np.random.default_rng(2 * hd + len(rows))
    nq, row, head = 10, max(rows) // 2, 7
    s = int(np.argmax(rows))
    cache = R.Cache(hip, rng, R.F16, rows, ctx, 2, hd, 16, table_extra=6300)
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)), R.F16)
    want = weights_of(eng, hip, cache, nq, q, 0.1, max_ctx)
    q[cache.starts[s] + row, head, 3] = R.to_type([np.nan], R.F16)[0]
    say(f"a row of NaN: rows {rows}, contexts {ctx}, max_ctx {max_ctx}, hd {hd}")
    got = weights_of(eng, hip, cache, nq, q, 0.1, max_ctx)
    for i in range(ctx[s] - rows[s] + row + 1):
        at = cache.table[s, i // 16], head // (nq // 2), i % 16
        assert np.isnan(got[at]), i
        got[at] = want[at]
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,ctx,max_ctx", [([1, 1], [400, 3], None), ([1], [2000], None), ([40], [700], 300),
                                              ([97], [2300], None), ([1, 70], [400, 500], 500)])
def test_fp16_probabilities_far_below_the_largest(eng, hip, rows, ctx, max_ctx, hd):
    """One key 2^20 times as likely as the others, with nothing in its value:
    the others' probabilities, all below fp16's normal numbers, are what there
    is, and keep a relative half step each."""
    rng = np.random.default_rng(hd)
    nq, scale = 4, 0.125
    cache = R.Cache(hip, rng, R.F16, rows, ctx, 1, hd, 16, table_extra=150)
    n = cache.n_rows
    # score of key 0: scale * 8 * x, of the others 0; x so that exp(score) is
    # 2^24 / 16.5: halfway between two of fp16's subnormal numbers
    q = np.zeros((n, nq, hd))
    q[..., 0], q[..., 1] = 8.0, 2.0 ** -10
    score = np.log(2.0 ** 24 / 16.5)
    hi = float(np.float16(score))
    lo = float(np.float16((score - hi) * 2.0 ** 13))
    for s, c in enumerate(ctx):
        for i in range(c):
            pg, r = cache.table[s, i // 16], i % 16
            cache.k[pg, :, r] = 0
            cache.v[pg, :, r] = R.to_type(1 + 0.1 * rng.standard_normal(hd), R.F16)
            if i == 0:
                cache.k[pg, 0, r, :2] = R.to_type([hi, lo], R.F16)
                cache.v[pg, :, r] = 0
    cache.dk.set(cache.k)
    cache.dv.set(cache.v)
    q = R.to_type(q, R.F16)
    say(f"far below the largest: rows {rows}, contexts {ctx}, max_ctx {max_ctx}, hd {hd}")
    out, lse, *_ = call(eng, hip, cache, nq, q, scale, out_t=R.F32, max_ctx=max_ctx)
    ref, rl, A, S, _, _ = R.attention(cache, R.from_type(q, R.F16), scale, nq)
    # attention_bound without the share of rounded-off terms: 2^-20 of the largest times 2^9 is a normal number
    d = R.score_error(S, hd)[..., None]
    bound = A * (R.HALF_STEP[R.F16] + 2 * d + (max(ctx) + 64) * 2.0 ** -24) * 1.01 + 1e-30
    err = np.abs(out - ref)
    say(f"  worst error {float((err / bound).max()):.3f} of the bound")
    assert np.all(err <= bound)
    assert np.all(np.abs(lse - rl) <= R.score_error(S, hd) + np.abs(rl) * 2.0 ** -22 + 2.0 ** -20)


@pytest.mark.parametrize("nkv,seqs", [(2, 1), (8, 8), (8, 9)])
@pytest.mark.parametrize("ctx", [255, 256, 257, 300, 511, 512, 513])
def test_short_contexts(eng, hip, ctx, nkv, seqs):
    """One range of keys and a few, at the lengths where that changes."""
    rng = np.random.default_rng(ctx + seqs)
    cache = R.Cache(hip, rng, R.BF16, [1] * seqs, [ctx] + [7] * (seqs - 1), nkv, 64, 16)
    nq = 2 * nkv
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, 64)) * 1.5, R.BF16)
    say(f"short contexts: {ctx} keys, {seqs} sequences of {nkv} kv heads")
    out, lse, *_, ws = call(eng, hip, cache, nq, q, 0.125)
    assert (ws > 0) == (ctx > (256 if seqs * nkv <= 64 else 512))
    check(cache, nq, q, 0.125, out, lse, R.BF16)


DECODE = [([1], [75]), ([1, 1, 1], [900, 3, 2111]), ([1, 70, 1, 1], [700, 90, 33, 400]), ([0, 3, 0, 1], [5, 50, 0, 300])]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,ctx", DECODE)
def test_decoding_rows_keep_their_probabilities(eng, hip, rows, ctx, hd):
    """bf16 pages, outputs in fp32: decoding sequences' probabilities are held
    in two terms, so that their outputs are off by far less than bf16's step."""
    rng = np.random.default_rng(hd + sum(ctx))
    nq, nkv = 8, 2
    cache = R.Cache(hip, rng, R.BF16, rows, ctx, nkv, hd, 16)
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)) * 1.5, R.BF16)
    say(f"two terms: rows {rows}, contexts {ctx}, hd {hd}")
    out, lse, *_ = call(eng, hip, cache, nq, q, 0.1, out_t=R.F32)
    ref, rl, A, S, _, _ = R.attention(cache, R.from_type(q, R.BF16), float(np.float32(0.1)), nq)
    # what the first term leaves is at most 2^-7 of a probability, and rounded by 2^-8 of that; the rest as in
    # attention_bound
    d = R.score_error(S, hd)[..., None]
    bound = A * (2.0 ** -15 + 2.0 ** -24 + 2 * d + (max(ctx) + 64) * 2.0 ** -24) * 1.01 + 1e-30
    for s, (r, c) in enumerate(zip(rows, ctx)):
        if r * nq // nkv > 16 and sum(rows) > len(rows):      # a chunk: rounded once
            continue
        at = slice(cache.starts[s], cache.starts[s + 1])
        assert np.all(np.abs(out[at] - ref[at]) <= bound[at]), s


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,ctx,max_ctx", [([1, 1], [400, 90], None), ([1], [3000], None), ([40], [700], None),
                                              ([97], [2300], None), ([1, 70], [400, 500], None)])
def test_infinities_that_all_rows_see(eng, hip, rows, ctx, max_ctx, hd, t):
    """Infinities and NaN in values of old keys, in tiles that every row sees
    whole: infinite of their sign, NaN where both meet."""
    rng = np.random.default_rng(hd + t)
    nq, nkv = 8, 2
    cache = R.Cache(hip, rng, t, rows, ctx, nkv, hd, 16)
    inf, nan = R.to_type([np.inf, -np.inf, np.nan], t)[:2], R.to_type([np.nan], t)[0]
    for s in range(len(ctx)):
        for i, col, x in ((0, 1, inf[0]), (9, 2, inf[1]), (20, 3, inf[0]), (21, 3, inf[1]), (16, 4, nan), (5, 6, inf[0]),
                          (17, 6, inf[0])):
            cache.row(cache.v, cache.table[s, i // 16], i % 16)[:, col] = x
    cache.dv.set(cache.v)
    q = R.to_type(rng.standard_normal((cache.n_rows, nq, hd)) * 0.5, t)
    say(f"infinities: rows {rows}, contexts {ctx}, hd {hd}, type {t}")
    out, lse, *_ = call(eng, hip, cache, nq, q, 0.1, out_t=R.F32, max_ctx=max_ctx)
    with np.errstate(all="ignore"):
        ref, rl, A, S, _, _ = R.attention(cache, R.from_type(q, t), float(np.float32(0.1)), nq)
    assert np.isposinf(ref).any() and np.isneginf(ref).any() and np.isnan(ref).any()
    for kind in (np.isnan, np.isposinf, np.isneginf):
        assert np.array_equal(kind(out), kind(ref))
    # finite values are below 10 (standard normal)
    ok = np.isfinite(ref)
    with np.errstate(all="ignore"):
        bound = R.attention_bound(t, R.F32, ref, A, S, np.full(S.shape, 10.0), hd, max(ctx))
    assert np.all(np.abs(out[ok] - ref[ok]) <= bound[ok])


def test_huge_values_that_a_row_does_not_see(eng, hip):
    """bf16's largest numbers behind a row's last key, and in absent pages,
    reach it by no share of them, however small."""
    rng = np.random.default_rng(5)
    for rows, ctx in (([1, 3, 0, 1], [33, 20, 4, 100]), ([30], [70])):
        cache = R.Cache(hip, rng, R.BF16, rows, ctx, 2, 128, 16, bad=[(0, 1)])
        q = R.to_type(rng.standard_normal((cache.n_rows, 8, 128)), R.BF16)
        outs = []
        for huge in (False, True):
            if huge:
                seen = np.zeros(cache.v.shape, bool)
                for s, (r, c) in enumerate(zip(rows, ctx)):
                    for i in range(c - r + 1 if r else 0):
                        if cache.ok(s, i):
                            seen[cache.table[s, i // 16], :, i % 16] = True
                cache.v = np.where(seen, cache.v, R.to_type([3.3e38], R.BF16)[0])
                cache.dv.set(cache.v)
            say(f"huge values {huge}: rows {rows}")
            out, lse, *_ = call(eng, hip, cache, 8, q, 0.1, out_t=R.F32)
            outs.append(out[[int(cache.starts[s]) for s in range(len(rows)) if rows[s]]])
        assert np.array_equal(outs[0], outs[1])
