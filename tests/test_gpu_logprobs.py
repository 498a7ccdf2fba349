"""Log probabilities of given tokens, entropy and the largest alternatives of
rows of logits, against float64 from the definition."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu

F = np.float32


@pytest.fixture()
def hip(eng):
    h = R.Hip()
    yield h
    h.free_all()


def say(*a):
    print(*a, flush=True)


def reference(x, targets, k):
    """(ln p of targets, entropy, top tokens, their ln p, ln l, E|d|) of a row of float64 logits."""
    x = np.where(np.isnan(x), -np.inf, x)
    V, m = len(x), x.max()
    lp = np.full(V, -np.inf)
    log_l = spread = 0.0
    if m == np.inf:
        lp[x == np.inf] = -np.log((x == np.inf).sum())
        log_l = -lp.max()
    elif m > -np.inf:
        d = x - m
        e = np.exp(d)
        log_l = np.log(e.sum())
        lp = d - log_l
        on = e > 0
        spread = float((e[on] * -d[on]).sum() / e.sum())
    p = np.exp(lp)
    entropy = -float((p[p > 0] * lp[p > 0]).sum())
    order = np.argsort(-x, kind="stable")[:k]
    order = order[x[order] > -np.inf]
    top = np.full(k, -1)
    top[:len(order)] = order
    tl = np.full(k, -np.inf)
    tl[:len(order)] = lp[order]
    inside = (targets >= 0) & (targets < V)
    tp = np.where(inside, lp[np.where(inside, targets, 0)], -np.inf)
    return tp, entropy, top, tl, log_l, spread


def run(eng, hip, x, t, targets=None, k=0, stride=None, offset=0, entropy=True, stream=None, want=True):
    """One call, checked; returns its outputs."""
    n, V = x.shape
    store = R.to_type(x, t)
    stride = V if stride is None else stride
    full = R.to_type(np.full((n, stride), 60.0, F), t)        # what lies between rows would change everything
    full[:, :V] = store
    d = hip.put(full, offset)
    nt = targets.shape[1] if targets is not None else 0
    dt = hip.put(np.ascontiguousarray(targets, np.int32)) if nt else None
    lp, en = hip.put(np.full((n, nt), 9.0, F)), hip.put(np.full(n, 9.0, F))
    top, tl = hip.put(np.full((n, k), -9, np.int32)), hip.put(np.full((n, k), 9.0, F))
    ws = int(eng.dpuf_amd_logprobs_workspace(n, V, k))
    dws = hip.put(np.full(max(ws, 16), 0xFF, np.uint8))
    rc = eng.dpuf_amd_logprobs(t, n, V, stride, d.p, nt, dt.p if nt else None, k, lp.p if nt else None,
                               en.p if entropy else None, top.p if k else None, tl.p if k else None, dws.p, ws, stream)
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    got = lp.get(), en.get(), top.get(), tl.get()
    if want:
        check(R.from_type(store, t).reshape(n, V), targets, k, got, entropy)
    hip.free_all()
    return got


def check(x64, targets, k, got, entropy=True):
    lp, en, top, tl = got
    # l: a thread adds at most 128 terms and their quarters, 6 + 2 pairs and a chunk's threads meet, 512 chunks at
    # most of which a thread adds two, 8 more pairs, and no more than 40 of these move by an exponential (2^-22)
    sums = (128 + 32 + 40) * 2.0 ** -24 + 40 * 2.0 ** -22
    for i in range(len(x64)):
        tg = targets[i] if targets is not None else np.zeros(0, int)
        tp, we, wt, wl, log_l, spread = reference(x64[i], tg, k)
        # a term: the difference and its product with log2 e round by half a step of d each, the constant by another
        rel = sums + 2.0 ** -22 + 3 * 2.0 ** -24 * (spread + 1)
        fin = lambda a: np.where(np.isfinite(a), np.abs(a), 0.0)
        for a, b in ((lp[i], tp), (tl[i], wl)):
            if not a.size:
                continue
            assert np.array_equal(np.isneginf(a), np.isneginf(b)), i
            on = np.isfinite(b)
            assert np.all(np.abs(a[on] - b[on]) <= rel + (2 * fin(b[on]) + 3 * log_l) * 2.0 ** -23 + 2.0 ** -24), i
        assert np.array_equal(top[i], wt), (i, top[i], wt)
        if entropy:
            # u / l: l's error and u's, both relative to sums of one sign, and ln l's
            assert abs(en[i] - we) <= (2 * rel + 2.0 ** -22) * (spread + 7) + 3 * log_l * 2.0 ** -23 + 2.0 ** -24, i
        else:
            assert np.all(en == 9.0)


def logits(rng, n, V, spread=2.5):
    x = rng.standard_normal((n, V)).astype(F) * F(spread)
    for i in range(n):
        hot = rng.integers(0, V, max(1, V // 50))[:20]
        x[i, hot] += rng.random(len(hot)).astype(F) * 9
    return x


@pytest.mark.parametrize("t", [R.F32, R.BF16, R.F16])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 129, 1000, 4099, 32003, 151936])
def test_sizes(eng, hip, V, t):
    rng = np.random.default_rng(V + t)
    for n, nt, k in ((1, 1, 20), (5, 3, 0), (3, 0, 1), (2, 70, 64), (7, 2, 5)):
        say(f"logprobs: {n} rows of {V}, type {t}, {nt} targets, {k} alternatives")
        targets = rng.integers(0, V, (n, nt)) if nt else None
        run(eng, hip, logits(rng, n, V), t, targets, k, entropy=n != 5)


@pytest.mark.parametrize("t", [R.F32, R.BF16, R.F16])
def test_strides_and_alignment(eng, hip, t):
    rng = np.random.default_rng(5)
    es = 4 if t == R.F32 else 2
    for stride, offset in ((1001, 0), (1003, es), (1024, 8), (1024, 0), (1016, 3 * es), (1001, 7 * es)):
        say(f"logprobs: rows {stride} apart, {offset} bytes in, type {t}")
        run(eng, hip, logits(rng, 5, 1001), t, rng.integers(0, 1001, (5, 4)), 9, stride=stride, offset=offset)


@pytest.mark.parametrize("V", [50, 20000])
def test_ties(eng, hip, V):
    """Few distinct values, all equal, both zeros: the lowest indices first."""
    rng = np.random.default_rng(6)
    x = rng.integers(-2, 3, (8, V)).astype(F)
    x[3:6] = 1.25
    x[6] = np.where(np.arange(V) % 2, 0.0, -0.0)
    x[7, :] = -1.0
    x[7, V // 2:] = 1.0
    for k in (1, 20, 64):
        for t in (R.F32, R.BF16):
            say(f"ties: V {V}, {k} alternatives, type {t}")
            run(eng, hip, x, t, rng.integers(0, V, (8, 2)), k)


@pytest.mark.parametrize("k", [32, 33, 64])
@pytest.mark.parametrize("t", [R.F32, R.BF16])
def test_long_runs_of_equal_logits(eng, hip, t, k):
    """More equal ones than a workgroup lists: with fewer larger ones than
    alternatives, a few distinct values, all that is left after a mask, and what
    lies with few of the threads; rows cut and not."""
    rng = np.random.default_rng(k)
    V = 70001
    x = np.zeros((8, V), F)
    x[1, rng.permutation(V)[:k - 1]] = 2 + rng.integers(0, 4, k - 1)
    x[2] = rng.integers(-2, 3, V)
    x[3, :V // 2] = -np.inf
    x[4] = -np.inf
    x[4, V - 5000:] = 0.5
    x[5] = np.nan
    x[5, 4096:4096 + 2000] = -1.0
    x[6, V - 40:] = 1.0
    x[7] = np.where(np.arange(V) % 1024 < 64, 3.0, 0.0)
    targets = rng.integers(0, V, (8, 2))
    say(f"long runs of equal logits: {k} alternatives, type {t}")
    run(eng, hip, x, t, targets, k)
    rows = np.arange(400) % 8
    got = run(eng, hip, x[rows], t, targets[rows], k, want=False)
    check(R.from_type(R.to_type(x, t), t).reshape(x.shape), targets, k, [g[:8] for g in got])
    for g in got:
        assert np.array_equal(g.view(np.uint32), g[rows].view(np.uint32))


def test_masked_and_odd_logits(eng, hip):
    """-infinity (a grammar's mask), NaN, +infinity, rows that leave nothing,
    the lowest finite value as a mask, huge values."""
    rng = np.random.default_rng(7)
    V = 6000
    x = logits(rng, 14, V)
    x[0, :] = -np.inf
    x[1, :] = np.nan
    x[2, rng.permutation(V)[:V - 5]] = -np.inf
    x[3, ::2] = np.nan
    x[4, [7, 90]] = np.inf
    x[5, rng.permutation(V)[:V - 3]] = np.finfo(F).min
    x[6, :] = np.finfo(F).min
    x[7, 1:] = -np.inf
    x[8] *= F(1e30)
    x[9, :] = np.finfo(F).max
    x[10, :4096] = -np.inf
    x[11, 4096:] = np.nan
    x[12, :] = np.inf
    x[13, 5000] = np.inf
    x[13, :100] = np.nan
    targets = np.concatenate([rng.integers(0, V, (14, 6)), np.tile([7, 90, 0, -1, V, 2 ** 31 - 1, -2 ** 31, 7], (14, 1))], 1)
    for k in (0, 3, 20, 64):
        say(f"odd logits, {k} alternatives")
        run(eng, hip, x, R.F32, targets, k)
    # the 16-bit types' own lowest values
    for t, low in ((R.BF16, -3.3895314e38), (R.F16, -65504.0)):
        y = logits(rng, 5, V)
        y[0, rng.permutation(V)[:V - 3]] = low
        y[1, :] = low
        y[2, ::3] = -np.inf
        y[3, :] = np.nan
        y[4, 5] = np.inf
        say(f"odd logits, type {t}")
        run(eng, hip, y, t, targets[:5], 20)


def test_signalling_nan(eng, hip):
    """Any NaN pattern is -infinity."""
    rng = np.random.default_rng(8)
    V = 3001
    x = logits(rng, 3, V)
    at = rng.permutation(V)[:1500]
    x.view(np.uint32)[:, at] = rng.choice(np.array([0x7F800001, 0xFF800001, 0x7FBFFFFF, 0x7FC00000, 0xFFFFFFFF], np.uint32),
                                          (3, 1500))
    say("NaN of every kind")
    run(eng, hip, x, R.F32, rng.integers(0, V, (3, 9)), 20)


@pytest.mark.parametrize("t", [R.F32, R.BF16])
def test_alternatives_that_crowd(eng, hip, t):
    """Masks that leave some threads of the workgroup nothing, so that the
    bound that others have says nothing, and the largest logits side by side."""
    rng = np.random.default_rng(9)
    V = 60000
    x = logits(rng, 6, V, 1.0)
    i = np.arange(V)
    x[0, i % 64 < 4] = -np.inf
    x[1, i % 64 >= 4] = -np.inf
    x[2, i % 256 != 77] = -np.inf
    x[3, 7000:7200] = 5 + rng.random(200)
    x[4, ::64] = 5 + rng.random(len(i[::64]))
    x[5, ::256] = 5 + 0.001 * np.arange(len(i[::256]))
    for k in (1, 20, 63, 64):
        say(f"crowds: {k} alternatives, type {t}")
        run(eng, hip, x, t, rng.integers(0, V, (6, 1)), k)


@pytest.mark.parametrize("t,V", [(R.F32, 300001), (R.BF16, 400003), (R.F32, 1 << 19), (R.F32, (1 << 20) + 3), (R.F16, (1 << 21) + 5), (R.F32, 1 << 24), (R.BF16, 1 << 24)])
def test_large_vocabularies(eng, hip, t, V):
    rng = np.random.default_rng(10)
    x = rng.standard_normal((1, V)).astype(F)
    x[0, V - 1] = 9.0
    say(f"logprobs: V {V}, type {t}")
    for k in (20, 64):
        run(eng, hip, x, t, np.array([[0, V - 1, V // 2]]), k)


@pytest.mark.parametrize("n,V,k", [(65536, 5, 2), (700, 300, 20), (3000, 1100, 0), (513, 9000, 5)])
def test_many_rows(eng, hip, n, V, k):
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((n, V)) * 3).astype(F)
    say(f"logprobs: {n} rows of {V}")
    targets = rng.integers(0, V, (n, 1))
    got = run(eng, hip, x, R.F32, targets, k, want=n < 1000)
    some = np.unique(np.concatenate([rng.integers(0, n, 40), [0, n - 1]]))
    check(x[some].astype(np.float64), targets[some], k, [g[some] for g in got])
    p = np.exp((x - x.max(1, keepdims=True)).astype(np.float64))
    lp = np.log(np.take_along_axis(p, targets, 1) / p.sum(1, keepdims=True))
    assert np.all(np.abs(got[0] - lp) < 1e-4)


@pytest.mark.parametrize("t,n,V,k", [(R.F32, 300, 20001, 20), (R.BF16, 256, 65536, 64), (R.F16, 384, 70001, 5),
                                     (R.BF16, 390, 151936, 20), (R.F32, 255, 20001, 33), (R.F32, 383, 70000, 0)])
def test_rows_that_a_workgroup_each_takes(eng, hip, t, n, V, k):
    """Around the numbers of rows from which a row is not cut; a thousand
    targets and more than a workgroup's threads."""
    rng = np.random.default_rng(n + V)
    x = (rng.standard_normal((n, V), np.float32) * 3).astype(F)
    x[1] = -np.inf
    x[2, ::2] = np.nan
    x[3] = 1e9
    say(f"logprobs: {n} rows of {V}, type {t}, {k} alternatives")
    targets = rng.integers(-1, V + 1, (n, 1024 if n < 300 else 257))
    got = run(eng, hip, x, t, targets, k, want=False)
    some = np.unique(np.concatenate([rng.integers(0, n, 8), [0, 1, 2, 3, n - 1]]))
    check(R.from_type(R.to_type(x[some], t), t).reshape(len(some), V), targets[some], k, [g[some] for g in got])


def test_flat_and_sharp_rows(eng, hip):
    """Equal logits (entropy ln V), a single likely token (entropy near 0, never
    below), logits far from 0, and logits that rise to the end."""
    V = 151936
    x = np.zeros((6, V), F)
    x[1] = 1000.25
    x[2, 77] = 100.0
    x[3] = np.linspace(-300, 300, V)
    x[4] = np.linspace(300, -300, V)
    x[5] = -5e4
    x[5, 9] = -4.9e4
    say("flat and sharp rows")
    got = run(eng, hip, x, R.F32, np.tile([77, 0, V - 1, 9], (6, 1)), 20)
    assert np.all(got[1] >= 0)


def test_two_streams_and_a_graph(eng, hip):
    """Two calls at once; a captured call replayed over new logits and targets
    between eager calls; the same inputs give the same bits."""
    rng = np.random.default_rng(11)
    shapes = [(3, 50001, R.F32, 20), (70, 9000, R.BF16, 7)]
    work = []
    for n, V, t, k in shapes:
        ws = int(eng.dpuf_amd_logprobs_workspace(n, V, k))
        work.append(dict(n=n, V=V, t=t, k=k, x=hip.put(R.to_type(logits(rng, n, V), t)),
                         tg=hip.put(rng.integers(0, V, (n, 2)).astype(np.int32)), lp=hip.put(np.zeros((n, 2), F)),
                         en=hip.put(np.zeros(n, F)), top=hip.put(np.zeros((n, k), np.int32)),
                         tl=hip.put(np.zeros((n, k), F)), ws=hip.put(np.zeros(max(ws, 16), np.uint8)), size=ws,
                         s=hip.stream()))

    def launch(w):
        assert eng.dpuf_amd_logprobs(w["t"], w["n"], w["V"], w["V"], w["x"].p, 2, w["tg"].p, w["k"], w["lp"].p, w["en"].p,
                                     w["top"].p, w["tl"].p, w["ws"].p, w["size"], w["s"]) == 0

    def outputs(w):
        assert hip.lib.hipStreamSynchronize(w["s"]) == 0
        return [w[o].get() for o in ("lp", "en", "top", "tl")]

    def right(w, got):
        check(R.from_type(w["x"].get(), w["t"]), w["tg"].get(), w["k"], got)

    say("two streams")
    for _ in range(3):
        for w in work:
            launch(w)
    for w in work:
        right(w, outputs(w))
    say("graph")
    for w in work:
        graph, ge = C.c_void_p(), C.c_void_p()
        assert hip.lib.hipStreamBeginCapture(w["s"], 1) == 0
        launch(w)
        assert hip.lib.hipStreamEndCapture(w["s"], C.byref(graph)) == 0
        assert hip.lib.hipGraphInstantiate(C.byref(ge), graph, None, None, 0) == 0
        for _ in range(3):
            w["x"].set(R.to_type(logits(rng, w["n"], w["V"]), w["t"]))
            w["tg"].set(rng.integers(0, w["V"], (w["n"], 2)).astype(np.int32))
            assert hip.lib.hipGraphLaunch(ge, w["s"]) == 0
            a = outputs(w)
            right(w, a)
            launch(w)
            for p, q in zip(a, outputs(w)):
                assert np.array_equal(p.view(np.uint32), q.view(np.uint32))
        hip.lib.hipGraphExecDestroy(ge)
        hip.lib.hipGraphDestroy(graph)
        hip.lib.hipStreamDestroy(w["s"])


@pytest.mark.parametrize("t", [R.F32, R.BF16, R.F16])
@pytest.mark.parametrize("V,n", [(5, 1500), (5000, 40), (40000, 12), (300000, 2)])
def test_no_log_probability_is_above_zero(eng, hip, V, n, t):
    """Rows of one finite logit, and rows where one token has nearly all the
    weight: ln p is 0 at most, of targets and of alternatives."""
    rng = np.random.default_rng(V + t)
    hot = rng.integers(0, V, n)
    x = np.full((n, V), -np.inf, F)
    x[1::2] = (rng.standard_normal((len(x[1::2]), V)) - 40).astype(F)
    x[np.arange(n), hot] = (5 + 55 * rng.random(n)).astype(F)
    say(f"one token alone: {n} rows of {V}, type {t}")
    for k in (0, 1, 33):
        lp, en, top, tl = run(eng, hip, x, t, np.stack([hot, rng.integers(0, V, n)], 1), k)
        assert np.all(lp <= 0.0) and np.all(tl <= 0.0) and np.all(en >= 0.0)
        assert k == 0 or np.array_equal(top[:, 0], hot)
