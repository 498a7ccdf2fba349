"""Sampling from given random numbers against float64 from the definition."""
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


def one(x, t, k, p, mp, u):
    """(token, log probability) of one row of float64 logits."""
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return -1, -np.inf
    if not t > 0:
        return int(np.argmax(x)), 0.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp(np.where(x == -np.inf, -np.inf, (x - x.max()) / t)))
        w = np.where(np.isnan(w), 0.0, w)
    if np.isinf(t):
        w = np.where(x == -np.inf, 0.0, 1.0)
    if x.max() == np.inf:       # an infinite logit leaves only its like
        w = np.where(x == np.inf, 1.0, 0.0)
    order = np.argsort(-x, kind="stable")
    n = k if 0 < k < len(x) else len(x)
    order = order[:n]
    if p < 1:
        run = np.cumsum(w[order])
        order = order[:max(1, int(np.searchsorted(run, p * run[-1])) + 1)]
    order = order[:max(1, int((w[order] >= min(1.0, mp)).sum()))] if mp > 0 else order
    ids = np.sort(order)
    run = np.cumsum(w[ids])
    u = min(max(u if u == u else 0.0, 0.0), 1.0)
    at = int(np.searchsorted(run, u * run[-1], side="right"))
    if at >= len(ids):
        at = int(np.nonzero(w[ids])[0][-1])
    return int(ids[at]), float(np.log(w[ids[at]] / run[-1]))


def arr(hip, v, t):
    return None if v is None else hip.put(np.asarray(v, t))


def sample(eng, hip, x, t, temp=None, top_k=None, top_p=None, min_p=None, u=None, stride=None, offset=0, logp=True):
    n, V = x.shape
    store = R.to_type(x, t)
    stride = V if stride is None else stride
    full = R.to_type(np.full((n, stride), 30.0, np.float32), t)     # what lies between rows would win
    full[:, :V] = store
    d = hip.put(full, offset)
    dt, dk, dp, dm, du = (arr(hip, v, np.int32 if v is top_k and v is not None else np.float32)
                          for v in (temp, top_k, top_p, min_p, u))
    tok, lp = hip.put(np.full(n, -9, np.int32)), hip.put(np.full(n, 9.0, np.float32))
    ws = int(eng.dpuf_amd_sample_workspace(n, V))
    dws = hip.put(np.full(max(ws, 16), 0xFF, np.uint8))
    at = lambda v: v.p if v is not None else None
    rc = eng.dpuf_amd_sample(t, n, V, stride, d.p, at(dt), at(dk), at(dp), at(dm), du.p, tok.p,
                             lp.p if logp else None, dws.p if ws else None, ws, None)
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    got, glp = tok.get(), lp.get()
    x64 = R.from_type(store, t).reshape(n, V)
    pick = lambda v, i, off: float(np.float32(v[i])) if v is not None else off
    for i in range(n):
        want, wl = one(x64[i], pick(temp, i, 1.0), int(pick(top_k, i, 0)), pick(top_p, i, 1.0), pick(min_p, i, 0.0),
                       float(np.float32(u[i])))
        assert got[i] == want, (i, int(got[i]), want)
        if logp:
            # weights are integers of 2^-38 of the largest or finer, V of them; one fp32 rounding
            assert glp[i] == wl or abs(glp[i] - wl) <= abs(wl) * 2.0 ** -23 + V * 2.0 ** -38 + 2.0 ** -30, \
                (i, float(glp[i]), wl)
    return got


def logits(rng, n, V, spread=2.5):
    x = rng.standard_normal((n, V)).astype(np.float32) * spread
    for i in range(n):
        hot = rng.integers(0, V, max(1, V // 50))[:20]
        x[i, hot] += rng.random(len(hot)).astype(np.float32) * 9
    return x


KINDS = [dict(), dict(k=1), dict(k=7), dict(p=0.9), dict(p=0.0), dict(p=0.3), dict(mp=0.05), dict(mp=1.0),
         dict(k=50, p=0.95), dict(k=1000, p=0.5, mp=0.01), dict(k=10 ** 9, p=1.5, mp=-1.0), dict(t=0.0), dict(t=0.05),
         dict(t=20.0), dict(t=20.0, p=0.999), dict(t=20.0, k=3000, p=0.9999), dict(t=-1.0), dict(p=1e-6, t=5.0),
         dict(k=4097, t=20.0), dict(mp=2.0, t=3.0)]


@pytest.mark.parametrize("t", [R.F32, R.BF16, R.F16])
@pytest.mark.parametrize("V", [1, 2, 63, 1000, 4099, 32000, 151936])
def test_settings(eng, hip, V, t):
    rng = np.random.default_rng(V + t)
    n = len(KINDS) * 2
    x = logits(rng, n, V)
    col = lambda f, off: [k.get(f, off) for k in KINDS] * 2
    say(f"sample: V {V}, type {t}")
    sample(eng, hip, x, t, temp=col("t", 0.8), top_k=np.array(np.minimum(col("k", 0), 2 ** 31 - 1), np.int32),
           top_p=col("p", 1.0), min_p=col("mp", 0.0), u=rng.random(n).astype(np.float32))


def test_everything_off(eng, hip):
    rng = np.random.default_rng(4)
    for V, t in ((77, R.F32), (5000, R.BF16)):
        sample(eng, hip, logits(rng, 3, V), t, u=rng.random(3), logp=V == 77)


@pytest.mark.parametrize("t", [R.F32, R.BF16])
def test_strides_and_alignment(eng, hip, t):
    rng = np.random.default_rng(5)
    for stride, offset in ((1001, 0), (1003, 4), (1024, 8), (1024, 0), (1016, 2 if t == R.BF16 else 4)):
        say(f"sample: rows {stride} apart, {offset} bytes in, type {t}")
        sample(eng, hip, logits(rng, 5, 1000), t, temp=[1.0] * 5, top_k=np.array([0, 9, 0, 40, 0], np.int32),
               top_p=[1, 1, .8, .8, 1], u=rng.random(5), stride=stride, offset=offset)


@pytest.mark.parametrize("V", [50, 20000])
def test_ties(eng, hip, V):
    """Few distinct values (top-k and top-p cut through runs of equal logits:
    the lowest indices stay), all logits equal, both zeros."""
    rng = np.random.default_rng(6)
    x = rng.integers(-2, 3, (8, V)).astype(np.float32)
    x[3:6] = 1.25
    x[6] = np.where(np.arange(V) % 2, 0.0, -0.0)
    say(f"ties: V {V}")
    for k, p in ((V // 3, 1.0), (0, 0.37), (V // 2, 0.5), (V - 1, 0.999)):
        sample(eng, hip, x, R.F32, temp=[1.0] * 8, top_k=np.full(8, k, np.int32), top_p=[p] * 8,
               u=(np.arange(8) + rng.random(8)) / 8)


def test_masked_and_odd_logits(eng, hip):
    """-infinity (a grammar's mask), NaN, +infinity, rows that leave nothing,
    the lowest finite value as a mask, draws at and outside [0, 1)."""
    rng = np.random.default_rng(7)
    V = 6000
    x = logits(rng, 12, V)
    x[0, :] = -np.inf
    x[1, :] = np.nan
    x[2, rng.permutation(V)[:V - 5]] = -np.inf
    x[3, ::2] = np.nan
    x[4, [7, 90]] = np.inf
    x[5, rng.permutation(V)[:V - 3]] = np.finfo(np.float32).min
    x[6, :] = np.finfo(np.float32).min
    x[7, 1:] = -np.inf
    x[8] *= 1e30
    u = np.array([.5, .5, .6, .4, .7, .3, .999, 0, 0.5, -1.0, 1.0, np.nan], np.float32)
    say("odd logits")
    for top_k, top_p in ((0, 1.0), (3, 1.0), (0, .9), (5000, .99)):
        sample(eng, hip, x, R.F32, temp=[1.0] * 12, top_k=np.full(12, top_k, np.int32), top_p=[top_p] * 12, u=u)
    sample(eng, hip, x, R.F32, temp=[np.inf, np.inf, np.inf, np.nan] * 3, u=u)


def test_draw_walks_the_distribution(eng, hip):
    """Draws spread over [0, 1) hit every kept token in index order, as often
    as its share: the running sums are those of the definition."""
    V, n = 40, 1000
    rng = np.random.default_rng(8)
    x = np.repeat(rng.standard_normal((1, V)).astype(np.float32), n, 0)
    u = (np.arange(n) + 0.5) / n
    got = sample(eng, hip, x, R.F32, temp=[0.7] * n, top_k=np.full(n, 20, np.int32), u=u)
    assert np.all(np.diff(got) >= 0) and len(set(got.tolist())) > 10


def test_large_vocabulary_and_many_rows(eng, hip):
    rng = np.random.default_rng(9)
    say("sample: V 2^20 + 3")
    sample(eng, hip, rng.standard_normal((2, (1 << 20) + 3)).astype(np.float32), R.F32, temp=[1.0, 1.0],
           top_k=np.array([0, 70000], np.int32), top_p=[0.5, 0.9], u=[0.3, 0.8])
    say("sample: 700 rows")
    sample(eng, hip, logits(rng, 700, 300), R.F16, temp=[0.9] * 700, top_p=[0.9] * 700, u=rng.random(700))


@pytest.mark.parametrize("spread", [0.3, 2.5])
def test_prefixes_around_the_list_lengths(eng, hip, spread):
    """Top-k around 64, 128 and 256 tokens, alone and with top-p and min-p, and
    top-p that keeps such numbers: what is ranked as it is, what is selected."""
    rng = np.random.default_rng(int(10 * spread))
    ks = [1, 2, 63, 64, 65, 100, 127, 128, 129, 150, 191, 192, 193, 200, 254, 255, 256, 257, 258, 300, 400]
    V = 20000
    x = logits(rng, 3 * len(ks), V, spread)
    top_k = np.array(ks * 3)
    top_p = np.repeat([1.0, 0.9, 0.97], len(ks))
    min_p = np.repeat([0.0, 0.0, 0.01], len(ks))
    u = rng.random(len(x))
    say(f"list lengths, spread {spread}: top-k")
    sample(eng, hip, x, R.F32, None, top_k, top_p, min_p, u)
    # top-p of the weight of the k largest, so that about k stay
    w = -np.sort(-np.exp((x[:len(ks)] - x[:len(ks)].max(1, keepdims=True)).astype(np.float64)), 1)
    p = np.array([w[i, :k].sum() / w[i].sum() for i, k in enumerate(ks)]) * (1 - 1e-5)
    say(f"list lengths, spread {spread}: top-p")
    sample(eng, hip, x[:len(ks)], R.F32, None, None, p, None, u[:len(ks)])


def both_calls(eng, hip, x, t, **kw):
    """The same call twice: the same tokens (each checked against float64)."""
    a, b = (sample(eng, hip, x, t, **kw) for _ in range(2))
    assert np.array_equal(a, b)


def settled(n, temp, k, p, mp):
    return dict(temp=[temp] * n, top_k=np.full(n, k, np.int32), top_p=[p] * n, min_p=[mp] * n)


@pytest.mark.parametrize("k,about", [(1000, 0), (0, 300), (0, 1000), (0, 2000), (1500, 1000)])
def test_min_p_border_in_a_crowd_behind_the_prefix(eng, hip, k, about):
    """One likely token over a narrow bell: min-p's border lies in the bell,
    among more tokens than a list holds, behind the last token that top-k, or
    top-p (about so many tokens), leaves."""
    rng = np.random.default_rng(k + about)
    n = 6
    row = (rng.standard_normal(151936) * 0.1).astype(np.float32)
    row[777] = 8.0
    w = np.exp(np.sort(row.astype(np.float64))[::-1] - 8.0)
    p = float(w[:about].sum() / (w[:k].sum() if k else w.sum())) if about else 1.0
    say(f"crowd behind the prefix: top-k {k}, top-p {p:.4f}")
    both_calls(eng, hip, np.repeat(row[None], n, 0), R.F32, u=(np.arange(n) + rng.random(n)) / n,
               **settled(n, 1.0, k, p, np.exp(-8.0)))


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("k", [257, 300, 500, 2000])
def test_min_p_border_among_coarse_values(eng, hip, k, t):
    """16-bit logits of such size that thousands of tokens share a value."""
    rng = np.random.default_rng(k)
    n = 4
    row = (rng.standard_normal(151936) * 2.2 + 20).astype(np.float32)
    say(f"coarse values: top-k {k}, type {t}")
    both_calls(eng, hip, np.repeat(row[None], n, 0), t, u=(np.arange(n) + rng.random(n)) / n,
               **settled(n, 1.5, k, 1.0, 0.0015))


@pytest.mark.parametrize("side", [-1, 0, 1])
@pytest.mark.parametrize("V,loose,k,p", [(4000, 700, 300, 1.0), (4000, 700, 0, 0.9), (4000, 700, 650, 0.99),
                                         (8000, 1000, 500, 1.0), (8000, 1000, 2000, 1.0), (60000, 2100, 2000, 1.0)])
def test_min_p_border_on_a_run_of_equal_logits(eng, hip, V, loose, k, p, side):
    """`loose` tokens between 5 and 10, the others all 0, and min-p a little
    below, about and above e^-10: one chunk and many, the run behind the prefix
    and (top-k 2 000 of 1 000 loose ones) within it."""
    rng = np.random.default_rng(V + k)
    n = 5
    row = np.zeros(V, np.float32)
    at = rng.permutation(V)[:loose]
    row[at] = 5 + 5 * rng.random(loose)
    row[at[0]] = 10.0
    say(f"run at min-p's border: V {V}, top-k {k}, top-p {p}, side {side}")
    both_calls(eng, hip, np.repeat(row[None], n, 0), R.F32, u=(np.arange(n) + rng.random(n)) / n,
               **settled(n, 1.0, k, p, np.exp(-10.0) * (1 + 1e-3 * side) + (0 if side else 1e-12)))


@pytest.mark.parametrize("temp", [1e22, 3e38, np.inf])
def test_min_p_at_temperatures_that_make_all_weights_equal(eng, hip, temp):
    """d / temperature below 2^-60: every weight is 1 in 64 bits, and min-p of
    1 keeps them all, whatever bin they lie in."""
    rng = np.random.default_rng(3)
    n = 6
    x = logits(rng, n, 20000)
    for k, p, mp in ((1000, 1.0, 1.0), (0, 0.05, 1.0), (3000, 0.9, 0.999), (0, 1.0, 1.0), (100, 1.0, 1.0)):
        say(f"temperature {temp}: top-k {k}, top-p {p}, min-p {mp}")
        both_calls(eng, hip, x, R.F32, u=(np.arange(n) + rng.random(n)) / n, **settled(n, temp, k, p, mp))
