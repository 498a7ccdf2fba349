"""RoPE with the append of new rows to a paged cache, and eviction by weight,
against float64 / exact copies from their definitions."""
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


def rotate(x, pos, turns, rot, inter, mscale):
    """x [rows][heads][hd] rotated by pos [rows]; also what its error scales with."""
    half = rot // 2
    ang = pos.astype(np.float64)[:, None] * turns[None, :half]
    ang = 2 * np.pi * (ang - np.rint(ang))
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y, size = x.copy(), np.abs(x)
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :half], x[..., half:rot])
    ra, rb = (a * c - b * s) * mscale, (a * s + b * c) * mscale
    z = (np.abs(a) + np.abs(b)) * abs(mscale)
    if inter:
        y[..., 0:rot:2], y[..., 1:rot:2] = ra, rb
        size[..., 0:rot:2], size[..., 1:rot:2] = z, z
    else:
        y[..., :half], y[..., half:rot] = ra, rb
        size[..., :half], size[..., half:rot] = z, z
    return y, size


def norm(x, w, eps):
    return x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * w


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("nq,nkv,hd,page,rot,inter,in_t,normed,scaling", [
    (4, 2, 64, 16, 64, 0, R.F32, True, 0), (4, 4, 128, 32, 128, 0, None, False, 1), (10, 2, 128, 16, 64, 1, R.F32, False, 3),
    (8, 1, 256, 64, 256, 1, None, True, 2), (6, 3, 256, 16, 70, 0, None, False, 0), (5, 1, 64, 32, 6, 1, R.F32, True, 3),
    (32, 8, 128, 16, 100, 0, R.F32, True, 2), (0, 2, 64, 16, 64, 0, None, True, 0), (3, 1, 128, 1024, 2, 0, R.BF16, True, 1)])
def test_rope_append(eng, hip, nq, nkv, hd, page, rot, inter, in_t, normed, scaling, t):
    in_t = t if in_t is None else in_t
    rng = np.random.default_rng(nq * 100 + hd + rot + t)
    rows, ctx = [1, 3, 0, 20, 4], [1, 40, 7, 33, 3]
    cache = R.Cache(hip, rng, t, rows, ctx, nkv, hd, page, slots_first=bool(nq & 1), bad=[(1, 37 // page)])
    n, extra = cache.n_rows, 2
    pos = rng.integers(0, 2 ** 20, n + extra).astype(np.int32)
    pos[0], pos[5] = 0, 2 ** 31 - 1
    # q, k and v as a fused projection leaves them, with gaps between and behind
    width = (nq + 2 * nkv) * hd + 24
    qkv = R.to_type(rng.standard_normal((n + extra, width)) * 2, in_t)
    spec = abi.DpufAmdRopeSpec(rot_dim=rot, theta=1e6, scaling=scaling, factor=4.0 if scaling else 1.0, low_freq=1.0,
                               high_freq=4.0, beta_fast=32.0, beta_slow=1.0, orig_max_pos=4096)
    turns, m = np.zeros(rot // 2), C.c_float(0)
    assert eng.dpuf_amd_rope_turns(C.byref(spec), turns.ctypes.data_as(C.c_void_p), C.byref(m)) == 0
    dt, dpos, dqkv = hip.put(turns), hip.put(pos), hip.put(qkv)
    qn, kn = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    dqn, dkn = hip.put(qn), hip.put(kn)
    fill = R.to_type(np.full((n + extra, max(nq, 1), hd), 7.5, np.float32), t)
    dq = hip.put(fill)
    rope = abi.DpufAmdRope(turns=dt.p, rot_dim=rot, interleaved=inter, scale=m.value)
    es = 4 if in_t == R.F32 else 2
    at = [dqkv.p, dqkv.p + nq * hd * es, dqkv.p + ((nq + nkv) * hd + 8) * es]
    say(f"rope: {nq}/{nkv} heads of {hd}, pages of {page}, {rot} columns, interleaved {inter}, in {in_t}, out {t}")
    b, p = cache.batch(n_rows=n + extra), cache.pages()
    rc = eng.dpuf_amd_rope_append(C.byref(b), C.byref(p), C.byref(rope), dpos.p, in_t, nq, at[0] if nq else None, at[1],
                                  at[2], width, width, width, dqn.p if normed else None, dkn.p if normed else None,
                                  1e-6, dq.p if nq else None, None)
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    x = R.from_type(qkv, in_t)[:n]
    q, k = x[:, :nq * hd].reshape(n, nq, hd), x[:, nq * hd:(nq + nkv) * hd].reshape(n, nkv, hd)
    v0 = (nq + nkv) * hd + 8
    v = qkv[:n, v0:v0 + nkv * hd].reshape(n, nkv, hd)
    if normed:
        q, k = norm(q, qn, 1e-6), norm(k, kn, 1e-6)
    q, qs = rotate(q, pos[:n], turns, rot, inter, m.value)
    k, ks = rotate(k, pos[:n], turns, rot, inter, m.value)
    # fp32: the norm's sum over the head, sine and cosine to 2^-21, three products and a sum
    slack = ((hd + 16) * 2.0 ** -24 if normed else 0.0) + 2.0 ** -20
    got = dq.get()
    if nq:
        g = R.from_type(got, t)
        assert np.all(np.abs(g[:n] - q) <= R.HALF_STEP[t] * np.abs(q) * 1.01 + slack * qs + 2.0 ** -24)
    assert np.array_equal(got[n:], fill[n:])
    gk, gv, gw = cache.dk.get(), cache.dv.get(), cache.dw.get()
    old = (cache.k.copy(), cache.v.copy(), cache.w.copy())
    for s, (r, c) in enumerate(zip(rows, ctx)):
        for i in range(r):
            slot, row = c - r + i, cache.starts[s] + i
            if slot < 0 or not cache.ok(s, slot):
                continue
            pg, at_ = cache.table[s, slot // page], slot % page
            gr = R.from_type(cache.row(gk, pg, at_), t)
            assert np.all(np.abs(gr - k[row]) <= R.HALF_STEP[t] * np.abs(k[row]) * 1.01 + slack * ks[row] + 2.0 ** -24), \
                (s, i)
            want = v[row] if in_t == t else R.to_type(R.from_type(v[row], in_t).astype(np.float32), t)
            assert np.array_equal(cache.row(gv, pg, at_), want), (s, i)
            assert np.all(gw[pg, :, at_] == 0.0)
            for pool, was in ((gk, old[0]), (gv, old[1])):
                cache.row(pool, pg, at_)[...] = cache.row(was, pg, at_)
            gw[pg, :, at_] = old[2][pg, :, at_]
    # nothing else moved (bit patterns: unused rows are NaN)
    for a, b_ in ((gk, old[0]), (gv, old[1]), (gw.view(np.uint32), old[2].view(np.uint32))):
        assert np.array_equal(a, b_)


def test_rope_in_place_and_without_weights(eng, hip):
    """d_q_out = d_q, pages without w, the append of a row at a time."""
    rng = np.random.default_rng(3)
    cache = R.Cache(hip, rng, R.BF16, [2, 1], [18, 5], 2, 128, 16)
    q = R.to_type(rng.standard_normal((3, 6, 128)), R.BF16)
    kv = hip.put(R.to_type(rng.standard_normal((3, 512)), R.BF16))
    turns = np.array([1e6 ** (-2 * j / 128) / (2 * np.pi) for j in range(64)])
    rope = abi.DpufAmdRope(turns=hip.put(turns).p, rot_dim=128, interleaved=0, scale=1.0)
    pos = hip.put(np.array([16, 17, 4], np.int32))
    outs = []
    say("rope in place")
    for in_place in (0, 1):
        dq = hip.put(q)
        do = dq if in_place else hip.put(np.zeros_like(q))
        b, p = cache.batch(), cache.pages(w=False)
        assert eng.dpuf_amd_rope_append(C.byref(b), C.byref(p), C.byref(rope), pos.p, R.BF16, 6, dq.p, kv.p,
                                        kv.p + 512, 768, 512, 512, None, None, 0.0, do.p, None) == 0
        outs.append(do.get())
    assert np.array_equal(outs[0], outs[1])
    assert np.array_equal(cache.dw.get().view(np.uint32), cache.w.view(np.uint32))


def keep_of(w, there, keep, sink, recent):
    """Kept rows of one (sequence, kv head), from the definition."""
    c = len(w)
    if c <= keep:
        return np.arange(c)
    mid = np.arange(sink, c - recent)
    key = np.where(there & ~np.isnan(w), w, -np.inf).astype(np.float64)
    lowest = ~there | np.isnan(w)
    order = sorted(mid, key=lambda i: (lowest[i], -key[i], i))[:keep - sink - recent]
    return np.sort(np.concatenate([np.arange(sink), order, np.arange(c - recent, c)]).astype(int))


def evict(eng, hip, cache, keep, sink, recent, dst_page, dst_first, bad_dst=()):
    rng = np.random.default_rng(99)
    n = [min(c, keep) for c in cache.ctx]
    dst = R.Cache(hip, rng, cache.t, [0] * len(n), n, cache.nkv, cache.hd, dst_page, slots_first=dst_first, bad=bad_dst,
                  table_extra=-(-keep // dst_page))
    kept = hip.put(np.full((len(n), cache.nkv, keep), -7, np.int32))
    new_len = hip.put(np.full(len(n), -7, np.int32))
    b, p, dp = cache.batch(n_rows=0), cache.pages(), dst.pages()
    rc = eng.dpuf_amd_paged_evict(C.byref(b), C.byref(p), keep, sink, recent, C.byref(dp), dst.d_table.p,
                                  dst.table.shape[1], kept.p, new_len.p, None)
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    gk, gv, gw, gkept = dst.dk.get(), dst.dv.get(), dst.dw.get(), kept.get()
    assert np.array_equal(new_len.get(), n)
    wk, wv, ww = dst.k.copy(), dst.v.copy(), dst.w.copy()
    want = np.full_like(gkept, -7)
    for s, c in enumerate(cache.ctx):
        there = cache.present(s)
        for h in range(cache.nkv):
            w = np.array([cache.w[cache.table[s, i // cache.page], h, i % cache.page] if there[i] else 0.0
                          for i in range(c)])
            rows = keep_of(w, there, keep, sink, recent)
            want[s, h, :len(rows)] = rows
            for i, r in enumerate(rows):
                if not dst.ok(s, i):
                    continue
                pg, at = dst.table[s, i // dst_page], i % dst_page
                if there[r]:
                    spg, sat = cache.table[s, r // cache.page], r % cache.page
                    dst.row(wk, pg, at)[h] = cache.row(cache.k, spg, sat)[h]
                    dst.row(wv, pg, at)[h] = cache.row(cache.v, spg, sat)[h]
                    ww[pg, h, at] = cache.w[spg, h, sat]
                else:
                    dst.row(wk, pg, at)[h] = 0
                    dst.row(wv, pg, at)[h] = 0
                    ww[pg, h, at] = 0.0
    assert np.array_equal(gkept, want)
    assert np.array_equal(gk, wk) and np.array_equal(gv, wv)
    assert np.array_equal(gw.view(np.uint32), ww.view(np.uint32))


@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (1, 0, 1), (1, 1, 0), (33, 4, 8), (64, 0, 64), (64, 64, 0),
                                              (99, 1, 0), (130, 0, 0), (700, 4, 16), (2000, 0, 0)])
@pytest.mark.parametrize("nkv,hd,page,t", [(2, 64, 16, R.BF16), (1, 256, 64, R.F16), (3, 128, 32, R.BF16)])
def test_evict(eng, hip, keep, sink, recent, nkv, hd, page, t):
    rng = np.random.default_rng(keep + hd)
    cache = R.Cache(hip, rng, t, [0] * 6, [1, 0, 64, 65, 131, 1025], nkv, hd, page, slots_first=hd == 128)
    say(f"evict: keep {keep} sink {sink} recent {recent}, {nkv} heads of {hd}, pages of {page}")
    evict(eng, hip, cache, keep, sink, recent, 128 if page == 16 else 16, hd == 64)


def test_evict_ties_and_odd_weights(eng, hip):
    """Equal weights (the earliest stay), zeros of both signs, infinities, NaN,
    negative weights, absent source and destination pages."""
    rng = np.random.default_rng(1)
    cache = R.Cache(hip, rng, R.BF16, [0] * 4, [200, 200, 200, 90], 2, 64, 16, bad=[(2, 3), (2, 7), (3, 0)])
    vals = np.array([0.0, -0.0, 1.0, 1.0, 2.0, np.inf, -np.inf, np.nan, -3.0, 1e-40], np.float32)
    for s in range(4):
        for i in range(cache.ctx[s]):
            if cache.ok(s, i):
                pg, r = cache.table[s, i // 16], i % 16
                cache.w[pg, :, r] = 0.25 if s == 0 else rng.choice(vals, 2)
    cache.dw.set(cache.w)
    for keep, sink, recent in ((50, 3, 7), (190, 0, 1), (120, 0, 0)):
        say(f"evict ties: keep {keep}")
        evict(eng, hip, cache, keep, sink, recent, 16, False, bad_dst=[(1, 1)])


def test_evict_long_rows(eng, hip):
    """More cached rows than the selection holds in LDS."""
    rng = np.random.default_rng(2)
    cache = R.Cache(hip, rng, R.F16, [0], [40000], 1, 64, 1024)
    say("evict: 40 000 rows")
    evict(eng, hip, cache, 37000, 4, 100, 256, False)


@pytest.mark.parametrize("extra", [0, 100, 200, 400, 700])
@pytest.mark.parametrize("keep,sink,recent", [(50, 3, 9), (1500, 0, 0), (60, 30, 30)])
def test_evict_under_longer_tables(eng, hip, keep, sink, recent, extra):
    """Tables that allow for more rows than the sequences have: selection from
    registers, by every number of keys a thread, and from LDS."""
    rng = np.random.default_rng(keep + extra)
    cache = R.Cache(hip, rng, R.BF16, [0] * 5, [1600, 0, 59, 61, 1100], 2, 64, 16, table_extra=2 + extra,
                    bad=[(0, 7), (0, 99), (4, 0)])
    cache.w = np.where(rng.random(cache.w.shape) < 0.3, np.float32(0.25), cache.w)       # ties
    cache.w.flat[::97] = -np.inf
    cache.w.flat[::89] = np.inf
    cache.w.flat[::83] = np.nan
    cache.dw.set(cache.w)
    say(f"evict: keep {keep} sink {sink} recent {recent}, {extra} spare table entries")
    evict(eng, hip, cache, keep, sink, recent, 32, False)


@pytest.mark.parametrize("ctx,keep", [([2047], 1000), ([4080, 30], 2000), ([8176], 3001), ([8193], 3001)])
def test_evict_at_the_ends_of_the_ranges(eng, hip, ctx, keep):
    rng = np.random.default_rng(keep)
    cache = R.Cache(hip, rng, R.F16, [0] * len(ctx), ctx, 1, 64, 16, table_extra=0)
    say(f"evict: {ctx} rows to {keep}")
    evict(eng, hip, cache, keep, 4, 32, 64, False)


@pytest.mark.parametrize("extra", [600, 1200])
def test_evict_under_much_longer_tables(eng, hip, extra):
    rng = np.random.default_rng(extra)
    cache = R.Cache(hip, rng, R.F16, [0] * 3, [1600, 70, 1100], 2, 64, 16, table_extra=2 + extra, bad=[(0, 9)])
    cache.w = np.where(rng.random(cache.w.shape) < 0.3, np.float32(0.25), cache.w)
    cache.dw.set(cache.w)
    say(f"evict: {extra} spare table entries")
    evict(eng, hip, cache, 700, 4, 16, 32, True)


@pytest.mark.parametrize("ctx,keep", [([12288], 5000), ([16384], 4097), ([16385, 5], 4097)])
def test_evict_at_the_ends_of_the_longer_ranges(eng, hip, ctx, keep):
    rng = np.random.default_rng(keep)
    cache = R.Cache(hip, rng, R.BF16, [0] * len(ctx), ctx, 1, 64, 64, table_extra=0)
    say(f"evict: {ctx} rows to {keep}")
    evict(eng, hip, cache, keep, 0, 100, 64, False)
