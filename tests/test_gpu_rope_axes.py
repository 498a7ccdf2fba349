"""RoPE of several position axes with the append of new rows to a paged cache,
against float64 from the definition."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from dpuf_amd import abi
from test_gpu_paged_cache import norm

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip(eng):
    h = R.Hip()
    yield h
    h.free_all()


def say(*a):
    print(*a, flush=True)


def axis_of(pairs, sections, in_turn):
    """Axis of each pair."""
    n, out = len(sections), np.zeros(pairs, int)
    if in_turn:
        for a in range(1, n):
            out[a:n * sections[a]:n] = a
    else:
        out[:] = np.repeat(np.arange(n), sections)
    assert np.array_equal(np.bincount(out, minlength=n), sections)
    return out


def rotate(x, pos, turns, rot, inter, mscale):
    """x [rows][heads][hd] rotated, pos [rows][pairs]; also what its error scales with."""
    half = rot // 2
    ang = pos.astype(np.float64) * turns[None, :half]
    ang = 2 * np.pi * (ang - np.rint(ang))
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y, size = x.copy(), np.abs(x)
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :half], x[..., half:rot])
    z = (np.abs(a) + np.abs(b)) * abs(mscale)
    at = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, half), slice(half, rot))
    y[..., at[0]], y[..., at[1]] = (a * c - b * s) * mscale, (a * s + b * c) * mscale
    size[..., at[0]], size[..., at[1]] = z, z
    return y, size


def axes_of(sections, in_turn):
    return abi.DpufAmdRopeAxes(n_axes=len(sections), sections=(C.c_int32 * 4)(*sections, *[-7] * (4 - len(sections))),
                               in_turn=in_turn)


# heads, page, rotated columns, pairs' layout, input type (None: the pages'), norms, sections, in turn
CASES = [(4, 2, 64, 16, 64, 0, R.F32, True, [12, 10, 10], 1), (32, 8, 128, 64, 128, 0, None, True, [24, 20, 20], 1),
         (32, 8, 128, 16, 128, 0, R.F32, False, [16, 24, 24], 0), (10, 2, 128, 16, 64, 1, R.F32, False, [0, 32], 0),
         (8, 1, 256, 64, 256, 1, None, True, [32, 32, 32, 32], 1), (6, 3, 256, 16, 70, 0, None, False, [35, 0, 0], 1),
         (5, 1, 64, 32, 6, 1, R.F32, True, [1, 1, 1], 1), (0, 2, 64, 16, 64, 0, None, True, [10, 0, 22], 0),
         (3, 1, 128, 1024, 2, 0, R.BF16, True, [0, 0, 0, 1], 0), (4, 4, 64, 16, 64, 0, None, False, [32], 0),
         (4, 4, 64, 16, 64, 0, None, False, [32], 1), (3, 1, 128, 32, 100, 1, R.F32, True, [26, 24], 1),
         (12, 4, 128, 16, 128, 0, None, False, [40, 3, 21], 1)]


@pytest.mark.parametrize("t", [R.BF16, R.F16])
@pytest.mark.parametrize("nq,nkv,hd,page,rot,inter,in_t,normed,sections,in_turn", CASES)
def test_rope_append_axes(eng, hip, nq, nkv, hd, page, rot, inter, in_t, normed, sections, in_turn, t):
    in_t = t if in_t is None else in_t
    rng = np.random.default_rng(nq * 100 + hd + rot + t)
    rows, ctx = [1, 3, 0, 20, 4], [1, 40, 7, 33, 3]
    cache = R.Cache(hip, rng, t, rows, ctx, nkv, hd, page, slots_first=bool(nq & 1), bad=[(1, 37 // page)])
    n, extra = cache.n_rows, 2
    # positions of an axis `gap` entries further than its rows; nothing between may count
    gap = 3
    pos = rng.integers(0, 2 ** 20, (len(sections), n + extra + gap)).astype(np.int32)
    pos[0, 0], pos[-1, 5], pos[:, n + extra:] = 0, 2 ** 31 - 1, -2 ** 31
    width = (nq + 2 * nkv) * hd + 24
    qkv = R.to_type(rng.standard_normal((n + extra, width)) * 2, in_t)
    spec = abi.DpufAmdRopeSpec(rot_dim=rot, theta=1e6, scaling=3, factor=4.0, beta_fast=32.0, beta_slow=1.0,
                               orig_max_pos=4096)
    turns, m = np.zeros(rot // 2), C.c_float(0)
    assert eng.dpuf_amd_rope_turns(C.byref(spec), turns.ctypes.data_as(C.c_void_p), C.byref(m)) == 0
    dt, dpos, dqkv = hip.put(turns), hip.put(pos), hip.put(qkv)
    qn, kn = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    dqn, dkn = hip.put(qn), hip.put(kn)
    fill = R.to_type(np.full((n + extra, max(nq, 1), hd), 7.5, np.float32), t)
    dq = hip.put(fill)
    rope = abi.DpufAmdRope(turns=dt.p, rot_dim=rot, interleaved=inter, scale=m.value)
    ax = axes_of(sections, in_turn)
    es = 4 if in_t == R.F32 else 2
    at = [dqkv.p, dqkv.p + nq * hd * es, dqkv.p + ((nq + nkv) * hd + 8) * es]
    say(f"axes: {nq}/{nkv} heads of {hd}, pages of {page}, {rot} columns, interleaved {inter}, in {in_t}, out {t}, "
        f"sections {sections}, in turn {in_turn}")
    b, p = cache.batch(n_rows=n + extra), cache.pages()
    rc = eng.dpuf_amd_rope_append_axes(C.byref(b), C.byref(p), C.byref(rope), C.byref(ax), dpos.p, pos.shape[1], in_t,
                                       nq, at[0] if nq else None, at[1], at[2], width, width, width,
                                       dqn.p if normed else None, dkn.p if normed else None, 1e-6,
                                       dq.p if nq else None, None)
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    x = R.from_type(qkv, in_t)[:n]
    q, k = x[:, :nq * hd].reshape(n, nq, hd), x[:, nq * hd:(nq + nkv) * hd].reshape(n, nkv, hd)
    v0 = (nq + nkv) * hd + 8
    v = qkv[:n, v0:v0 + nkv * hd].reshape(n, nkv, hd)
    if normed:
        q, k = norm(q, qn, 1e-6), norm(k, kn, 1e-6)
    by_pair = pos[axis_of(rot // 2, sections, in_turn)][:, :n].T
    q, qs = rotate(q, by_pair, turns, rot, inter, m.value)
    k, ks = rotate(k, by_pair, turns, rot, inter, m.value)
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


@pytest.mark.parametrize("rows,sections,in_turn", [(1, [24, 20, 20], 1), (9, [16, 24, 24], 0), (300, [64], 0),
                                                   (300, [22, 21, 21], 1)])
def test_equal_positions_are_one_axis(eng, hip, rows, sections, in_turn):
    """Text, whose positions agree on all axes: the bits of dpuf_amd_rope_append;
    in place too, and captured into a graph that is replayed over new positions."""
    rng = np.random.default_rng(rows)
    nq, nkv, hd = 16, 8, 128
    cache = R.Cache(hip, rng, R.BF16, [rows], [rows + 5], nkv, hd, 16)
    qkv = R.to_type(rng.standard_normal((rows, (nq + 2 * nkv) * hd)), R.BF16)
    turns = np.array([1e6 ** (-2 * j / hd) / (2 * np.pi) for j in range(hd // 2)])
    rope = abi.DpufAmdRope(turns=hip.put(turns).p, rot_dim=hd, interleaved=0, scale=1.0)
    ax, b, p = axes_of(sections, in_turn), cache.batch(), cache.pages()
    qn = hip.put((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32))
    d = hip.put(qkv)
    q = hip.put(np.ascontiguousarray(qkv[:, :nq * hd]))
    out = hip.put(np.zeros((rows, nq, hd), np.uint16))
    dpos = hip.put(np.zeros((len(sections), rows), np.int32))
    k, v, w = d.p + nq * hd * 2, d.p + (nq + nkv) * hd * 2, (nq + 2 * nkv) * hd

    def both(pos, run):
        """One axis, then several: outputs and pools."""
        got = []
        for many in (0, 1):
            cache.upload_into()
            out.set(np.zeros((rows, nq, hd), np.uint16))
            dpos.set(np.repeat(pos[None], len(sections), 0))
            if many:
                run()
            else:
                assert eng.dpuf_amd_rope_append(C.byref(b), C.byref(p), C.byref(rope), dpos.p, R.BF16, nq, q.p, k, v,
                                                nq * hd, w, w, qn.p, qn.p, 1e-6, out.p, None) == 0
            got.append((out.get(), cache.dk.get(), cache.dv.get()))
        for x, y in zip(*got):
            assert np.array_equal(x, y)
        return got[1][0]

    def axes(o, s=None):
        rc = eng.dpuf_amd_rope_append_axes(C.byref(b), C.byref(p), C.byref(rope), C.byref(ax), dpos.p, rows, R.BF16, nq,
                                           q.p, k, v, nq * hd, w, w, qn.p, qn.p, 1e-6, o, s)
        assert rc == 0, (rc, eng.dpuf_amd_last_error())

    say(f"equal positions: {rows} rows, sections {sections}")
    pos = rng.integers(0, 10 ** 6, rows).astype(np.int32)
    want = both(pos, lambda: axes(out.p))
    s = hip.stream()
    graph, ge = C.c_void_p(), C.c_void_p()
    assert hip.lib.hipStreamBeginCapture(s, 1) == 0
    axes(out.p, s)
    assert hip.lib.hipStreamEndCapture(s, C.byref(graph)) == 0
    assert hip.lib.hipGraphInstantiate(C.byref(ge), graph, None, None, 0) == 0

    def replay():
        assert hip.lib.hipGraphLaunch(ge, s) == 0 and hip.lib.hipStreamSynchronize(s) == 0

    for _ in range(3):
        both(rng.integers(0, 10 ** 6, rows).astype(np.int32), replay)
    hip.lib.hipGraphExecDestroy(ge)
    hip.lib.hipGraphDestroy(graph)
    hip.lib.hipStreamDestroy(s)
    dpos.set(np.repeat(pos[None], len(sections), 0))
    axes(q.p)
    assert np.array_equal(q.get().reshape(rows, nq, hd), want)
