"""The paged-serving operators one after the other, as a serving loop runs
them: a step captured into a graph, steps on two streams at once, and the
arguments that may not share memory."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from dpuf_amd import abi

pytestmark = pytest.mark.gpu

NQ, NKV, HD, V, KEEP = 8, 2, 128, 5000, 40


@pytest.fixture()
def hip(eng):
    h = R.Hip()
    yield h
    h.free_all()


class Step:
    """One decode step of a batch, everything on the device: append, attention,
    weights, eviction into pages of another pool, sampling."""

    def __init__(self, eng, hip, seed, rows, ctx):
        rng = np.random.default_rng(seed)
        self.eng, self.hip, self.rng = eng, hip, rng
        n = len(ctx)
        self.cache = c = R.Cache(hip, rng, R.BF16, rows, ctx, NKV, HD, 32)
        self.dst = R.Cache(hip, rng, R.BF16, [0] * n, [KEEP] * n, NKV, HD, 16)
        self.stream = hip.stream()
        width = (NQ + 2 * NKV) * HD
        self.qkv = hip.put(np.zeros((c.n_rows, width), np.float32))
        self.pos = hip.put(np.zeros(c.n_rows, np.int32))
        self.q = hip.put(np.zeros((c.n_rows, NQ, HD), np.uint16))
        self.out = hip.put(np.zeros((c.n_rows, NQ, HD), np.float32))
        self.lse = hip.put(np.zeros((c.n_rows, NQ), np.float32))
        self.kept = hip.put(np.zeros((n, NKV, KEEP), np.int32))
        self.new_len = hip.put(np.zeros(n, np.int32))
        self.x = hip.put(np.zeros((n, V), np.float32))
        self.settings = [hip.put(np.zeros(n, t)) for t in (np.float32, np.int32, np.float32, np.float32, np.float32)]
        self.tok, self.lp = hip.put(np.zeros(n, np.int32)), hip.put(np.zeros(n, np.float32))
        self.rope = abi.DpufAmdRope(turns=hip.put(1e4 ** (-np.arange(64) / 64) / 6.283185307179586).p, rot_dim=HD,
                                    interleaved=0, scale=1.0)
        self.b, self.p, self.dp = c.batch(), c.pages(), self.dst.pages()
        self.ws_n = int(eng.dpuf_amd_paged_attn_workspace(C.byref(self.b), C.byref(self.p), NQ))
        self.ws = hip.put(np.full(max(16, self.ws_n), 0xFF, np.uint8))
        self.sws_n = int(eng.dpuf_amd_sample_workspace(n, V))
        self.sws = hip.put(np.full(self.sws_n, 0xFF, np.uint8))

    def enter(self, seed):
        """Inputs of one step: new activations, lengths and settings, the
        caches as they were."""
        rng, c, n = np.random.default_rng(seed), self.cache, len(self.cache.ctx)
        c.upload_into()
        self.qkv.set(rng.standard_normal(self.qkv.like.shape).astype(np.float32))
        self.pos.set(rng.integers(0, 1 << 20, c.n_rows).astype(np.int32))
        c.d_ctx.set(np.array([rng.integers(0, m + 1) for m in c.ctx], np.int32))
        self.x.set((rng.standard_normal((n, V)) * 3).astype(np.float32))
        for d, v in zip(self.settings, (rng.random(n) + 0.3, rng.integers(0, 60, n), rng.random(n) + 0.3,
                                        rng.random(n) * 0.1, rng.random(n))):
            d.set(v.astype(d.like.dtype))

    def run(self, stream):
        e, r, b, p, es = self.eng, C.byref, self.b, self.p, 4
        at = self.qkv.p
        w = self.qkv.like.shape[1]
        assert e.dpuf_amd_rope_append(r(b), r(p), r(self.rope), self.pos.p, R.F32, NQ, at, at + NQ * HD * es,
                                      at + (NQ + NKV) * HD * es, w, w, w, None, None, 0.0, self.q.p, stream) == 0
        assert e.dpuf_amd_paged_attn(r(b), r(p), NQ, self.q.p, 0.09, R.F32, self.out.p, self.lse.p, self.ws.p,
                                     self.ws_n, stream) == 0
        assert e.dpuf_amd_paged_attn_weights(r(b), r(p), NQ, self.q.p, 0.09, self.lse.p, 0.9, self.cache.dw.p,
                                             stream) == 0
        assert e.dpuf_amd_paged_evict(r(b), r(p), KEEP, 2, 8, r(self.dp), self.dst.d_table.p, self.dst.table.shape[1],
                                      self.kept.p, self.new_len.p, stream) == 0
        s = self.settings
        assert e.dpuf_amd_sample(R.F32, len(self.cache.ctx), V, V, self.x.p, s[0].p, s[1].p, s[2].p, s[3].p, s[4].p,
                                 self.tok.p, self.lp.p, self.sws.p, self.sws_n, stream) == 0

    def results(self):
        """Everything the step writes, as bits."""
        assert self.hip.lib.hipStreamSynchronize(self.stream) == 0
        d = (self.q, self.out, self.lse, self.kept, self.new_len, self.tok, self.lp, self.cache.dk, self.cache.dv,
             self.cache.dw, self.dst.dk, self.dst.dv, self.dst.dw)
        return [x.get().tobytes() for x in d]

    def clear(self):
        """Outputs that no step leaves."""
        for d in (self.q, self.out, self.lse, self.kept, self.new_len, self.tok, self.lp):
            d.set(np.full(d.like.shape, 77, d.like.dtype))
        self.dst.upload_into()


BATCHES = [([1, 1, 1], [900, 70, 1500]), ([1, 60, 0, 2], [33, 700, 20, 1200]), ([140], [300])]


@pytest.mark.parametrize("rows,ctx", BATCHES)
def test_a_captured_step_replays(eng, hip, rows, ctx):
    print(f"graph: rows {rows}, contexts {ctx}", flush=True)
    st = Step(eng, hip, 1, rows, ctx)
    st.enter(0)
    graph, ge = C.c_void_p(), C.c_void_p()
    assert hip.lib.hipStreamBeginCapture(st.stream, 1) == 0
    st.run(st.stream)
    assert hip.lib.hipStreamEndCapture(st.stream, C.byref(graph)) == 0
    assert hip.lib.hipGraphInstantiate(C.byref(ge), graph, None, None, 0) == 0
    for seed in range(5):
        st.enter(seed)
        st.clear()
        st.run(st.stream)
        want = st.results()
        for _ in range(2):
            st.enter(seed)
            st.clear()
            assert hip.lib.hipGraphLaunch(ge, st.stream) == 0
            assert st.results() == want, seed
    hip.lib.hipGraphExecDestroy(ge)
    hip.lib.hipGraphDestroy(graph)
    hip.lib.hipStreamDestroy(st.stream)


def test_steps_on_two_streams(eng, hip):
    print("two streams", flush=True)
    steps = [Step(eng, hip, 10 + i, *BATCHES[i]) for i in range(2)]
    want = []
    for i, st in enumerate(steps):
        st.enter(50 + i)
        st.clear()
        st.run(st.stream)
        want.append(st.results())
    for turn in range(3):
        for i, st in enumerate(steps):
            st.enter(50 + i)
            st.clear()
        hip.sync()
        for st in steps:
            st.run(st.stream)
        for i, st in enumerate(steps):
            assert st.results() == want[i], (turn, i)
    for st in steps:
        hip.lib.hipStreamDestroy(st.stream)


def test_a_query_with_nan_is_alone(eng, hip):
    """NaN in one row's query stays in that row, whichever kernel takes it."""
    for rows, ctx in (([5, 1, 1, 1, 1, 1, 1], [60, 3, 2, 90, 1, 1, 1]), ([100], [150])):
        rng = np.random.default_rng(4)
        cache = R.Cache(hip, rng, R.F16, rows, ctx, NKV, HD, 16)
        q = R.to_type(rng.standard_normal((cache.n_rows, NQ, HD)), R.F16)
        outs = []
        print(f"NaN query: rows {rows}", flush=True)
        for odd in (False, True):
            if odd:
                q[2, 3, 7] = R.to_type([np.nan], R.F16)[0]
            dq, do = hip.put(q), hip.put(np.zeros((cache.n_rows, NQ, HD), np.float32))
            dl = hip.put(np.zeros((cache.n_rows, NQ), np.float32))
            b, p = cache.batch(), cache.pages(w=False)
            n = int(eng.dpuf_amd_paged_attn_workspace(C.byref(b), C.byref(p), NQ))
            ws = hip.put(np.zeros(max(n, 16), np.uint8))
            assert eng.dpuf_amd_paged_attn(C.byref(b), C.byref(p), NQ, dq.p, 0.1, R.F32, do.p, dl.p, ws.p, n, None) == 0
            outs.append((do.get(), dl.get()))
        (o0, l0), (o1, l1) = outs
        assert np.isnan(o1[2, 3]).all() and np.isnan(l1[2, 3])
        o1[2, 3], l1[2, 3] = o0[2, 3], l0[2, 3]
        assert np.array_equal(o0, o1) and np.array_equal(l0, l1)


def test_arguments_that_share_memory_are_refused(eng, hip):
    st = Step(eng, hip, 5, [1, 1], [900, 1500])
    st.enter(0)
    e, r, b, p = eng, C.byref, st.b, st.p
    assert st.ws_n > 0
    attn = dict(q=st.q.p, out=st.out.p, lse=st.lse.p, ws=st.ws.p)

    def attention(**kw):
        a = dict(attn, **kw)
        return e.dpuf_amd_paged_attn(r(b), r(p), NQ, a["q"], 0.09, R.F32, a["out"], a["lse"], a["ws"], st.ws_n, None)

    assert attention() == 0
    for kw in (dict(lse=st.out.p), dict(lse=st.q.p + 16), dict(ws=st.out.p), dict(ws=st.q.p), dict(ws=st.lse.p),
               dict(out=st.q.p)):
        assert attention(**kw) == -1, kw
    assert e.dpuf_amd_paged_attn_weights(r(b), r(p), NQ, st.q.p, 0.09, st.cache.dw.p, 1.0, None, None) == -1
    s = st.settings
    smp = dict(x=st.x.p, u=s[4].p, tok=st.tok.p, lp=st.lp.p, ws=st.sws.p)

    def sample(**kw):
        a = dict(smp, **kw)
        return e.dpuf_amd_sample(R.F32, 2, V, V, a["x"], s[0].p, s[1].p, s[2].p, s[3].p, a["u"], a["tok"], a["lp"],
                                 a["ws"], st.sws_n, None)

    assert sample() == 0
    for kw in (dict(tok=st.x.p), dict(lp=st.tok.p), dict(tok=s[4].p), dict(ws=st.x.p), dict(tok=st.sws.p + 64),
               dict(u=st.sws.p), dict(lp=st.sws.p)):
        assert sample(**kw) == -1, kw
    hip.sync()
    hip.lib.hipStreamDestroy(st.stream)


def test_pools_beyond_32_bits(eng, hip):
    """Pages 2^27 elements apart, 24 of them: the same bits as side by side."""
    rng = np.random.default_rng(6)
    rows, ctx, page = [1, 70, 0, 2], [130, 90, 3, 60], 16
    c = R.Cache(hip, rng, R.F16, rows, ctx, NKV, 64, page)
    stride, size = 1 << 27, page * NKV * 64
    far = []
    print("far pages", flush=True)
    for pool in (c.k, c.v):
        d = C.c_void_p()
        assert hip.lib.hipMalloc(C.byref(d), c.n * stride * 2) == 0
        far.append(d.value)
        for p in range(c.n):
            assert hip.lib.hipMemcpy(d.value + p * stride * 2, pool[p].ctypes.data, size * 2, R.H2D) == 0
    assert c.n >= 20
    dw = hip.put(c.w)
    near, wide = c.pages(), c.pages(dw=dw)
    wide.k, wide.v, wide.page_stride = far[0], far[1], stride
    qkv = hip.put(rng.standard_normal((c.n_rows, (4 + 2 * NKV) * 64)).astype(np.float32))
    turns = hip.put(1e4 ** (-np.arange(32) / 32) / 6.283185307179586)
    rope = abi.DpufAmdRope(turns=turns.p, rot_dim=64, interleaved=1, scale=1.0)
    pos = hip.put(np.arange(c.n_rows, dtype=np.int32))
    got = []
    for p in (near, wide):
        b, w = c.batch(), (4 + 2 * NKV) * 64
        dq, do = hip.put(np.zeros((c.n_rows, 4, 64), np.uint16)), hip.put(np.zeros((c.n_rows, 4, 64), np.uint16))
        dl, kept = hip.put(np.zeros((c.n_rows, 4), np.float32)), hip.put(np.zeros((4, NKV, 40), np.int32))
        new = hip.put(np.zeros(4, np.int32))
        dst = R.Cache(hip, np.random.default_rng(7), R.F16, [0] * 4, [40] * 4, NKV, 64, page)
        assert eng.dpuf_amd_rope_append(C.byref(b), C.byref(p), C.byref(rope), pos.p, R.F32, 4, qkv.p, qkv.p + 4 * 256,
                                        qkv.p + (4 + NKV) * 256, w, w, w, None, None, 0.0, dq.p, None) == 0
        n = int(eng.dpuf_amd_paged_attn_workspace(C.byref(b), C.byref(p), 4))
        ws = hip.put(np.zeros(max(n, 16), np.uint8))
        assert eng.dpuf_amd_paged_attn(C.byref(b), C.byref(p), 4, dq.p, 0.1, R.F16, do.p, dl.p, ws.p, n, None) == 0
        assert eng.dpuf_amd_paged_attn_weights(C.byref(b), C.byref(p), 4, dq.p, 0.1, dl.p, 0.5, p.w, None) == 0
        dp = dst.pages()
        assert eng.dpuf_amd_paged_evict(C.byref(b), C.byref(p), 40, 1, 4, C.byref(dp), dst.d_table.p,
                                        dst.table.shape[1], kept.p, new.p, None) == 0
        got.append([x.get().tobytes() for x in (dq, do, dl, kept, new, dst.dk, dst.dv, dst.dw)])
    assert got[0] == got[1]
    back = np.empty_like(c.k)
    for f, d in zip(far, (c.dk, c.dv)):
        want = d.get()
        for p in range(c.n):
            assert hip.lib.hipMemcpy(back[p].ctypes.data, f + p * stride * 2, size * 2, R.D2H) == 0
        assert np.array_equal(back, want)
        hip.lib.hipFree(f)
    assert np.array_equal(dw.get().view(np.uint32), c.dw.get().view(np.uint32))


def test_many_sequences(eng, hip):
    """Hundreds of sequences of none to a few rows and one chunk among them."""
    rng = np.random.default_rng(8)
    n = 700
    ctx = rng.integers(0, 50, n).tolist()
    rows = [int(rng.integers(0, min(4, c + 1))) for c in ctx]
    ctx[333], rows[333] = 200, 150
    c = R.Cache(hip, rng, R.BF16, rows, ctx, 1, 64, 16)
    q = R.to_type(rng.standard_normal((c.n_rows, 4, 64)), R.BF16)
    dq, do = hip.put(q), hip.put(np.zeros((c.n_rows, 4, 64), np.float32))
    dl = hip.put(np.zeros((c.n_rows, 4), np.float32))
    ref, rl, A, S, vmax, fresh = R.attention(c, R.from_type(q, R.BF16), float(np.float32(0.1)), 4)
    bound = R.attention_bound(R.BF16, R.F32, ref, A, S, vmax, 64, 200)
    seen = np.isfinite(rl)
    for max_ctx in (50, 3000):
        print(f"{n} sequences, max_ctx {max_ctx}", flush=True)
        b, p = c.batch(max_ctx=max_ctx), c.pages()
        b.table_stride = c.table.shape[1]
        ws_n = int(eng.dpuf_amd_paged_attn_workspace(C.byref(b), C.byref(p), 4))
        ws = hip.put(np.full(max(ws_n, 16), 0xFF, np.uint8))
        assert eng.dpuf_amd_paged_attn(C.byref(b), C.byref(p), 4, dq.p, 0.1, R.F32, do.p, dl.p, ws.p, ws_n, None) == 0
        out, lse = do.get(), dl.get()
        assert np.all(np.abs(out - ref) <= bound)
        assert np.array_equal(np.isneginf(lse), ~seen)
        c.dw.set(c.w)
        assert eng.dpuf_amd_paged_attn_weights(C.byref(b), C.byref(p), 4, dq.p, 0.1, dl.p, 1.0, None, None) == 0
        w = c.dw.get()
        # as the weights' own tests: two score errors, the log sum's rounding, sums of every row's share
        rel = 2 * R.score_error(S.max(), 64) + np.abs(rl[seen]).max() * 2.0 ** -22 + 2.0 ** -20 + 640 * 2.0 ** -24
        for s in range(n):
            for i in range(ctx[s]):
                x = w[c.table[s, i // 16], 0, i % 16]
                assert abs(x - fresh[s][0, i]) <= rel * fresh[s][0, i] + 1e-30, (s, i)


def test_outputs_in_memory_that_a_call_reads_are_refused(eng, hip):
    """Every output and workspace of every operator, laid into each of the
    inputs, tables and pools that the call reads or also writes: refused, and
    nothing of the call is done."""
    st = Step(eng, hip, 5, [1, 1, 2], [900, 1500, 40])
    st.enter(0)
    e, r, c = eng, C.byref, st.cache
    assert st.ws_n > 0
    width = (NQ + 2 * NKV) * HD
    scratch = hip.put(np.zeros(1 << 20, np.uint8))
    tables = dict(starts=c.d_starts.p, ctx=c.d_ctx.p, table=c.d_table.p)
    pools = dict(k=c.dk.p + 4096, v=c.dv.p + 4096, w=c.dw.p + 64)

    def pages(w=None, k=None, v=None):
        p = c.pages()
        p.w, p.k, p.v = w or p.w, k or p.k, v or p.v
        return p

    at = st.qkv.p
    ok_rope = dict(q=at, k=at + NQ * HD * 4, v=at + (NQ + NKV) * HD * 4, pos=st.pos.p, out=st.q.p, turns=st.rope.turns,
                   norm=scratch.p, p=pages())

    def rope(**kw):
        a = dict(ok_rope, **kw)
        s = abi.DpufAmdRope(turns=a["turns"], rot_dim=HD, interleaved=0, scale=1.0)
        return e.dpuf_amd_rope_append(r(st.b), r(a["p"]), r(s), a["pos"], R.F32, NQ, a["q"], a["k"], a["v"], width,
                                      width, width, a["norm"], None, 1e-6, a["out"], st.stream)

    def attn(**kw):
        a = dict(dict(q=st.q.p, out=st.out.p, lse=st.lse.p, ws=st.ws.p), **kw)
        return e.dpuf_amd_paged_attn(r(st.b), r(st.p), NQ, a["q"], 0.09, R.F32, a["out"], a["lse"], a["ws"], st.ws_n,
                                     st.stream)

    def weights(**kw):
        a = dict(dict(p=pages(), q=st.q.p, lse=st.lse.p, w_in=None), **kw)
        return e.dpuf_amd_paged_attn_weights(r(st.b), r(a["p"]), NQ, a["q"], 0.09, a["lse"], 0.9, a["w_in"], st.stream)

    def evict(**kw):
        a = dict(dict(p=pages(), dp=st.dp, dt=st.dst.d_table.p, kept=st.kept.p, new=st.new_len.p), **kw)
        return e.dpuf_amd_paged_evict(r(st.b), r(a["p"]), KEEP, 2, 8, r(a["dp"]), a["dt"], st.dst.table.shape[1],
                                      a["kept"], a["new"], st.stream)

    # what stays allowed, weights in place among it
    for call in (rope, attn, weights, evict):
        assert call() == 0
    assert weights(w_in=c.dw.p) == 0
    hip.sync()
    before = [x.get().tobytes() for x in (st.q, st.out, st.lse, st.kept, st.new_len, c.dk, c.dv, c.dw, c.d_starts,
                                          c.d_ctx, c.d_table, st.qkv, st.dst.dk, st.dst.dv, st.dst.dw, st.dst.d_table)]
    bad = []
    for name, x in {**tables, **pools, "pos": st.pos.p, "turns": st.rope.turns, "norm": scratch.p}.items():
        bad.append((f"rope: out in {name}", lambda x=x: rope(out=x & ~15)))
    for name in ("q", "k", "v", "pos", "turns"):
        for pool, x in pools.items():
            bad.append((f"rope: {name} in {pool}", lambda x=x, name=name: rope(**{name: x})))
    bad += [("rope: w in k", lambda: rope(p=pages(w=pools["k"]))), ("rope: w in v", lambda: rope(p=pages(w=pools["v"]))),
            ("rope: w in the table", lambda: rope(p=pages(w=c.d_table.p)))]
    for name, x in {**tables, "k": pools["k"], "v": pools["v"], "q": st.q.p}.items():
        for what in ("out", "lse", "ws"):
            bad.append((f"attention: {what} in {name}", lambda x=x, what=what: attn(**{what: x & ~15})))
        if name != "v":
            bad.append((f"weights: w in {name}", lambda x=x: weights(p=pages(w=x))))
    bad += [("weights: w in lse", lambda: weights(p=pages(w=st.lse.p))),
            ("weights: w_in beside w", lambda: weights(w_in=c.dw.p + 4))]
    dst = dict(dst_k=st.dst.dk.p, dst_v=st.dst.dv.p, dst_w=st.dst.dw.p, dst_table=st.dst.d_table.p)
    for name, x in {**tables, **pools, **dst}.items():
        for what in ("kept", "new"):
            if name != "starts":
                bad.append((f"evict: {what} in {name}", lambda x=x, what=what: evict(**{what: x})))

    def dst_pages(**kw):
        p = st.dst.pages()
        for k, x in kw.items():
            setattr(p, k, x)
        return p

    for kw in (dict(w=pools["k"]), dict(w=pools["v"]), dict(w=c.d_table.p), dict(w=st.dst.dk.p), dict(k=c.dw.p),
               dict(v=c.dw.p), dict(k=c.d_table.p & ~15), dict(w=st.dst.d_table.p), dict(v=st.dst.d_table.p & ~15)):
        bad.append((f"evict: destination {list(kw)}", lambda kw=kw: evict(dp=dst_pages(**kw))))
    print(f"{len(bad)} calls with shared memory", flush=True)
    for name, call in bad:
        assert call() == -1, name
    hip.sync()
    after = [x.get().tobytes() for x in (st.q, st.out, st.lse, st.kept, st.new_len, c.dk, c.dv, c.dw, c.d_starts,
                                         c.d_ctx, c.d_table, st.qkv, st.dst.dk, st.dst.dv, st.dst.dw, st.dst.d_table)]
    assert before == after
    hip.lib.hipStreamDestroy(st.stream)


def test_keys_and_values_in_one_allocation(eng, hip):
    """K and V rows interleaved page by page, and eviction into other pages of
    the same pool: the same bits as in pools of their own."""
    rng = np.random.default_rng(21)
    page, n = 16, 24
    size = NKV * page * HD
    kv = R.to_type(rng.standard_normal((n, 2, NKV, page, HD)), R.BF16)
    w = np.exp(rng.standard_normal((n, NKV, page))).astype(np.float32)
    table = np.array([[3, 9, 1, 20], [7, 0, -1, -1]], np.int32)
    dst_table = np.array([[4, 5], [6, 8]], np.int32)
    ctx, starts = np.array([60, 20], np.int32), np.array([0, 2, 3], np.int32)
    qkv = rng.standard_normal((3, (NQ + 2 * NKV) * HD)).astype(np.float32)
    turns, pos = 1e4 ** (-np.arange(64) / 64) / 6.283185307179586, np.array([100, 101, 30], np.int32)
    got = []
    print("interleaved pages", flush=True)
    for together in (0, 1):
        if together:
            d = hip.put(kv)
            k, v, stride = d.p, d.p + 2 * size, 2 * size
        else:
            d = [hip.put(np.ascontiguousarray(kv[:, i])) for i in range(2)]
            k, v, stride = d[0].p, d[1].p, size
        put = hip.put
        dw, dt, dd, dc, ds = put(w), put(table), put(dst_table), put(ctx), put(starts)
        p = abi.DpufAmdPages(type=R.BF16, n_pages=n, page_size=page, n_kv_heads=NKV, head_dim=HD, page_stride=stride,
                             head_stride=page * HD, row_stride=HD, k=k, v=v, w=dw.p)
        b = abi.DpufAmdBatch(n_seqs=2, n_rows=3, table_stride=4, max_ctx=60, row_start=ds.p, ctx_len=dc.p,
                             page_table=dt.p)
        dq = put(qkv)
        q, out, lse = (put(np.zeros(s, t)) for s, t in (((3, NQ, HD), np.uint16), ((3, NQ, HD), np.float32),
                                                        ((3, NQ), np.float32)))
        kept, new, dp = put(np.zeros((2, NKV, 32), np.int32)), put(np.zeros(2, np.int32)), put(pos)
        rope = abi.DpufAmdRope(turns=put(turns).p, rot_dim=HD, interleaved=0, scale=1.0)
        wid = (NQ + 2 * NKV) * HD
        assert eng.dpuf_amd_rope_append(C.byref(b), C.byref(p), C.byref(rope), dp.p, R.F32, NQ, dq.p, dq.p + NQ * HD * 4,
                                        dq.p + (NQ + NKV) * HD * 4, wid, wid, wid, None, None, 0.0, q.p, None) == 0
        ws_n = int(eng.dpuf_amd_paged_attn_workspace(C.byref(b), C.byref(p), NQ))
        ws = put(np.zeros(max(16, ws_n), np.uint8))
        assert eng.dpuf_amd_paged_attn(C.byref(b), C.byref(p), NQ, q.p, 0.09, R.F32, out.p, lse.p, ws.p, ws_n, None) == 0
        assert eng.dpuf_amd_paged_attn_weights(C.byref(b), C.byref(p), NQ, q.p, 0.09, lse.p, 0.9, dw.p, None) == 0
        assert eng.dpuf_amd_paged_evict(C.byref(b), C.byref(p), 32, 2, 4, C.byref(p), dd.p, 2, kept.p, new.p, None) == 0
        pools = [d.get()[:, i] for i in range(2)] if together else [x.get() for x in d]
        got.append([x.tobytes() for x in (q.get(), out.get(), lse.get(), kept.get(), new.get(), dw.get(), *pools)])
    assert got[0] == got[1]
