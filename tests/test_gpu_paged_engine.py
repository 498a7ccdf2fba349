"""The engine over a paged cache and with sampling.

The pass over pages is checked bit for bit against its parts put together by
hand: the oracle's embedding, norms, projections and SwiGLU on the host, and
between them the paged operators (each tested against float64 by itself) on a
cache of the test's own.  A conversation runs as a serving program has it:
prompts, chunks of prompts and single tokens of several sequences in one pass,
weights kept, eviction, sampling, and on from there."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from dpuf_amd import abi
from dpuf_amd import model as M
from test_gpu_sample import one

pytestmark = pytest.mark.gpu

V = 768


@pytest.fixture()
def hip(eng):
    h = R.Hip()
    yield h
    h.free_all()


def say(*a):
    print(*a, flush=True)


class Parts:
    """A Mode 12 model's pass over pages, put together from its parts."""

    def __init__(self, eng, orc, hip, model, n_pages, page, t):
        self.eng, self.orc, self.hip, self.m, self.t = eng, orc, hip, model, t
        c = self.c = model.cfg.contents
        self.H, self.I, self.L = c.hidden_size, c.intermediate_size, c.num_layers
        self.nq, self.nkv, self.hd = c.num_q_heads, c.num_kv_heads, c.head_dim
        z = np.zeros((n_pages, self.nkv, page, self.hd), np.uint16)
        self.pool = [(hip.put(z), hip.put(z), hip.put(np.zeros((n_pages, self.nkv, page), np.float32)))
                     for _ in range(self.L)]
        self.n_pages, self.page = n_pages, page
        spec = abi.DpufAmdRopeSpec(rot_dim=self.hd, theta=c.rope_theta, scaling=0, factor=1.0)
        turns, s = np.zeros(self.hd // 2), C.c_float(0)
        assert eng.dpuf_amd_rope_turns(C.byref(spec), turns.ctypes.data_as(C.c_void_p), C.byref(s)) == 0
        self.turns = hip.put(turns)
        self.rope = abi.DpufAmdRope(turns=self.turns.p, rot_dim=self.hd, interleaved=0, scale=s.value)

    def pages(self, l):
        k, v, w = self.pool[l]
        it = self.hd
        return abi.DpufAmdPages(type=self.t, n_pages=self.n_pages, page_size=self.page, n_kv_heads=self.nkv, head_dim=it,
                                page_stride=self.nkv * self.page * it, head_stride=self.page * it, row_stride=it,
                                k=k.p, v=v.p, w=w.p)

    def matmul(self, d, x):
        out = np.zeros((x.shape[0], d.rows), np.float32)
        self.orc.orc_matmul_f32(x.shape[0], d.rows, d.cols, d.n_tiles, M.ptr(np.ascontiguousarray(x)), d.tensor_base,
                                d.tile_offsets, d.sign_bits, M.ptr(out))
        return out

    def norm(self, h, res, w):
        """(h + res, its norm), row by row."""
        h = h.copy()
        out = np.zeros_like(h)
        for i in range(h.shape[0]):
            r = M.ptr(res[i].copy()) if res is not None else None
            row, o = h[i].copy(), np.zeros(h.shape[1], np.float32)
            self.orc.orc_add_rmsnorm(h.shape[1], M.ptr(row), r, w, C.c_float(self.c.rms_eps), M.ptr(o))
            h[i], out[i] = row, o
        return h, out

    def forward(self, rows, ctx, table, ids, pos, decay):
        eng, hip = self.eng, self.hip
        n, rows_n = len(rows), int(sum(rows))
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        ds, dc, dt, dp = hip.put(starts), hip.put(ctx), hip.put(table), hip.put(pos)
        b = abi.DpufAmdBatch(n_seqs=n, n_rows=rows_n, table_stride=table.shape[1], max_ctx=int(max(ctx)),
                             row_start=ds.p, ctx_len=dc.p, page_table=dt.p)
        tok = self.m.tok.contents
        h = np.zeros((rows_n, self.H), np.float32)
        self.orc.orc_embed(rows_n, self.H, M.ptr(ids), tok.tensor_base, tok.tile_offsets, tok.sign_bits, M.ptr(h))
        res = None
        scale = float(np.float32(1.0) / np.sqrt(np.float32(self.hd)))
        for l in range(self.L):
            lw, p = self.m.layers[l], self.pages(l)
            h, x = self.norm(h, res, lw.attn_norm)
            q, k, v = (hip.put(self.matmul(d, x)) for d in (lw.w_q, lw.w_k, lw.w_v))
            qn, kn = (hip.put(np.ctypeslib.as_array(C.cast(a, C.POINTER(C.c_float)), (self.hd,)).copy()) if a else None
                      for a in (lw.attn_q_norm, lw.attn_k_norm))
            q16 = hip.put(np.zeros((rows_n, self.nq, self.hd), np.uint16))
            ao, lse = hip.put(np.zeros((rows_n, self.nq * self.hd), np.float32)), hip.put(
                np.zeros((rows_n, self.nq), np.float32))
            assert eng.dpuf_amd_rope_append(C.byref(b), C.byref(p), C.byref(self.rope), dp.p, R.F32, self.nq, q.p, k.p,
                                            v.p, self.nq * self.hd, self.nkv * self.hd, self.nkv * self.hd,
                                            qn.p if qn else None, kn.p if kn else None, self.c.rms_eps, q16.p,
                                            None) == 0
            need = int(eng.dpuf_amd_paged_attn_workspace(C.byref(b), C.byref(p), self.nq))
            ws = hip.put(np.zeros(max(need, 16), np.uint8))
            assert eng.dpuf_amd_paged_attn(C.byref(b), C.byref(p), self.nq, q16.p, scale, R.F32, ao.p, lse.p, ws.p, need,
                                           None) == 0
            if decay >= 0:
                assert eng.dpuf_amd_paged_attn_weights(C.byref(b), C.byref(p), self.nq, q16.p, scale, lse.p, decay, p.w,
                                                       None) == 0
            o = self.matmul(lw.w_o, ao.get())
            h, x = self.norm(h, o, lw.ffn_norm)
            g, u = self.matmul(lw.w_gate, x), self.matmul(lw.w_up, x)
            sw = np.array([self.orc.orc_swiglu1(C.c_float(a), C.c_float(c_), C.c_float(0.005)) for a, c_ in
                           zip(g.ravel().tolist(), u.ravel().tolist())], np.float32).reshape(g.shape)
            res = self.matmul(lw.w_down, sw)
        last = starts[1:] - 1
        _, x = self.norm(h[last], res[last], self.m.out_norm)
        return self.matmul(self.m.lm.contents, x)

    def evict(self, ctx, table, dst, keep, sink, recent):
        hip = self.hip
        n = len(ctx)
        dc, dt, dd = hip.put(ctx), hip.put(table), hip.put(dst)
        kept, new = hip.put(np.zeros((n, self.nkv, keep), np.int32)), hip.put(np.zeros(n, np.int32))
        b = abi.DpufAmdBatch(n_seqs=n, n_rows=0, table_stride=table.shape[1], max_ctx=1, row_start=None, ctx_len=dc.p,
                             page_table=dt.p)
        for l in range(self.L):
            p = self.pages(l)
            assert self.eng.dpuf_amd_paged_evict(C.byref(b), C.byref(p), keep, sink, recent, C.byref(p), dd.p,
                                                 dst.shape[1], kept.p, new.p, None) == 0
        return new.get()


def settings(n, rng):
    """Host arrays of n sequences' settings, the first greedy."""
    t = (0.3 + rng.random(n)).astype(np.float32)
    t[0] = 0.0
    a = dict(temperature=t, top_k=rng.integers(0, 40, n).astype(np.int32),
             top_p=(0.5 + 0.6 * rng.random(n)).astype(np.float32), min_p=(0.1 * rng.random(n)).astype(np.float32),
             u=rng.random(n).astype(np.float32))
    return a, abi.DpufAmdSampling(**{k: v.ctypes.data for k, v in a.items()})


def drawn(a, i, logits):
    return one(logits.astype(np.float64), *(float(a[k][i]) for k in ("temperature",)), int(a["top_k"][i]),
               float(a["top_p"][i]), float(a["min_p"][i]), float(a["u"][i]))


@pytest.mark.parametrize("nq,nkv,hd,page,t,qk_norm", [(4, 2, 64, 16, R.BF16, 1), (8, 1, 128, 32, R.F16, 1),
                                                     (3, 3, 256, 16, R.BF16, 0)])
def test_conversation(eng, orc, hip, nq, nkv, hd, page, t, qk_norm):
    shape = dict(hidden_size=256, intermediate_size=512, num_layers=2, num_q_heads=nq, num_kv_heads=nkv, head_dim=hd,
                 vocab_size=V, tie_word_embeddings=1)
    m = M.Model.build(shape, max_seq_len=32, seed=77)
    m.cfg.contents.has_qk_norm = qk_norm
    if not qk_norm:
        for l in range(2):
            m.layers[l].attn_q_norm = m.layers[l].attn_k_norm = None
    h = eng.dpuf_engine_create(*m.create_args())
    assert h
    n_pages = 48
    assert eng.dpuf_amd_engine_pages_create(h, n_pages, page, t) == 0
    parts = Parts(eng, orc, hip, m, n_pages, page, t)
    rng = np.random.default_rng(78)
    free = list(rng.permutation(n_pages))
    seqs = {}      # name -> [pages, cached rows, next position]

    def step(work, decay):
        """work: [(name, token ids)] in one pass; returns (logits, drawn tokens)."""
        for name, ids in work:
            s = seqs.setdefault(name, [[], 0, 0])
            s[1] += len(ids)
            while len(s[0]) * page < s[1]:
                s[0].append(free.pop())
        width = max(len(seqs[name][0]) for name, _ in work) + 1
        table = np.full((len(work), width), -1, np.int32)
        rows = np.array([len(ids) for _, ids in work], np.int32)
        ctx = np.array([seqs[name][1] for name, _ in work], np.int32)
        pos = []
        for i, (name, ids) in enumerate(work):
            s = seqs[name]
            table[i, :len(s[0])] = s[0]
            pos += list(range(s[2], s[2] + len(ids)))
            s[2] += len(ids)
        pos = np.array(pos, np.int32)
        ids = np.concatenate([np.asarray(i, np.int32) for _, i in work])
        a, smp = settings(len(work), rng)
        lg, toks = np.zeros((len(work), V), np.float32), np.full(len(work), -9, np.int32)
        lp = np.zeros(len(work), np.float32)
        say(f"  pass: rows {rows.tolist()}, contexts {ctx.tolist()}, decay {decay}")
        rc = eng.dpuf_amd_engine_forward_pages(h, len(work), M.ptr(rows), M.ptr(ctx), M.ptr(table), width, M.ptr(ids),
                                               M.ptr(pos), decay, C.byref(smp), M.ptr(lg), M.ptr(toks), M.ptr(lp))
        assert rc == 0, (rc, eng.dpuf_amd_last_error())
        want = parts.forward(rows, ctx, table, ids, pos, decay)
        assert np.array_equal(lg.view(np.uint32), want.view(np.uint32)), np.abs(lg - want).max()
        for i in range(len(work)):
            tok, wl = drawn(a, i, lg[i])
            assert toks[i] == tok and abs(lp[i] - wl) <= abs(wl) * 2.0 ** -23 + 2.0 ** -27
        return lg, toks

    say(f"conversation: {nq}/{nkv} heads of {hd}, pages of {page}, type {t}")
    prompt = lambda n: rng.integers(0, V, n)
    _, a = step([("a", prompt(5)), ("b", prompt(37)), ("c", prompt(1))], 1.0)
    _, a = step([("a", [a[0]]), ("b", [a[1]]), ("c", prompt(20))], 0.9)
    for _ in range(2):
        _, a = step([("c", [a[2]]), ("a", [a[0]]), ("b", [a[1]])], 0.9)
        a = a[[1, 2, 0]]
    lone, _ = step([("b", [a[1]])], -1.0)            # one row of one sequence: the one-row projections
    # every sequence down to 18 rows at most, in pages of its own
    names = ["a", "b", "c"]
    keep = 18
    width = max(len(seqs[x][0]) for x in names)
    table = np.full((3, width), -1, np.int32)
    dst = np.full((3, -(-keep // page)), -1, np.int32)
    ctx = np.array([seqs[x][1] for x in names], np.int32)
    for i, x in enumerate(names):
        table[i, :len(seqs[x][0])] = seqs[x][0]
        need = -(-min(int(ctx[i]), keep) // page)
        dst[i, :need] = [free.pop() for _ in range(need)]
    new = np.zeros(3, np.int32)
    say(f"  evict: contexts {ctx.tolist()} to {keep}")
    rc = eng.dpuf_amd_engine_evict_pages(h, 3, M.ptr(ctx), M.ptr(table), width, keep, 2, 5, M.ptr(dst), dst.shape[1],
                                         M.ptr(new))
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    assert np.array_equal(new, np.minimum(ctx, keep)) and np.array_equal(parts.evict(ctx, table, dst, keep, 2, 5), new)
    for i, x in enumerate(names):
        free.extend(seqs[x][0])
        seqs[x][0], seqs[x][1] = [p for p in dst[i] if p >= 0], int(new[i])
    _, a = step([("a", [a[0]]), ("b", [3]), ("c", prompt(33))], 0.5)
    step([("b", [a[1]]), ("d", prompt(3))], 0.5)
    # every layer's pages hold what the operators left in the test's own
    for l in range(2):
        p = abi.DpufAmdPages()
        assert eng.dpuf_amd_engine_pages(h, l, C.byref(p)) == 0
        for mine, theirs in zip(parts.pool[l], (p.k, p.v, p.w)):
            got = np.empty_like(mine.like)
            assert hip.lib.hipMemcpy(M.ptr(got), theirs, got.nbytes, R.D2H) == 0
            want = mine.get()
            assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
    assert eng.dpuf_amd_engine_pages_create(h, 0, 0, 0) == 0
    eng.dpuf_engine_destroy(h)


def _engine(eng, max_seq=64):
    shape = dict(hidden_size=256, intermediate_size=256, num_layers=2, num_q_heads=4, num_kv_heads=2, head_dim=64,
                 vocab_size=V, tie_word_embeddings=1)
    m = M.Model.build(shape, max_seq_len=max_seq, seed=5)
    return m, eng.dpuf_engine_create(*m.create_args())


def test_pages_agree_with_slots(eng):
    """The same prompt through pages and through a slot: the 16-bit cache moves
    the first layer's logits by about its rounding; with the pass cut into
    chunks the pages' logits stay as close.  (Bounds: a bf16 cache rounds keys,
    values, queries and probabilities by 2^-8 each; of logits with a standard
    deviation s the rows here move by well under s, a wrong position or mask by
    about s.)"""
    shape = dict(hidden_size=256, intermediate_size=256, num_layers=1, num_q_heads=4, num_kv_heads=2, head_dim=64,
                 vocab_size=V, tie_word_embeddings=1)
    m = M.Model.build(shape, max_seq_len=64, seed=5)
    h = eng.dpuf_engine_create(*m.create_args())
    rng = np.random.default_rng(6)
    ids = rng.integers(0, V, 40).astype(np.int32)
    want = np.zeros(V, np.float32)
    assert eng.dpuf_engine_forward_batch(h, 40, M.ptr(ids), 0, 1, M.ptr(want)) == 0
    assert eng.dpuf_amd_engine_pages_create(h, 4, 16, R.BF16) == 0
    table = np.array([[2, 0, 3]], np.int32)
    for cuts in ([40], [17, 23], [39, 1]):
        at = 0
        got = np.zeros((1, V), np.float32)
        for n in cuts:
            rows, ctx = np.array([n], np.int32), np.array([at + n], np.int32)
            pos = np.arange(at, at + n, dtype=np.int32)
            assert eng.dpuf_amd_engine_forward_pages(h, 1, M.ptr(rows), M.ptr(ctx), M.ptr(table), 3, M.ptr(ids[at:at + n].copy()),
                                                     M.ptr(pos), -1.0, None, M.ptr(got), None, None) == 0
            at += n
        off = np.abs(got[0] - want).max() / want.std()
        say(f"  cuts {cuts}: {off:.4f} standard deviations off")
        assert off < 0.5
    eng.dpuf_engine_destroy(h)


def test_sampled_steps_of_slots(eng, hip):
    """forward_sample (eager and replayed) and forward_slots_sample: the logits
    of the greedy entry points, and tokens drawn from exactly those."""
    m, h = _engine(eng)
    rng = np.random.default_rng(9)
    ids = rng.integers(0, V, 12).astype(np.int32)
    a, smp = settings(3, rng)
    one_of = lambda i: {k: v[i:i + 1] for k, v in a.items()}
    tok, lp = np.zeros(1, np.int32), np.zeros(1, np.float32)
    for n, pos in ((12, 0), (1, 12), (1, 13), (1, 12)):
        for i in range(3):
            x = one_of(i)
            s = abi.DpufAmdSampling(**{k: v.ctypes.data for k, v in x.items()})
            lg, ref, g = np.zeros(V, np.float32), np.zeros(V, np.float32), np.zeros(1, np.int32)
            for graph in (0, 1):
                assert eng.dpuf_amd_engine_forward_argmax(h, n, M.ptr(ids), pos, None, graph, M.ptr(g), M.ptr(ref)) == 0
                assert eng.dpuf_amd_engine_forward_sample(h, n, M.ptr(ids), pos, None, graph, C.byref(s), M.ptr(tok),
                                                          M.ptr(lp), M.ptr(lg)) == 0
                assert np.array_equal(lg.view(np.uint32), ref.view(np.uint32))
                want, wl = drawn(x, 0, lg)
                assert tok[0] == want and abs(lp[0] - wl) <= abs(wl) * 2.0 ** -23 + 2.0 ** -27
                if x["temperature"][0] == 0:
                    assert tok[0] == g[0]
    # three sessions, the middle one long enough for the other attention path
    slots, pos = np.array([4, 0, 2], np.int32), np.array([0, 13, 3], np.int32)
    toks = rng.integers(0, V, 3).astype(np.int32)
    lg, ref = np.zeros((3, V), np.float32), np.zeros((3, V), np.float32)
    out, lps = np.zeros(3, np.int32), np.zeros(3, np.float32)
    assert eng.dpuf_amd_engine_forward_slots(h, 3, M.ptr(slots), M.ptr(toks), M.ptr(pos), M.ptr(ref), M.ptr(out)) == 0
    assert eng.dpuf_amd_engine_forward_slots_sample(h, 3, M.ptr(slots), M.ptr(toks), M.ptr(pos), C.byref(smp),
                                                    M.ptr(lg), M.ptr(out), M.ptr(lps)) == 0
    assert np.array_equal(lg.view(np.uint32), ref.view(np.uint32))
    for i in range(3):
        want, wl = drawn(a, i, lg[i])
        assert out[i] == want and abs(lps[i] - wl) <= abs(wl) * 2.0 ** -23 + 2.0 ** -27
    eng.dpuf_engine_destroy(h)


def test_engine_refusals(eng):
    m, h = _engine(eng)
    i32 = lambda *v: np.array(v, np.int32)
    tok, lg = np.zeros(4, np.int32), np.zeros((4, V), np.float32)
    base = dict(n=2, rows=i32(1, 2), ctx=i32(3, 17), table=i32(0, -1, 2, 5), stride=2, ids=i32(1, 2, 3),
                pos=i32(0, 1, 2), decay=-1.0, smp=None, lg=lg, tok=tok, lp=None)

    def run(**kw):
        d = dict(base, **kw)
        p = lambda x: M.ptr(x) if x is not None else None
        return eng.dpuf_amd_engine_forward_pages(h, d["n"], p(d["rows"]), p(d["ctx"]), p(d["table"]), d["stride"],
                                                 p(d["ids"]), p(d["pos"]), d["decay"],
                                                 C.byref(d["smp"]) if d["smp"] else None, p(d["lg"]), p(d["tok"]),
                                                 p(d["lp"]))

    assert run() == -1                                     # no pages yet
    for args, code in (((-1, 16, 1), -2), ((8, 8, 1), -2), ((8, 24, 1), -2), ((8, 2048, 1), -2), ((8, 16, 0), -5),
                       ((8, 16, 3), -5), ((8, 16, 1), 0)):
        assert eng.dpuf_amd_engine_pages_create(h, *args) == code, args
    assert eng.dpuf_amd_engine_pages_create(None, 8, 16, 1) == -1
    assert run() == 0
    assert eng.dpuf_amd_engine_pages(h, 2, C.byref(abi.DpufAmdPages())) == -1
    none = abi.DpufAmdSampling()
    u = np.full(2, 0.5, np.float32)
    some = abi.DpufAmdSampling(u=u.ctypes.data)
    lp = np.zeros(2, np.float32)
    for kw, code in ((dict(rows=None), -1), (dict(ids=None), -1), (dict(pos=None), -1), (dict(table=None), -1),
                     (dict(lg=None, tok=None), -1), (dict(smp=none), -1), (dict(smp=some, tok=None), -1),
                     (dict(lp=lp), -1), (dict(decay=float("nan")), -1), (dict(decay=float("inf")), -1),
                     (dict(n=0), -2), (dict(n=513), -2), (dict(stride=0), -2), (dict(stride=1 << 27), -2),
                     (dict(rows=i32(0, 2)), -2), (dict(rows=i32(1, 512)), -2), (dict(ctx=i32(0, 17)), -3),
                     (dict(ctx=i32(3, 33)), -3), (dict(ctx=i32(17, 17)), -3), (dict(table=i32(8, -1, 2, 5)), -3),
                     (dict(table=i32(0, -1, 2, -5)), -3), (dict(pos=i32(0, -1, 2)), -3), (dict(ids=i32(1, 2, V)), -4),
                     (dict(ids=i32(-1, 2, 3)), -4), (dict(table=i32(2, -1, 2, 5)), -1),
                     (dict(table=i32(0, -1, 5, 5)), -1)):
        assert run(**kw) == code, kw
    # a shared first page is fine to read (the second sequence's new rows lie behind it), not with weights kept
    shared = dict(rows=i32(1, 1), ctx=i32(18, 17), table=i32(2, 4, 2, 5), ids=i32(1, 2), pos=i32(0, 1))
    assert run(**shared) == 0 and run(**dict(shared, decay=1.0)) == -1
    new = i32(0, 0)

    def evict(**kw):
        d = dict(dict(n=2, ctx=i32(3, 17), table=i32(0, -1, 2, 5), stride=2, keep=4, sink=1, recent=2, dst=i32(1, 3),
                      dstride=1), **kw)
        return eng.dpuf_amd_engine_evict_pages(h, d["n"], M.ptr(d["ctx"]), M.ptr(d["table"]), d["stride"], d["keep"],
                                               d["sink"], d["recent"], M.ptr(d["dst"]), d["dstride"], M.ptr(new))

    assert evict() == 0 and new.tolist() == [3, 4]
    for kw, code in ((dict(n=0), -2), (dict(keep=0), -2), (dict(keep=17), -2), (dict(sink=-1), -2), (dict(recent=4), -2),
                     (dict(dst=i32(1, 1)), -1), (dict(dst=i32(0, 3)), -1), (dict(dst=i32(5, 3)), -1),
                     (dict(dst=i32(8, 3)), -3), (dict(ctx=i32(3, 33)), -3), (dict(table=i32(0, -1, 2, 9)), -3)):
        assert evict(**kw) == code, kw
    s = abi.DpufAmdSampling()
    assert eng.dpuf_amd_engine_forward_sample(h, 1, M.ptr(i32(1)), 0, None, 1, C.byref(s), M.ptr(tok), None, None) == -1
    assert eng.dpuf_amd_engine_forward_sample(h, 1, M.ptr(i32(1)), 0, None, 1, None, M.ptr(tok), None, None) == -1
    assert eng.dpuf_amd_engine_forward_slots_sample(h, 1, M.ptr(i32(0)), M.ptr(i32(1)), M.ptr(i32(0)), C.byref(some),
                                                    None, None, None) == -1
    eng.dpuf_engine_destroy(h)


def test_sampled_steps_do_not_exit_early(eng, monkeypatch):
    """The LM head's early exit vouches for the largest logit alone: with it on
    (and firing for the greedy call) a sampled step has the whole vocabulary's
    logits, and draws from them."""
    n = 40960
    shape = dict(hidden_size=256, intermediate_size=512, num_layers=2, num_q_heads=4, num_kv_heads=2, head_dim=64,
                 vocab_size=n, tie_word_embeddings=1)
    m = M.Model.build(shape, max_seq_len=32, seed=9)
    h = eng.dpuf_engine_create(*m.create_args())
    ids = np.random.default_rng(3).integers(0, n, 6).astype(np.int32)
    monkeypatch.delenv("DPUF_EARLY_TILES", raising=False)
    tok, lp, g = np.zeros(1, np.int32), np.zeros(1, np.float32), np.zeros(1, np.int32)
    full, lg, zone = np.zeros(n, np.float32), np.zeros(n, np.float32), np.zeros(n, np.float32)
    col = lambda v, t: np.array([v], t)
    beyond = 0
    for count, pos in ((6, 0), (1, 6), (1, 7)):
        monkeypatch.delenv("DPUF_EARLY_TILES", raising=False)
        assert eng.dpuf_amd_engine_forward_argmax(h, count, M.ptr(ids), pos, None, 1, M.ptr(g), M.ptr(full)) == 0
        monkeypatch.setenv("DPUF_EARLY_TILES", "300")
        monkeypatch.setenv("DPUF_EARLY_MARGIN", "1e-7")
        assert eng.dpuf_amd_engine_forward_argmax(h, count, M.ptr(ids), pos, None, 1, M.ptr(g), M.ptr(zone)) == 0
        assert np.all(zone[300 * 16:] == -1e9)
        exits = eng.dpuf_amd_engine_early_exit_count(h)
        for graph in (0, 1, 1):
            for u, t in ((0.1, 1.0), (0.6, 0.7), (0.95, 1.5), (0.5, 0.0)):
                a = dict(temperature=col(t, np.float32), top_k=col(0, np.int32), top_p=col(1.0, np.float32),
                         min_p=col(0.0, np.float32), u=col(u, np.float32))
                s = abi.DpufAmdSampling(**{k: v.ctypes.data for k, v in a.items()})
                lg[:] = 0
                assert eng.dpuf_amd_engine_forward_sample(h, count, M.ptr(ids), pos, None, graph, C.byref(s),
                                                          M.ptr(tok), M.ptr(lp), M.ptr(lg)) == 0
                assert np.array_equal(lg.view(np.uint32), full.view(np.uint32))
                want, wl = drawn(a, 0, full)
                assert tok[0] == want and abs(lp[0] - wl) <= abs(wl) * 2.0 ** -23 + n * 2.0 ** -38 + 2.0 ** -30
                beyond += int(tok[0]) >= 300 * 16
        assert eng.dpuf_amd_engine_early_exit_count(h) == exits
    assert beyond > 0
    eng.dpuf_engine_destroy(h)


def test_eviction_that_keeps_all(eng, hip):
    """keep far beyond every length: all rows move to the other pages, whatever
    sink and recent are, and the list of rows that stay is as long as the
    sequences, not as keep (20 x 2 x 2^30 entries would not fit the card)."""
    m, h = _engine(eng)
    n, page = 20, 1024
    assert eng.dpuf_amd_engine_pages_create(h, 2 * n, page, R.BF16) == 0
    rng = np.random.default_rng(11)
    rows = np.array([1 + i % 7 for i in range(n)], np.int32)
    table = np.arange(n, dtype=np.int32)[:, None].copy()
    ids, pos = rng.integers(0, V, rows.sum()).astype(np.int32), np.concatenate([np.arange(r) for r in rows]).astype(np.int32)
    lg = np.zeros((n, V), np.float32)
    assert eng.dpuf_amd_engine_forward_pages(h, n, M.ptr(rows), M.ptr(rows), M.ptr(table), 1, M.ptr(ids), M.ptr(pos), 1.0,
                                             None, M.ptr(lg), None, None) == 0
    stride = 1 << 20
    dst = np.full((n, stride), -1, np.int32)
    dst[:, 0] = n + rng.permutation(n)
    new = np.zeros(n, np.int32)
    say(f"keep {page * stride} of up to 7 rows")
    assert eng.dpuf_amd_engine_evict_pages(h, n, M.ptr(rows), M.ptr(table), 1, page * stride, 5, 9, M.ptr(dst), stride,
                                           M.ptr(new)) == 0, eng.dpuf_amd_last_error()
    assert np.array_equal(new, rows)
    for l in range(2):
        p = abi.DpufAmdPages()
        assert eng.dpuf_amd_engine_pages(h, l, C.byref(p)) == 0
        for at, width, t in ((p.k, 64, np.uint16), (p.v, 64, np.uint16), (p.w, 1, np.float32)):
            got = np.empty((2 * n, 2, page, width), t)
            assert hip.lib.hipMemcpy(M.ptr(got), at, got.nbytes, R.D2H) == 0
            for i in range(n):
                assert got[i, :, :rows[i]].any()
                assert np.array_equal(got[i, :, :rows[i]], got[dst[i, 0], :, :rows[i]])
    eng.dpuf_engine_destroy(h)
