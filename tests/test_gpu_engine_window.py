"""The engine's pass over pages with sliding windows, and its scores of every
new row: bit for bit against the parts put together by hand, and the scores
against float64 from those logits."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
import test_gpu_logprobs as LP
from dpuf_amd import abi
from dpuf_amd import model as M
from test_gpu_paged_engine import Parts, V, _engine

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip(eng):
    h = R.Hip()
    yield h
    h.free_all()


def say(*a):
    print(*a, flush=True)


class Windowed:
    """The library with windows in its paged attention, layer after layer."""

    def __init__(self, eng, windows, sink):
        self.eng, self.windows, self.sink, self.at = eng, windows, sink, 0

    def __getattr__(self, name):
        return getattr(self.eng, name)

    def dpuf_amd_paged_attn_workspace(self, b, p, nq):
        w = self.windows[self.at % len(self.windows)]
        if not w:
            return self.eng.dpuf_amd_paged_attn_workspace(b, p, nq)
        return self.eng.dpuf_amd_paged_attn_window_workspace(b, p, nq, w, self.sink)

    def dpuf_amd_paged_attn(self, b, p, nq, q, scale, *rest):
        w = self.windows[self.at % len(self.windows)]
        self.at += 1
        if not w:
            return self.eng.dpuf_amd_paged_attn(b, p, nq, q, scale, *rest)
        return self.eng.dpuf_amd_paged_attn_window(b, p, nq, q, scale, w, self.sink, *rest)


class AllRows(Parts):
    """... whose `rows` are the logits of every new row of the last pass."""

    def forward(self, *a):
        self.norms, self.mats = [], []
        last = super().forward(*a)
        h, res = self.norms[-2][0], self.mats[-2]
        self.rows = self.matmul(self.m.lm.contents, super().norm(h, res, self.m.out_norm)[1])
        return last

    def norm(self, *a):
        self.norms.append(super().norm(*a))
        return self.norms[-1]

    def matmul(self, *a):
        self.mats.append(super().matmul(*a))
        return self.mats[-1]


@pytest.mark.parametrize("nq,nkv,hd,page,t,windows,sink", [
    (4, 2, 64, 16, R.BF16, (20, 33), 4), (8, 1, 128, 32, R.F16, (0, 16), 0), (3, 3, 256, 16, R.BF16, (1, 50), 18),
    (4, 2, 64, 16, R.BF16, (0, 0), 3)])
def test_conversation(eng, orc, hip, nq, nkv, hd, page, t, windows, sink):
    """Prompts, chunks and single tokens in one pass; pages go back to the free
    list as soon as every layer's window has left them."""
    shape = dict(hidden_size=256, intermediate_size=512, num_layers=2, num_q_heads=nq, num_kv_heads=nkv, head_dim=hd,
                 vocab_size=V, tie_word_embeddings=1)
    m = M.Model.build(shape, max_seq_len=32, seed=77)
    h = eng.dpuf_engine_create(*m.create_args())
    assert h
    n_pages = 40
    assert eng.dpuf_amd_engine_pages_create(h, n_pages, page, t) == 0
    w = np.array(windows, np.int32)
    assert eng.dpuf_amd_engine_pages_window(h, M.ptr(w), sink) == 0
    parts = AllRows(Windowed(eng, windows, sink), orc, hip, m, n_pages, page, t)
    rng = np.random.default_rng(78)
    free = list(rng.permutation(n_pages))
    seqs = {}      # name -> [pages (-1: given back), cached rows]
    gone = 0

    def step(work, score=None):
        nonlocal gone
        for name, ids in work:
            s = seqs.setdefault(name, [[], 0])
            s[1] += len(ids)
            lo = s[1] - len(ids) - max(windows) + 1
            for j in range(len(s[0])):
                if all(windows) and (j + 1) * page <= lo and j * page >= sink and s[0][j] >= 0:
                    free.append(s[0][j])
                    s[0][j] = rng.choice([-1, n_pages, 2 ** 31 - 1])
                    gone += 1
            while len(s[0]) * page < s[1]:
                s[0].append(free.pop(0))
        width = max(len(seqs[name][0]) for name, _ in work) + 1
        table = np.full((len(work), width), -1, np.int32)
        rows = np.array([len(ids) for _, ids in work], np.int32)
        ctx = np.array([seqs[name][1] for name, _ in work], np.int32)
        for i, (name, _) in enumerate(work):
            table[i, :len(seqs[name][0])] = seqs[name][0]
        pos = np.concatenate([np.arange(c - r, c) for r, c in zip(rows, ctx)]).astype(np.int32)
        ids = np.concatenate([np.asarray(i, np.int32) for _, i in work])
        say(f"  pass: rows {rows.tolist()}, contexts {ctx.tolist()}, scored {score}")
        want = parts.forward(rows, ctx, table, ids, pos, -1.0)
        args = (h, len(work), M.ptr(rows), M.ptr(ctx), M.ptr(table), width, M.ptr(ids), M.ptr(pos))
        if score is None:
            lg = np.zeros((len(work), V), np.float32)
            rc = eng.dpuf_amd_engine_forward_pages(*args, -1.0, None, M.ptr(lg), None, None)
            assert rc == 0, (rc, eng.dpuf_amd_last_error())
            assert np.array_equal(lg.view(np.uint32), want.view(np.uint32)), np.abs(lg - want).max()
            return
        nt, k, ent = score
        n = int(rows.sum())
        tg = rng.integers(-1, V + 1, (n, nt)).astype(np.int32)
        lp, en = np.full((n, nt), 9.0, np.float32), np.full(n, 9.0, np.float32)
        top, tl = np.full((n, k), -9, np.int32), np.full((n, k), 9.0, np.float32)
        p = lambda a, on: M.ptr(a) if on else None
        rc = eng.dpuf_amd_engine_score_pages(*args, nt, p(tg, nt), k, p(lp, nt), p(en, ent), p(top, k), p(tl, k))
        assert rc == 0, (rc, eng.dpuf_amd_last_error())
        LP.check(parts.rows.astype(np.float64), tg, k, (lp, en, top, tl), ent)

    say(f"windows {windows}, sink {sink}: {nq}/{nkv} heads of {hd}, pages of {page}, type {t}")
    prompt = lambda n: rng.integers(0, V, n)
    step([("a", prompt(5)), ("b", prompt(37)), ("c", prompt(1))])
    step([("a", prompt(1)), ("b", prompt(70)), ("c", prompt(20))], (1, 5, True))
    step([("c", prompt(1)), ("a", prompt(1)), ("b", prompt(1))], (3, 0, False))
    step([("b", prompt(60)), ("a", prompt(55))])
    step([("b", prompt(1))], (0, 20, True))
    step([("a", prompt(90)), ("b", prompt(1)), ("c", prompt(33))], (2, 64, True))
    for _ in range(3):
        step([("b", prompt(1)), ("c", prompt(1)), ("a", prompt(1))])
    assert (gone > 0) == all(windows)
    eng.dpuf_engine_destroy(h)


def test_refusals(eng):
    m, h = _engine(eng)
    i32 = lambda *v: np.array(v, np.int32)
    f32 = lambda *s: np.zeros(s, np.float32)
    tg, lp, en, top, tl = i32(*range(6)), f32(3, 2), f32(3), np.zeros((3, 4), np.int32), f32(3, 4)
    base = dict(n=2, rows=i32(1, 2), ctx=i32(3, 17), table=i32(0, -1, 2, 5), stride=2, ids=i32(1, 2, 3),
                pos=i32(0, 1, 2), nt=2, tg=tg, k=4, lp=lp, en=en, top=top, tl=tl)
    p = lambda x: M.ptr(x) if x is not None else None

    def score(handle=h, **kw):
        d = dict(base, **kw)
        return eng.dpuf_amd_engine_score_pages(handle, d["n"], p(d["rows"]), p(d["ctx"]), p(d["table"]), d["stride"],
                                               p(d["ids"]), p(d["pos"]), d["nt"], p(d["tg"]), d["k"], p(d["lp"]),
                                               p(d["en"]), p(d["top"]), p(d["tl"]))

    def forward(decay, table=None, ctx=None, rows=None):
        t = base["table"] if table is None else table
        lg = f32(2, V)
        return eng.dpuf_amd_engine_forward_pages(h, 2, M.ptr(base["rows"] if rows is None else rows),
                                                 M.ptr(base["ctx"] if ctx is None else ctx), M.ptr(t), len(t) // 2,
                                                 M.ptr(base["ids"]), M.ptr(base["pos"]), decay, None, M.ptr(lg), None, None)

    assert score() == -1                                   # no pages yet
    assert eng.dpuf_amd_engine_pages_create(h, 8, 16, 1) == 0
    assert score() == 0 and score(None) == -1
    for kw, code in ((dict(rows=None), -1), (dict(tg=None), -1), (dict(lp=None), -1), (dict(nt=0), -1), (dict(k=0), -1),
                     (dict(top=None), -1), (dict(tl=None), -1),
                     (dict(nt=0, tg=None, lp=None, k=0, top=None, tl=None, en=None), -1),
                     (dict(nt=0, tg=None, lp=None, k=0, top=None, tl=None), 0), (dict(en=None), 0),
                     (dict(nt=1025), -2), (dict(k=65), -2), (dict(nt=-1, tg=None, lp=None), -2),
                     (dict(k=-1, top=None, tl=None), -2), (dict(n=0), -2), (dict(n=513), -2), (dict(rows=i32(1, 512)), -2),
                     (dict(ctx=i32(3, 33)), -3), (dict(table=i32(8, -1, 2, 5)), -3), (dict(pos=i32(0, -1, 2)), -3),
                     (dict(ids=i32(1, 2, V)), -4), (dict(table=i32(2, -1, 2, 5)), -1)):
        assert score(**kw) == code, kw
    window = lambda w, s: eng.dpuf_amd_engine_pages_window(h, p(w), s)
    assert eng.dpuf_amd_engine_pages_window(None, M.ptr(i32(1, 1)), 0) == -1
    for w, s, code in ((i32(1, -1), 0, -2), (i32(1, (1 << 30) + 1), 0, -2), (i32(1, 1), -1, -2),
                       (i32(1, 1), (1 << 30) + 1, -2)):
        assert window(w, s) == code
    # sequences of 3 and 50 rows; the second's first two pages are gone
    gone = i32(0, -1, -1, -1, -1, 9, 2, 5)
    ctx = i32(3, 50)
    assert forward(0.5) == 0 and forward(-1.0, gone, ctx) == -3
    assert window(i32(16, 0), 0) == 0 and forward(-1.0, gone, ctx) == -3 and forward(0.5) == -1 and forward(-1.0) == 0
    assert window(i32(16, 10), 0) == 0 and forward(-1.0, gone, ctx) == 0 and forward(0.5, gone, ctx) == -1
    assert window(i32(16, 18), 0) == 0 and forward(-1.0, gone, ctx) == -3     # rows 31 to 49 of pages 1 to 3
    assert window(i32(16, 17), 0) == 0 and forward(-1.0, gone, ctx) == 0
    assert window(i32(16, 10), 1) == 0 and forward(-1.0, gone, ctx) == -3     # the first page
    assert window(i32(0, 0), 1) == 0 and forward(0.5) == 0 and forward(-1.0, gone, ctx) == -3
    assert window(i32(5, 5), 0) == 0 and window(None, 0) == 0 and forward(-1.0, gone, ctx) == -3 and forward(0.5) == 0
    eng.dpuf_engine_destroy(h)


def test_scores_of_a_full_call(eng):
    """512 rows at once, then one: the sums of a prompt's log probabilities are
    those of its tokens one at a time (but for the cache's rounding)."""
    m, h = _engine(eng)
    assert eng.dpuf_amd_engine_pages_create(h, 70, 16, R.BF16) == 0
    rng = np.random.default_rng(3)
    ids = rng.integers(0, V, 513).astype(np.int32)
    table = rng.permutation(70)[None, :33].astype(np.int32)
    one = lambda v: np.array([v], np.int32)

    def score(at, n):
        lp, en = np.zeros((n, 1), np.float32), np.zeros(n, np.float32)
        pos = np.arange(at, at + n, dtype=np.int32)
        nxt = np.append(ids, 0)[at + 1:at + n + 1].astype(np.int32)
        assert eng.dpuf_amd_engine_score_pages(h, 1, M.ptr(one(n)), M.ptr(one(at + n)), M.ptr(table), 33,
                                               M.ptr(ids[at:at + n].copy()), M.ptr(pos), 1, M.ptr(nxt), 0, M.ptr(lp),
                                               M.ptr(en), None, None) == 0, eng.dpuf_amd_last_error()
        return lp[:, 0], en

    say("512 rows")
    lp, en = score(0, 512)
    assert np.all(lp < 0) and np.all((en > 0) & (en <= np.log(V) + 1e-4))
    for at in (511, 200, 0):
        one_lp, one_en = score(at, 1)
        assert abs(one_lp[0] - lp[at]) < 0.1 and abs(one_en[0] - en[at]) < 0.1
    eng.dpuf_engine_destroy(h)


def test_entries_of_pages_given_back_stay(eng, orc, hip):
    """A conversation without end on a few pages: each page that both windows
    have left is taken again for the next rows, and the table's old entries
    still name it."""
    page, windows, sink, n_pages = 16, (20, 33), 4, 7
    shape = dict(hidden_size=256, intermediate_size=512, num_layers=2, num_q_heads=4, num_kv_heads=2, head_dim=64,
                 vocab_size=V, tie_word_embeddings=1)
    m = M.Model.build(shape, max_seq_len=32, seed=79)
    h = eng.dpuf_engine_create(*m.create_args())
    assert h
    assert eng.dpuf_amd_engine_pages_create(h, n_pages, page, R.BF16) == 0
    assert eng.dpuf_amd_engine_pages_window(h, M.ptr(np.array(windows, np.int32)), sink) == 0
    parts = Parts(Windowed(eng, windows, sink), orc, hip, m, n_pages, page, R.BF16)
    rng = np.random.default_rng(80)
    free, held, ctx, again = list(range(n_pages)), [], 0, 0
    for rows in [30] + [20, 1, 1, 14, 1, 25] * 3:
        ctx += rows
        lo = ctx - rows - max(windows) + 1
        for j, (pg, there) in enumerate(held):
            if there and (j + 1) * page <= lo and j * page >= sink:
                free.append(pg)
                held[j] = (pg, False)
        while len(held) * page < ctx:
            pg = free.pop(0)
            again += any(pg == old for old, _ in held)
            held.append((pg, True))
        stale = np.array([[pg for pg, _ in held]], np.int32)
        clean = np.array([[pg if there else -1 for pg, there in held]], np.int32)
        pos, ids = np.arange(ctx - rows, ctx, dtype=np.int32), rng.integers(0, V, rows).astype(np.int32)
        one = lambda v: np.array([v], np.int32)
        say(f"  {rows} rows, {ctx} cached, {again} pages taken again")
        want = parts.forward(one(rows), one(ctx), clean, ids, pos, -1.0)
        lg = np.zeros((1, V), np.float32)
        rc = eng.dpuf_amd_engine_forward_pages(h, 1, M.ptr(one(rows)), M.ptr(one(ctx)), M.ptr(stale), stale.shape[1],
                                               M.ptr(ids), M.ptr(pos), -1.0, None, M.ptr(lg), None, None)
        assert rc == 0, (rc, eng.dpuf_amd_last_error())
        assert np.array_equal(lg.view(np.uint32), want.view(np.uint32)), np.abs(lg - want).max()
    assert again > 5
    eng.dpuf_engine_destroy(h)


def test_every_row_of_a_full_call(eng, orc, hip):
    """512 scored rows in three sequences: targets, entropies and alternatives
    against float64 from the logits of the parts put together."""
    m, h = _engine(eng)
    page, n_pages = 16, 40
    assert eng.dpuf_amd_engine_pages_create(h, n_pages, page, R.BF16) == 0
    parts = AllRows(eng, orc, hip, m, n_pages, page, R.BF16)
    rng = np.random.default_rng(81)
    rows = ctx = np.array([300, 1, 211], np.int32)
    table, order = np.full((3, 19), -1, np.int32), list(rng.permutation(n_pages))
    for i, c in enumerate(ctx):
        for j in range(-(-int(c) // page)):
            table[i, j] = order.pop()
    pos = np.concatenate([np.arange(c) for c in ctx]).astype(np.int32)
    ids = rng.integers(0, V, 512).astype(np.int32)
    say("512 rows of three sequences")
    parts.forward(rows, ctx, table, ids, pos, -1.0)
    tg = rng.integers(0, V, (512, 3)).astype(np.int32)
    lp, en = np.zeros((512, 3), np.float32), np.zeros(512, np.float32)
    top, tl = np.zeros((512, 5), np.int32), np.zeros((512, 5), np.float32)
    rc = eng.dpuf_amd_engine_score_pages(h, 3, M.ptr(rows), M.ptr(ctx), M.ptr(table), 19, M.ptr(ids), M.ptr(pos), 3,
                                         M.ptr(tg), 5, M.ptr(lp), M.ptr(en), M.ptr(top), M.ptr(tl))
    assert rc == 0, (rc, eng.dpuf_amd_last_error())
    LP.check(parts.rows.astype(np.float64), tg, 5, (lp, en, top, tl))
    eng.dpuf_engine_destroy(h)
