"""The refusals of windowed attention, RoPE of several axes and log
probabilities (no GPU needed: every refusal comes before anything is launched),
and their workspaces."""
import ctypes as C
import math

import pytest

from dpuf_amd import abi
from test_cpu_paged import A, BAD_BATCH, BAD_PAGES, LSE, OUT, Q, WS, batch, pages


@pytest.fixture(scope="module")
def lib():
    return abi.load_engine()


def window(lib, b=None, p=None, nq=4, q=Q, scale=0.1, win=20, sink=4, out_t=1, out=OUT, lse=LSE, ws=WS, n=1 << 30):
    b, p = b if b is not None else batch(), p if p is not None else pages()
    return lib.dpuf_amd_paged_attn_window(C.byref(b), C.byref(p), nq, q, scale, win, sink, out_t, out, lse, ws, n, None)


@pytest.mark.parametrize("over,code", BAD_PAGES)
def test_window_pages_refused(lib, over, code):
    assert window(lib, p=pages(**over)) == code
    assert lib.dpuf_amd_paged_attn_window_workspace(C.byref(batch()), C.byref(pages(**over)), 4, 20, 4) == 0


@pytest.mark.parametrize("over,code", BAD_BATCH)
def test_window_batch_refused(lib, over, code):
    assert window(lib, b=batch(**over)) == code


@pytest.mark.parametrize("kw,code", [(dict(win=0), -2), (dict(win=-1), -2), (dict(win=(1 << 30) + 1), -2),
                                     (dict(sink=-1), -2), (dict(sink=(1 << 30) + 1), -2), (dict(nq=0), -2),
                                     (dict(nq=3), -2), (dict(nq=66), -2), (dict(q=None), -1), (dict(q=Q + 8), -1),
                                     (dict(out=None), -1), (dict(out=Q + 512), -1), (dict(scale=0.0), -2),
                                     (dict(scale=math.nan), -2), (dict(out_t=2), -5), (dict(lse=LSE + 1), -1),
                                     (dict(lse=OUT + 16), -1), (dict(win=1 << 30, sink=1 << 30), -1)])
def test_window_refused(lib, kw, code):
    """The last of them is in order but for the memory."""
    assert window(lib, **kw) == code


def test_window_workspace(lib):
    b, p = batch(max_ctx=50000, table_stride=4000), pages()
    need = lambda w, s, b=b: lib.dpuf_amd_paged_attn_window_workspace(C.byref(b), C.byref(p), 4, w, s)
    assert need(0, 0) == 0 and need(5, -1) == 0
    n = need(5000, 4)
    assert n > 0 and window(lib, b=b, win=5000, n=n - 1) == -7 and window(lib, b=b, win=5000, n=n) == -1
    assert window(lib, b=b, win=5000, ws=None) == -1 and window(lib, b=b, win=5000, ws=WS + 4) == -1
    # what a window leaves is split as such, and one that reaches everything as a call without
    assert need(100, 0) < n <= need(1 << 30, 0)
    assert need(1 << 30, 0) == need(1 << 30, 1 << 30) == need(7, 1 << 30)
    assert need(1 << 30, 0) == lib.dpuf_amd_paged_attn_workspace(C.byref(b), C.byref(p), 4)
    assert window(lib, b=batch(n_rows=0)) == 0
    for over in (dict(n_seqs=16384, n_rows=65536, table_stride=1 << 16, max_ctx=1 << 20),):
        big = batch(**over)
        for w in (1, 4096, 1 << 30):
            assert lib.dpuf_amd_paged_attn_window_workspace(C.byref(big), C.byref(pages(n_kv_heads=8)), 32, w, 4) < 1 << 30


def axes(lib, n_axes=3, sections=(12, 10, 10), in_turn=1, x=1, pos=LSE, pos_stride=3, **kw):
    d = dict(in_t=0, rope=1, rot=64, turns=A, nq=4, q=Q, q_out=OUT, k=WS, v=WS + 4096, qs=256, ks=128, vs=128, eps=1e-6,
             b=batch(), p=pages())
    d.update(kw)
    rope = abi.DpufAmdRope(turns=d["turns"], rot_dim=d["rot"], interleaved=0, scale=1.0)
    ax = abi.DpufAmdRopeAxes(n_axes=n_axes, sections=(C.c_int32 * 4)(*sections), in_turn=in_turn)
    return lib.dpuf_amd_rope_append_axes(C.byref(d["b"]), C.byref(d["p"]), C.byref(rope) if d["rope"] else None,
                                         C.byref(ax) if x else None, pos, pos_stride, d["in_t"], d["nq"], d["q"], d["k"],
                                         d["v"], d["qs"], d["ks"], d["vs"], Q + 4, Q + 8, d["eps"], d["q_out"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(x=0), -1), (dict(rope=0), -1), (dict(n_axes=0), -2), (dict(n_axes=5), -2), (dict(sections=(13, 10, 10)), -2),
    (dict(sections=(12, 10, 9)), -2), (dict(sections=(42, -10, 0)), -2), (dict(sections=(11, 11, 10)), -1), (dict(sections=(10, 11, 11)), -2),
    (dict(sections=(9, 11, 12)), -2), (dict(sections=(9, 11, 12), in_turn=0), -1), (dict(sections=(12, 10, 10, 99)), -1),
    (dict(n_axes=4, sections=(8, 8, 8, 8)), -1), (dict(n_axes=4, sections=(7, 8, 8, 9)), -2),
    (dict(n_axes=2, sections=(15, 17)), -2), (dict(n_axes=1, sections=(32,), pos_stride=0), -1),
    (dict(sections=(0x7fffffff, 0x7fffffff, 34), in_turn=0), -2), (dict(pos_stride=2), -4), (dict(pos_stride=-5), -4),
    (dict(pos=None), -1), (dict(pos=LSE + 2), -1), (dict(rot=62), -2), (dict(rot=66), -2), (dict(in_t=3), -5),
    (dict(qs=248), -4), (dict(eps=-1.0), -2), (dict(nq=65), -2), (dict(q_out=None), -1),
    # the positions of the last axis reach into an output
    (dict(pos=OUT - 4 * 70, pos_stride=35), -1), (dict(b=batch(n_rows=0)), 0)])
def test_axes_refused(lib, kw, code):
    """-1 of those in order: the memory."""
    assert axes(lib, **kw) == code


@pytest.mark.parametrize("over,code", BAD_PAGES)
def test_axes_pages_refused(lib, over, code):
    assert axes(lib, p=pages(**over)) == code


def logprobs(lib, t=0, n=3, V=20000, stride=20000, x=A, nt=2, tg=Q, k=5, lp=OUT, en=LSE, top=OUT + 4096, tl=OUT + 8192, ws=WS,
             size=None):
    if size is None:
        size = lib.dpuf_amd_logprobs_workspace(max(1, min(n, 65536)), max(1, min(V, 1 << 24)), max(0, min(k, 64)))
    return lib.dpuf_amd_logprobs(t, n, V, stride, x, nt, tg, k, lp, en, top, tl, ws, size, None)


@pytest.mark.parametrize("kw,code", [
    (dict(t=3), -5), (dict(t=-1), -5), (dict(n=0), -2), (dict(n=65537), -2), (dict(V=0), -2), (dict(V=(1 << 24) + 1), -2),
    (dict(nt=-1), -2), (dict(nt=1025), -2), (dict(k=-1), -2), (dict(k=65), -2), (dict(stride=19999), -4), (dict(x=None), -1),
    (dict(x=A + 2), -1), (dict(t=1, x=A + 1), -1), (dict(tg=None), -1), (dict(lp=None), -1), (dict(nt=0), -1),
    (dict(nt=0, tg=None), -1), (dict(k=0), -1), (dict(top=None), -1), (dict(tl=None), -1),
    (dict(nt=0, tg=None, lp=None, k=0, top=None, tl=None, en=None), -1), (dict(tg=Q + 2), -1), (dict(en=LSE + 1), -1),
    (dict(lp=A + 400), -1), (dict(en=Q + 4), -1), (dict(en=OUT + 4), -1), (dict(tl=OUT + 4096 + 4), -1),
    (dict(ws=None), -1), (dict(ws=WS + 8), -1), (dict(n=1, ws=WS + 8), -1), (dict(ws=OUT), -1), (dict(size=0), -7),
    (dict(), -1)])
def test_logprobs_refused(lib, kw, code):
    """The last of them is in order but for the memory."""
    assert logprobs(lib, **kw) == code


def test_logprobs_workspace(lib):
    size = lib.dpuf_amd_logprobs_workspace
    assert size(0, 9, 0) == size(1, 0, 0) == size(1, 9, 65) == size(1, 9, -1) == size(65537, 9, 1) == 0
    for n, V, k in ((1, 1, 0), (1, 151936, 20), (512, 151936, 0), (2048, 151936, 20), (7, 1 << 24, 64), (65536, 5, 2)):
        need = size(n, V, k)
        over = dict(n=n, V=V, stride=V, k=k, **({} if k else dict(top=None, tl=None)))
        assert logprobs(lib, size=need, **over) == -1
        assert need == 0 or (logprobs(lib, size=need - 1, **over) == -7 and logprobs(lib, ws=None, **over) == -1)
        assert need <= n * V // 8 + 32 * (n + 4096)       # a fraction of the logits


def test_structure_size():
    assert C.sizeof(abi.DpufAmdRopeAxes) == 24


@pytest.mark.parametrize("n_seqs,n_rows", [(1, 1), (1, 40), (1, 512), (9, 9), (9, 270), (48, 48)])
def test_workspaces_of_whole_windows_do_not_depend_on_the_table(lib, n_seqs, n_rows):
    """Windows and first tokens as long as the longest context: the same need
    where the table holds fewer rows than those, as many or more."""
    p = pages()
    for ctx in (100, 1000, 5000, 16384):
        for w, s in ((2 * ctx, 0), (2 * ctx, 4), (3, 2 * ctx), (1 << 30, 1 << 30)):
            got = set()
            for rows in (ctx, 2 * ctx - 16, 2 * ctx, 2 * ctx + 16, 1 << 20):
                b = batch(n_seqs=n_seqs, n_rows=n_rows, max_ctx=ctx, table_stride=-(-rows // p.page_size))
                got.add(lib.dpuf_amd_paged_attn_window_workspace(C.byref(b), C.byref(p), 32, w, s))
            assert len(got) == 1, (ctx, w, s, got)
