"""The paged-serving entry points' checks of their arguments (no GPU needed:
every refusal comes before anything is launched), and the rotation table."""
import ctypes as C
import math

import numpy as np
import pytest

from dpuf_amd import abi


@pytest.fixture(scope="module")
def lib():
    return abi.load_engine()


A = 0x7F0000000000       # an aligned address that is no memory: nothing here may read it


def pages(**over):
    d = dict(type=1, n_pages=8, page_size=16, n_kv_heads=2, head_dim=64, page_stride=2 * 16 * 64, head_stride=16 * 64,
             row_stride=64, k=A, v=A + (1 << 20), w=A + (2 << 20))
    d.update(over)
    return abi.DpufAmdPages(**d)


def batch(**over):
    d = dict(n_seqs=2, n_rows=3, table_stride=4, max_ctx=40, row_start=A + (3 << 20), ctx_len=A + (4 << 20),
             page_table=A + (5 << 20))
    d.update(over)
    return abi.DpufAmdBatch(**d)


Q, OUT, LSE, WS = A + (6 << 20), A + (7 << 20), A + (8 << 20), A + (9 << 20)


def attn(lib, b=None, p=None, nq=4, q=Q, scale=0.1, out_t=1, out=OUT, lse=LSE, ws=WS, n=1 << 30):
    b, p = b if b is not None else batch(), p if p is not None else pages()
    return lib.dpuf_amd_paged_attn(C.byref(b), C.byref(p), nq, q, scale, out_t, out, lse, ws, n, None)


BAD_PAGES = [(dict(type=0), -5), (dict(type=3), -5), (dict(head_dim=96), -5), (dict(head_dim=0), -5),
             (dict(n_pages=0), -2), (dict(n_kv_heads=0), -2), (dict(n_kv_heads=1025), -2), (dict(page_size=8), -2),
             (dict(page_size=48), -2), (dict(page_size=2048), -2), (dict(page_stride=2 * 16 * 64 + 4), -4),
             (dict(row_stride=56), -4), (dict(head_stride=0), -4), (dict(row_stride=-64), -4), (dict(k=None), -1),
             (dict(v=A + 8), -1)]
BAD_BATCH = [(dict(n_seqs=0), -2), (dict(n_seqs=16385), -2), (dict(n_rows=-1), -2), (dict(n_rows=65537), -2),
             (dict(table_stride=0), -2), (dict(table_stride=(1 << 26) + 1), -2), (dict(row_start=None), -1),
             (dict(ctx_len=A + 2), -1), (dict(page_table=None), -1)]


@pytest.mark.parametrize("over,code", BAD_PAGES)
def test_pages_refused(lib, over, code):
    assert attn(lib, p=pages(**over)) == code
    assert lib.dpuf_amd_paged_attn_workspace(C.byref(batch()), C.byref(pages(**over)), 4) == 0


@pytest.mark.parametrize("over,code", BAD_BATCH)
def test_batch_refused(lib, over, code):
    assert attn(lib, b=batch(**over)) == code


@pytest.mark.parametrize("kw,code", [(dict(nq=0), -2), (dict(nq=3), -2), (dict(nq=66), -2), (dict(q=None), -1),
                                     (dict(q=Q + 8), -1), (dict(out=None), -1), (dict(out=Q + 512), -1),
                                     (dict(scale=0.0), -2), (dict(scale=-1.0), -2), (dict(scale=math.nan), -2),
                                     (dict(scale=math.inf), -2), (dict(out_t=2), -5), (dict(out_t=7), -5),
                                     (dict(lse=LSE + 1), -1)])
def test_attention_refused(lib, kw, code):
    assert attn(lib, **kw) == code


def test_attention_workspace(lib):
    b, p = batch(max_ctx=5000, table_stride=400), pages()
    need = lib.dpuf_amd_paged_attn_workspace(C.byref(b), C.byref(p), 4)
    assert need > 0
    assert attn(lib, b=b, n=need - 1) == -7
    assert attn(lib, b=b, ws=None) == -1
    assert attn(lib, b=b, ws=WS + 4) == -1
    assert attn(lib, b=b, n=need) == -1          # everything in order but the memory
    assert attn(lib, b=batch(n_rows=0)) == 0     # nothing to do
    # the workspace is bounded by the rows that are split, not by sequences times rows
    big = batch(n_seqs=16384, n_rows=65536, table_stride=1 << 16, max_ctx=1 << 20)
    assert lib.dpuf_amd_paged_attn_workspace(C.byref(big), C.byref(pages(n_kv_heads=8)), 32) < 1 << 30


@pytest.mark.parametrize("kw,code", [(dict(w=None), -1), (dict(decay=math.nan), -2), (dict(decay=math.inf), -2),
                                     (dict(scale=0.0), -2), (dict(nq=5), -2), (dict(q=None), -1), (dict(lse=None), -1),
                                     (dict(w_in=A + (2 << 20) + 64), -1)])
def test_weights_refused(lib, kw, code):
    d = dict(w=A + (2 << 20), decay=1.0, scale=0.1, nq=4, q=Q, lse=LSE, w_in=None)
    d.update(kw)
    assert lib.dpuf_amd_paged_attn_weights(C.byref(batch()), C.byref(pages(w=d["w"])), d["nq"], d["q"], d["scale"],
                                           d["lse"], d["decay"], d["w_in"], None) == code


@pytest.mark.parametrize("kw,code", [(dict(keep=0), -2), (dict(sink=-1), -2), (dict(recent=-1), -2),
                                     (dict(sink=5, recent=4), -2), (dict(keep=65), -2), (dict(stride=0), -2),
                                     (dict(stride=1 << 27), -2), (dict(table=None), -1), (dict(kept=None), -1),
                                     (dict(new_len=None), -1), (dict(new_len=A + (4 << 20)), -1),
                                     (dict(new_len=A + (4 << 20) + 4), -1), (dict(kept=A + (5 << 20)), -1),
                                     (dict(kept=LSE, new_len=LSE + 16), -1), (dict(dst=dict(type=2)), -5),
                                     (dict(dst=dict(head_dim=128, row_stride=128)), -5),
                                     (dict(dst=dict(n_kv_heads=4)), -2), (dict(dst=dict(w=None)), -1),
                                     (dict(src=dict(w=None)), -1), (dict(dst=dict(row_stride=60)), -4)])
def test_eviction_refused(lib, kw, code):
    d = dict(keep=8, sink=2, recent=3, dst={}, src={}, table=Q, stride=4, kept=OUT, new_len=LSE)
    d.update(kw)
    src, dst = pages(**d["src"]), pages(**d["dst"])
    assert lib.dpuf_amd_paged_evict(C.byref(batch()), C.byref(src), d["keep"], d["sink"], d["recent"], C.byref(dst),
                                    d["table"], d["stride"], d["kept"], d["new_len"], None) == code


@pytest.mark.parametrize("kw,code", [(dict(in_t=3), -5), (dict(rope=None), -1), (dict(rot=0), -2), (dict(rot=63), -2),
                                     (dict(rot=66), -2), (dict(rscale=math.nan), -2), (dict(turns=None), -1),
                                     (dict(turns=A + 4), -1), (dict(nq=-1), -2), (dict(nq=65), -2), (dict(q=None), -1),
                                     (dict(q_out=None), -1), (dict(nq=0), -1), (dict(pos=None), -1), (dict(k=None), -1),
                                     (dict(k=A + 2), -1), (dict(qs=248), -4), (dict(ks=132), -4), (dict(vs=120), -4),
                                     (dict(eps=-1.0), -2), (dict(eps=math.nan), -2), (dict(q_out=Q + 256), -1),
                                     (dict(q_out=Q, in_t=0), -1), (dict(q_out=Q, in_t=1, qs=264), -1),
                                     (dict(q_out=OUT, k=OUT + 16), -1)])
def test_rope_refused(lib, kw, code):
    d = dict(in_t=0, rope=1, rot=64, rscale=1.0, turns=A, nq=4, q=Q, q_out=OUT, pos=LSE, k=WS, v=WS + 4096, qs=256,
             ks=128, vs=128, eps=1e-6)
    d.update(kw)
    rope = abi.DpufAmdRope(turns=d["turns"], rot_dim=d["rot"], interleaved=0, scale=d["rscale"])
    assert lib.dpuf_amd_rope_append(C.byref(batch()), C.byref(pages()), C.byref(rope) if d["rope"] else None, d["pos"],
                                    d["in_t"], d["nq"], d["q"], d["k"], d["v"], d["qs"], d["ks"], d["vs"], Q + 4, Q + 8,
                                    d["eps"], d["q_out"], None) == code


@pytest.mark.parametrize("kw,code", [(dict(t=3), -5), (dict(n=0), -2), (dict(n=65537), -2), (dict(V=0), -2),
                                     (dict(V=(1 << 24) + 1), -2), (dict(stride=99), -4), (dict(x=None), -1),
                                     (dict(x=A + 2), -1), (dict(u=None), -1), (dict(tok=None), -1), (dict(temp=A + 1), -1),
                                     (dict(tok=A + 64), -1), (dict(logp=OUT + 4), -1), (dict(tok=LSE + 4), -1)])
def test_sampling_refused(lib, kw, code):
    d = dict(t=0, n=3, V=100, stride=100, x=A, temp=None, u=LSE, tok=OUT, logp=None)
    d.update(kw)
    n = lib.dpuf_amd_sample_workspace(max(1, d["n"]), max(1, min(d["V"], 1 << 24)))
    assert lib.dpuf_amd_sample(d["t"], d["n"], d["V"], d["stride"], d["x"], d["temp"], None, None, None, d["u"],
                               d["tok"], d["logp"], WS, n, None) == code


def spec(**kw):
    d = dict(rot_dim=64, theta=10000.0, scaling=0, factor=1.0, low_freq=1.0, high_freq=4.0, beta_fast=32.0,
             beta_slow=1.0, orig_max_pos=8192)
    d.update(kw)
    return abi.DpufAmdRopeSpec(**d)


def turns(lib, **kw):
    s = spec(**kw)
    out, scale = np.zeros(128), C.c_float(0)
    rc = lib.dpuf_amd_rope_turns(C.byref(s), out.ctypes.data_as(C.c_void_p), C.byref(scale))
    return rc, out, scale.value


def test_rope_table(lib):
    base = np.array([10000.0 ** (-2 * j / 64) for j in range(32)]) / (2 * math.pi)
    rc, t, m = turns(lib)
    assert rc == 0 and m == 1.0 and np.allclose(t[:32], base, rtol=1e-14) and np.all(t[32:] == 0)
    assert np.allclose(turns(lib, scaling=1, factor=4.0)[1][:32], base / 4, rtol=1e-14)
    # llama3: pairs of more than 4 turns over 8 192 positions stay, of less than 1 are divided, linear in between
    t = turns(lib, scaling=2, factor=8.0)[1][:32]
    n = 8192 * base
    assert np.allclose(t[n >= 4], base[n >= 4], rtol=1e-14) and np.allclose(t[n <= 1], base[n <= 1] / 8, rtol=1e-14)
    mid = (n > 1) & (n < 4)
    s = (n[mid] - 1) / 3
    assert mid.any() and np.allclose(t[mid], (1 - s) * base[mid] / 8 + s * base[mid], rtol=1e-13)
    # yarn: as is up to the pair of 32 turns, divided past the pair of one turn
    rc, t, m = turns(lib, scaling=3, factor=4.0)
    assert rc == 0 and abs(m - (0.1 * math.log(4.0) + 1)) < 1e-7
    where = lambda b: 64 * math.log(8192 / (b * 2 * math.pi)) / (2 * math.log(10000.0))
    lo, hi = math.floor(where(32.0)), math.ceil(where(1.0))
    ramp = np.clip((np.arange(32) - lo) / (hi - lo), 0, 1)
    assert 0 < lo < hi < 32 and np.allclose(t[:32], base / 4 * ramp + base * (1 - ramp), rtol=1e-13)
    assert turns(lib, scaling=3, factor=1.0)[2] == 1.0


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=258), dict(theta=1.0),
                                dict(theta=math.inf), dict(scaling=4), dict(scaling=-1), dict(scaling=1, factor=0.5),
                                dict(scaling=1, factor=math.nan), dict(scaling=2, orig_max_pos=0),
                                dict(scaling=2, low_freq=4.0), dict(scaling=3, beta_slow=0.0),
                                dict(scaling=3, beta_fast=1.0)])
def test_rope_table_refused(lib, kw):
    assert turns(lib, **kw)[0] == -2


def test_null_descriptors(lib):
    assert lib.dpuf_amd_rope_turns(None, A, C.byref(C.c_float())) == -1
    assert lib.dpuf_amd_paged_attn(None, C.byref(pages()), 4, Q, 0.1, 1, OUT, LSE, WS, 0, None) == -1
    assert lib.dpuf_amd_paged_attn(C.byref(batch()), None, 4, Q, 0.1, 1, OUT, LSE, WS, 0, None) == -1


def test_structure_sizes():
    assert C.sizeof(abi.DpufAmdPages) == 72 and C.sizeof(abi.DpufAmdBatch) == 40
    assert C.sizeof(abi.DpufAmdRopeSpec) == 36 and C.sizeof(abi.DpufAmdRope) == 24


def test_workspaces_are_those_of_the_arguments(lib):
    """A workspace of the size given for a call's own arguments is enough, one
    byte less is not, and a smaller call may need a larger one."""
    V, sizes = 151936, []
    for n in (1, 2, 7, 56, 57, 1024, 5000):
        need = lib.dpuf_amd_sample_workspace(n, V)
        run = lambda size: lib.dpuf_amd_sample(0, n, V, V, A, None, None, None, None, LSE + (1 << 40), OUT + (1 << 41), None,
                                               WS + (1 << 42), size, None)
        assert run(need - 1) == -7 and run(need) == -1      # -1: no device memory
        sizes.append(need)
    assert sizes[3] > sizes[4]
    p, nq, sizes = pages(n_kv_heads=8, page_stride=8 * 16 * 64), 32, []
    for seqs, rows, ctx in ((1, 1, 4096), (1, 512, 4096), (4, 512, 4096), (64, 64, 4096), (512, 512, 4096),
                            (2048, 2048, 4096)):
        b = batch(n_seqs=seqs, n_rows=rows, table_stride=1 << 10, max_ctx=ctx)
        need = lib.dpuf_amd_paged_attn_workspace(C.byref(b), C.byref(p), nq)
        if need:
            assert attn(lib, b=b, p=p, nq=nq, n=need - 1) == -7
        assert attn(lib, b=b, p=p, nq=nq, n=need) == -1
        sizes.append(need)
    assert max(sizes[:-1]) > sizes[-1]
