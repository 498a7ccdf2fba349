"""The operators of a step one after the other on one stream, as a serving
program has them: RoPE of three axes with the append, attention over the pages
with a window, and the scores of what comes out.  Two such steps (prompts'
chunks, single tokens) are captured into graphs that share a workspace, and
replayed in turn over new values with eager steps between."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
import test_gpu_logprobs as LP
import test_gpu_paged_window as PW
from dpuf_amd import abi
from test_gpu_rope_axes import axes_of, axis_of, rotate

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip(eng):
    h = R.Hip()
    yield h
    h.free_all()


def say(*a):
    print(*a, flush=True)


class Step:
    """One batch's calls, its inputs and outputs on the device."""

    def __init__(self, eng, hip, cache, rng, nq, window, sink, sections):
        self.eng, self.cache, self.rng, self.nq, self.window, self.sink = eng, cache, rng, nq, window, sink
        self.sections, hd, n = sections, cache.hd, cache.n_rows
        self.width = (nq + 2 * cache.nkv) * hd
        self.turns = np.array([1e4 ** (-2 * j / hd) / (2 * np.pi) for j in range(hd // 2)])
        z = lambda *s: hip.put(np.zeros(s, np.float32))
        self.qkv, self.pos = z(n, self.width), hip.put(np.zeros((3, n), np.int32))
        self.q, self.out, self.lse = hip.put(np.zeros((n, nq, hd), np.uint16)), z(n, nq, hd), z(n, nq)
        self.targets, self.logp, self.entropy = hip.put(np.zeros((n, 2), np.int32)), z(n, 2), z(n)
        self.top, self.top_logp = hip.put(np.zeros((n, 5), np.int32)), z(n, 5)
        self.d_turns = hip.put(self.turns)
        self.rope = abi.DpufAmdRope(turns=self.d_turns.p, rot_dim=hd, interleaved=0, scale=1.0)
        self.axes, self.b, self.p = axes_of(sections, 1), cache.batch(), cache.pages(w=False)

    def workspace(self):
        a = self.eng.dpuf_amd_paged_attn_window_workspace(C.byref(self.b), C.byref(self.p), self.nq, self.window, self.sink)
        return max(int(a), int(self.eng.dpuf_amd_logprobs_workspace(self.cache.n_rows, self.nq * self.cache.hd, 5)), 16)

    def new_inputs(self):
        n, V = self.cache.n_rows, self.nq * self.cache.hd
        self.qkv.set(self.rng.standard_normal((n, self.width)).astype(np.float32))
        self.pos.set(self.rng.integers(0, 5000, (3, n)).astype(np.int32))
        self.targets.set(self.rng.integers(0, V, (n, 2)).astype(np.int32))

    def enqueue(self, ws, size, s):
        e, c, nq, hd = self.eng, self.cache, self.nq, self.cache.hd
        n, at = c.n_rows, self.qkv.p
        assert e.dpuf_amd_rope_append_axes(C.byref(self.b), C.byref(self.p), C.byref(self.rope), C.byref(self.axes),
                                           self.pos.p, n, R.F32, nq, at, at + nq * hd * 4, at + (nq + c.nkv) * hd * 4,
                                           self.width, self.width, self.width, None, None, 0.0, self.q.p, s) == 0
        assert e.dpuf_amd_paged_attn_window(C.byref(self.b), C.byref(self.p), nq, self.q.p, 0.125, self.window, self.sink,
                                            R.F32, self.out.p, self.lse.p, ws.p, size, s) == 0
        assert e.dpuf_amd_logprobs(R.F32, n, nq * hd, nq * hd, self.out.p, 2, self.targets.p, 5, self.logp.p,
                                   self.entropy.p, self.top.p, self.top_logp.p, ws.p, size, s) == 0

    def results(self):
        return [d.get() for d in (self.q, self.out, self.lse, self.logp, self.entropy, self.top, self.top_logp,
                                  self.cache.dk, self.cache.dv)]

    def check(self, got):
        q, out, lse, logp, entropy, top, top_logp, k, v = got
        c, hd, n = self.cache, self.cache.hd, self.cache.n_rows
        x = self.qkv.get().astype(np.float64)
        by_pair = self.pos.get()[axis_of(hd // 2, self.sections, True)].T
        heads = x[:, :(self.nq + c.nkv) * hd].reshape(n, -1, hd)
        want, size = rotate(heads, by_pair, self.turns, hd, 0, 1.0)
        near = lambda a, b, z: np.all(np.abs(R.from_type(a, c.t) - b) <= R.HALF_STEP[c.t] * np.abs(b) * 1.01 +
                                      2.0 ** -20 * z + 2.0 ** -24)
        assert near(q, want[:, :self.nq], size[:, :self.nq])
        c.k, c.v = k, v
        for s, (r, ctx) in enumerate(zip(c.rows, c.ctx)):
            for i in range(r):
                pg, at, row = c.table[s, (ctx - r + i) // c.page], (ctx - r + i) % c.page, c.starts[s] + i
                assert near(c.row(k, pg, at), want[row, self.nq:], size[row, self.nq:])
        PW.check(c, self.nq, q, 0.125, out.astype(np.float64), lse, R.F32, self.window, self.sink)
        LP.check(out.reshape(n, -1).astype(np.float64), self.targets.get(), 5, (logp, entropy, top, top_logp))


def test_steps(eng, hip):
    rng = np.random.default_rng(21)
    nq, window, sink = 8, 90, 4
    steps = [Step(eng, hip, R.Cache(hip, rng, R.BF16, rows, ctx, 2, 64, 16), rng, nq, window, sink, [12, 10, 10])
             for rows, ctx in (([40, 1, 70], [40, 33, 200]), ([1, 1, 1, 1], [41, 700, 1, 201]))]
    size = max(s.workspace() for s in steps)
    ws, stream = hip.put(np.full(size, 0xFF, np.uint8)), hip.stream()
    drain = lambda: hip.lib.hipStreamSynchronize(stream)
    graphs = []
    for s in steps:
        say(f"eager: rows {s.cache.rows}")
        s.new_inputs()
        s.enqueue(ws, size, stream)
        assert drain() == 0
        s.check(s.results())
        graph, ge = C.c_void_p(), C.c_void_p()
        assert hip.lib.hipStreamBeginCapture(stream, 1) == 0
        s.enqueue(ws, size, stream)
        assert hip.lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.lib.hipGraphInstantiate(C.byref(ge), graph, None, None, 0) == 0
        graphs.append((graph, ge))
    for turn in range(3):
        say(f"replays {turn}")
        for s in steps:
            s.new_inputs()
        for _, ge in graphs:
            assert hip.lib.hipGraphLaunch(ge, stream) == 0
        assert drain() == 0
        for s in steps:
            got = s.results()
            s.check(got)
            s.enqueue(ws, size, stream)
            assert drain() == 0
            for a, b in zip(got, s.results()):
                assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    for graph, ge in graphs:
        hip.lib.hipGraphExecDestroy(ge)
        hip.lib.hipGraphDestroy(graph)
    hip.lib.hipStreamDestroy(stream)
