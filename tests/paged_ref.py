"""Helpers of the paged-serving tests: device buffers through the HIP runtime
the library links, 16-bit element types in numpy, a paged KV cache on the
host, and the operators in float64 from their definitions."""
import ctypes as C

import numpy as np

from dpuf_amd import abi
from dpuf_amd import model as M

F32, BF16, F16 = 0, 1, 2
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}   # of a value, after rounding to nearest
H2D, D2H, D2D = 1, 2, 3


def to_type(x, t):
    """float array -> storage (uint16 of bf16 / fp16, float32), nearest even."""
    x = np.asarray(x, np.float32)
    if t == F32:
        return x.copy()
    if t == F16:
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_type(s, t):
    """storage -> float64."""
    if t == F32:
        return s.astype(np.float64)
    if t == F16:
        return s.view(np.float16).astype(np.float64)
    return (s.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Hip:
    """The HIP runtime as the library's process has it."""

    def __init__(self):
        lib = C.CDLL("libamdhip64.so.7")
        P = C.c_void_p
        for name, args in (("hipMalloc", [C.POINTER(P), C.c_size_t]), ("hipFree", [P]),
                           ("hipMemcpy", [P, P, C.c_size_t, C.c_int]), ("hipDeviceSynchronize", []),
                           ("hipStreamCreateWithFlags", [C.POINTER(P), C.c_uint]), ("hipStreamDestroy", [P]),
                           ("hipStreamSynchronize", [P]), ("hipStreamBeginCapture", [P, C.c_int]),
                           ("hipStreamEndCapture", [P, C.POINTER(P)]),
                           ("hipGraphInstantiate", [C.POINTER(P), P, P, P, C.c_size_t]), ("hipGraphLaunch", [P, P]),
                           ("hipGraphExecDestroy", [P]), ("hipGraphDestroy", [P])):
            getattr(lib, name).argtypes = args
        self.lib = lib
        self.kept = []

    def put(self, host, offset=0):
        """A device copy of a host array, `offset` bytes into its allocation."""
        d = Dev(self, np.ascontiguousarray(host), offset)
        self.kept.append(d)
        return d

    def sync(self):
        assert self.lib.hipDeviceSynchronize() == 0

    def stream(self):
        s = C.c_void_p()
        assert self.lib.hipStreamCreateWithFlags(C.byref(s), 1) == 0
        return s

    def free_all(self):
        for d in self.kept:
            d.free()
        self.kept = []


class Dev:
    def __init__(self, hip, host, offset):
        self.hip, self.like = hip, host
        self.base = C.c_void_p()
        assert hip.lib.hipMalloc(C.byref(self.base), max(host.nbytes, 16) + offset) == 0
        self.p = self.base.value + offset
        self.set(host)

    def set(self, host):
        host = np.ascontiguousarray(host)
        assert host.nbytes == self.like.nbytes
        if host.nbytes:
            assert self.hip.lib.hipMemcpy(self.p, M.ptr(host), host.nbytes, H2D) == 0

    def get(self):
        self.hip.sync()
        out = np.empty_like(self.like)
        if out.nbytes:
            assert self.hip.lib.hipMemcpy(M.ptr(out), self.p, out.nbytes, D2H) == 0
        return out

    def free(self):
        if self.base:
            self.hip.lib.hipFree(self.base)
            self.base = None


class Cache:
    """A paged cache of several sequences on the host and on the device.

    `rows[s]`: new rows, `ctx[s]`: cached rows with them.  Unused rows of a
    page, and whole unused pages, hold NaN: nothing may come from them."""

    def __init__(self, hip, rng, t, rows, ctx, nkv, hd, page, slots_first=False, spare=3, kscale=1.0, bad=(),
                 table_extra=2):
        self.hip, self.t, self.rows, self.ctx = hip, t, list(rows), list(ctx)
        self.nkv, self.hd, self.page, self.slots_first = nkv, hd, page, slots_first
        per = [-(-c // page) for c in ctx]
        n = sum(per) + spare
        ids = rng.permutation(n).astype(np.int32)
        self.table = np.full((len(ctx), max(1, max(per)) + table_extra), -1, np.int32)
        at = 0
        for s, m in enumerate(per):
            self.table[s, :m] = ids[at:at + m]
            at += m
        for s, i in bad:        # pages outside the pool
            self.table[s, i] = rng.choice([-1, n, 2 ** 31 - 1, -2 ** 31])
        self.n = n
        shape = (n, page, nkv, hd) if slots_first else (n, nkv, page, hd)
        self.k = to_type(np.full(shape, np.nan, np.float32), t)
        self.v = self.k.copy()
        self.w = np.full((n, nkv, page), np.nan, np.float32)
        for s, c in enumerate(ctx):
            for i in range(c):
                if not self.ok(s, i):
                    continue
                pg, r = self.table[s, i // page], i % page
                self.row(self.k, pg, r)[...] = to_type(rng.standard_normal((nkv, hd)) * kscale, t)
                self.row(self.v, pg, r)[...] = to_type(rng.standard_normal((nkv, hd)), t)
                self.w[pg, :, r] = np.exp(2 * rng.standard_normal(nkv))
        self.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.n_rows = int(self.starts[-1])
        self.upload()

    def ok(self, s, i):
        return 0 <= self.table[s, i // self.page] < self.n

    def row(self, pool, pg, r):
        return pool[pg, r] if self.slots_first else pool[pg, :, r]

    def upload(self):
        put = self.hip.put
        self.dk, self.dv, self.dw = put(self.k), put(self.v), put(self.w)
        self.d_starts, self.d_ctx, self.d_table = put(self.starts), put(np.array(self.ctx, np.int32)), put(self.table)

    def upload_into(self):
        """The pools as they were, in the same device memory."""
        for d, host in ((self.dk, self.k), (self.dv, self.v), (self.dw, self.w)):
            d.set(host)

    def gather(self, pool, s, h):
        """Cached rows of (s, kv head h) in float64, NaN where absent."""
        out = np.full((self.ctx[s], self.hd), np.nan)
        for i in range(self.ctx[s]):
            if self.ok(s, i):
                out[i] = from_type(self.row(pool, self.table[s, i // self.page], i % self.page)[h], self.t)
        return out

    def present(self, s):
        return np.array([self.ok(s, i) for i in range(self.ctx[s])], bool)

    def pages(self, w=True, dw=None):
        it = self.hd
        if self.slots_first:
            st = (self.page * self.nkv * it, it, self.nkv * it)
        else:
            st = (self.page * self.nkv * it, self.page * it, it)
        d = dw if dw is not None else self.dw
        return abi.DpufAmdPages(type=self.t, n_pages=self.n, page_size=self.page, n_kv_heads=self.nkv,
                                head_dim=self.hd, page_stride=st[0], head_stride=st[1], row_stride=st[2],
                                k=self.dk.p, v=self.dv.p, w=d.p if w else None)

    def batch(self, max_ctx=None, n_rows=None):
        return abi.DpufAmdBatch(n_seqs=len(self.ctx), n_rows=self.n_rows if n_rows is None else n_rows,
                                table_stride=self.table.shape[1],
                                max_ctx=max(self.ctx) if max_ctx is None else max_ctx,
                                row_start=self.d_starts.p, ctx_len=self.d_ctx.p, page_table=self.d_table.p)


def attention(cache, q, scale, nq):
    """Outputs [rows][nq][hd], lse [rows][nq] and, per output, what the bounds
    need: A = sum p |v|, the largest |score| sum of products, p's sum over
    rows per cached row (weights)."""
    G = nq // cache.nkv
    n = cache.n_rows
    out = np.zeros((n, nq, cache.hd))
    lse = np.full((n, nq), -np.inf)
    A = np.zeros((n, nq, cache.hd))
    S = np.zeros((n, nq))
    vmax = np.zeros((n, nq))
    weights = [np.zeros((cache.nkv, c)) for c in cache.ctx]
    for s, (r, c) in enumerate(zip(cache.rows, cache.ctx)):
        there = cache.present(s)
        for h in range(cache.nkv):
            k, v = cache.gather(cache.k, s, h), cache.gather(cache.v, s, h)
            for i in range(r):
                see = np.where(there & (np.arange(c) <= c - r + i))[0]
                if len(see) == 0:
                    continue
                row = cache.starts[s] + i
                for j in range(h * G, (h + 1) * G):
                    x = k[see] @ q[row, j] * scale
                    m = x.max()
                    e = np.exp(x - m)
                    lse[row, j] = m + np.log(e.sum())
                    p = e / e.sum()
                    out[row, j] = p @ v[see]
                    A[row, j] = p @ np.abs(v[see])
                    S[row, j] = (np.abs(k[see]) @ np.abs(q[row, j])).max() * scale
                    vmax[row, j] = np.abs(v[see]).max()
                    weights[s][h, see] += p
    return out, lse, A, S, vmax, weights


def score_error(S, hd):
    """Bound of a score's absolute error (and so of ln p): hd products and
    sums in fp32, then the scale, the base-2 product and the exponential."""
    return S * (hd + 4) * 2.0 ** -24 + 2.0 ** -21


def attention_bound(t, out_t, out, A, S, vmax, hd, ctx):
    """A probability is rounded to type t before the product with V (half a
    step of each term; fp16 below 2^-14: 2^-25 at most, of a sum of at least
    one), the sum runs in fp32 over at most ctx terms and their rescales."""
    d = score_error(S, hd)[..., None]
    under = ctx * 2.0 ** -25 * vmax[..., None] if t == F16 else 0.0
    return HALF_STEP[out_t] * np.abs(out) + A * (HALF_STEP[t] + 2 * d + (ctx + 64) * 2.0 ** -24) * 1.01 + under + 1e-30
