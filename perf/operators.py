"""The operators of paged serving as timed cases: RoPE with the append to the
cache's pages, attention of new tokens over pages, the accumulation of
attention weights per cached row, eviction by those weights, and sampling.

Each case is one call as a serving program makes it, with everything already
on the device: `own` selects the library's entry points (include/dpuf_amd.h,
through ctypes) or the same operator in elementary torch operations.

A batch is a list of sequences; sequence s has rows_s new tokens (the last
rows_s of its ctx_s cached rows) and a page table.  The first `chunks`
sequences in the batch's order have `rows` new tokens, the others one; context
lengths are spread evenly from `ctx_lo` to `ctx_hi`.

Head counts and head dims are those of the Qwen3-0.6B (16 / 8 / 128) and
Qwen3-8B (32 / 8 / 128) shapes of dpuf_amd.model, or generic; the vocabulary
is theirs.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False

DEV = "cuda"
VOCAB = 151936
THETA = 1e6
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TYPE_IDS = {"f32": 0, "bf16": 1, "f16": 2}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _batch(op, **kw):
    c = dict(op=op, type="bf16", seqs=1, chunks=0, rows=1, ctx_lo=64, ctx_hi=64, nq=32, nkv=8, hd=128, page=64,
             slots_first=False)
    c.update(kw)
    return c


def _rope(**kw):
    return _batch("rope", **{**dict(in_type="f32", norm=True, interleaved=False, rot=128, scaling="none", factor=1.0,
                                    pos=0), **kw})


def _sample(**kw):
    return {**dict(op="sample", type="f32", n=1, vocab=VOCAB, mixed=False, temperature=0.8, top_k=0, top_p=1.0,
                   min_p=0.0), **kw}


def listed():
    return [
        # a chat reply of the small model, a few dozen tokens in
        _batch("attn", name="attn_token", nq=16, ctx_lo=75, ctx_hi=75, page=16),
        # one decode step of a serving batch with contexts of every length
        _batch("attn", name="attn_serve", seqs=48, ctx_lo=310, ctx_hi=6000),
        # two prompts' chunks scheduled together with the decoding sequences
        _batch("attn", name="attn_mixed", type="f16", seqs=9, chunks=2, rows=131, ctx_lo=700, ctx_hi=4100, page=32,
               slots_first=True),
        # the last call's worth of a long document
        _batch("attn", name="attn_prompt", rows=512, chunks=1, ctx_lo=16384, ctx_hi=16384, page=128),
        # the weights of a decode step, for a batch whose caches are near their budget
        _batch("weights", name="weights_step", seqs=24, ctx_lo=900, ctx_hi=4096),
        # the weights of the last 256-token chunk of a prompt
        _batch("weights", name="weights_chunk", type="f16", rows=256, chunks=1, ctx_lo=4096, ctx_hi=4096, page=32),
        # a conversation that reached its budget of 1 024 rows
        _batch("evict", name="evict_one", nq=16, ctx_lo=1290, ctx_hi=1290, keep=1024, sink=4, recent=64, page=16),
        # long prompts cut to half after their prefill
        _batch("evict", name="evict_many", seqs=8, ctx_lo=6100, ctx_hi=9000, keep=4096, sink=4, recent=256),
        # a decode step of eight sessions, projections in fp32, norms on q and k
        _rope(name="rope_step", seqs=8, ctx_lo=60, ctx_hi=2600, pos=2600),
        # a full prefill call of a model with interleaved pairs over half the head, stretched for long contexts
        _rope(name="rope_chunk", rows=512, chunks=1, ctx_lo=16384, ctx_hi=16384, in_type="bf16", norm=False,
              interleaved=True, rot=64, scaling="yarn", factor=4.0, pos=130000, page=128),
        # one session's next token
        _sample(name="sample_one", top_k=50, top_p=0.95),
        # a serving batch, every request with settings of its own
        _sample(name="sample_many", n=64, mixed=True),
    ]


_PAIRS = 512 * 16384       # (row, key) pairs of the largest listed attention
_KEYS = 48 * 3155          # cached rows of the largest listed batch


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def _draw_batch(rng, op, max_ctx):
    nkv, group = rng.choice([2, 4, 8]), rng.choice([1, 2, 4, 5, 8])
    d = dict(type=rng.choice(["bf16", "f16"]), nkv=nkv, nq=min(32, nkv * group) // nkv * nkv,
             hd=rng.choice([64, 128, 128, 128, 256]), page=rng.choice([16, 32, 64, 128, 256]),
             slots_first=rng.random() < 0.3)
    seqs = _log_int(rng, 1, 48)
    rows = 1 if rng.random() < 0.5 else _log_int(rng, 2, 512)
    chunks = 0 if rows == 1 else rng.randint(1, min(seqs, max(1, 512 // rows)))
    heads = d["nq"] * d["hd"] / (32 * 128)
    top = min(max_ctx, int(_KEYS / seqs * 8 * 128 / (d["nkv"] * d["hd"])),
              int(_PAIRS / (max(1, chunks) * rows + seqs) / heads))
    top = max(top, rows + 1)
    hi = _log_int(rng, rows, top)
    return _batch(op, seqs=seqs, chunks=chunks, rows=rows, ctx_lo=_log_int(rng, rows, hi), ctx_hi=hi, **d)


def draw(rng):
    op = rng.choice(["attn", "attn", "weights", "evict", "rope", "sample"])
    if op == "sample":
        n = _log_int(rng, 1, 64)
        return _sample(n=n, vocab=_log_int(rng, 1000, VOCAB), mixed=rng.random() < 0.5,
                       type=rng.choice(["f32", "bf16", "f16"]), temperature=rng.uniform(0.1, 1.8),
                       top_k=rng.choice([0, _log_int(rng, 1, 5000)]), top_p=rng.choice([1.0, rng.uniform(0.05, 1.0)]),
                       min_p=rng.choice([0.0, rng.uniform(0.0, 0.3)]))
    c = _draw_batch(rng, op, 16384)
    if op == "evict":
        c["chunks"], c["rows"] = 0, 1
        c["keep"] = _log_int(rng, 1, c["ctx_hi"])
        c["sink"] = rng.randint(0, min(8, c["keep"]))
        c["recent"] = rng.randint(0, c["keep"] - c["sink"])
    if op == "rope":
        c = _rope(**{k: v for k, v in c.items() if k != "op"})
        half = c["hd"] // 2
        c.update(in_type=rng.choice(["f32", c["type"]]), norm=rng.random() < 0.5, interleaved=rng.random() < 0.5,
                 rot=rng.choice([2 * half, half, 2 * rng.randint(1, half)]),
                 scaling=rng.choice(["none", "linear", "llama3", "yarn"]), pos=_log_int(rng, c["ctx_hi"], 1000000))
        c["factor"] = 1.0 if c["scaling"] == "none" else rng.choice([2.0, 4.0, 8.0])
    return c


def _lens(case):
    """(new rows, context) of every sequence, chunks first."""
    n, lo, hi = case["seqs"], case["ctx_lo"], case["ctx_hi"]
    ctx = [int(round(hi - (hi - lo) * i / max(1, n - 1))) for i in range(n)]
    return [(min(case["rows"], c) if i < case["chunks"] else min(1, c), c) for i, c in enumerate(ctx)]


def _pairs(case):
    """(row, visible key) pairs of one head."""
    return sum(r * c - r * (r - 1) // 2 for r, c in _lens(case))


def work(case):
    op = case["op"]
    if op == "sample":
        size = 4 if case["type"] == "f32" else 2
        # one pass over the logits; a difference, a product and an exponential each
        return {"bytes": case["n"] * (case["vocab"] * size + 28), "flops": 3 * case["n"] * case["vocab"]}
    lens, nq, nkv, hd = _lens(case), case["nq"], case["nkv"], case["hd"]
    rows, keys = sum(r for r, _ in lens), sum(c for _, c in lens)
    table = 4 * sum(-(-c // case["page"]) for _, c in lens)
    if op == "attn":
        return {"bytes": 2 * (2 * keys * nkv * hd + 2 * rows * nq * hd) + 4 * rows * nq + table,
                "flops": 4 * hd * nq * _pairs(case)}
    if op == "weights":
        return {"bytes": 2 * (keys * nkv * hd + rows * nq * hd) + 4 * rows * nq + 8 * keys * nkv + table,
                "flops": 2 * hd * nq * _pairs(case)}
    if op == "evict":
        kept = sum(min(c, case["keep"]) for _, c in lens)
        return {"bytes": nkv * (4 * keys + kept * (2 * 2 * hd * 2 + 2 * 4 + 4)) + table, "flops": nkv * keys}
    size = 4 if case["in_type"] == "f32" else 2
    width = (nq + 2 * nkv) * hd
    return {"bytes": rows * (width * (size + 2) + 8), "flops": rows * width * (6 if case["norm"] else 3)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class _State:
    pass


def _gen(seed, *what):
    g = torch.Generator(device=DEV)
    for w in what:
        seed = (seed * 1000003 + w + 1) % (1 << 61)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, type=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).mul_(scale).to(type)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pool_shape(case, pages):
    inner = (case["page"], case["nkv"]) if case["slots_first"] else (case["nkv"], case["page"])
    return (pages, *inner, case["hd"])


def _head_first(case, pool):
    """A pool as [page][kv head][slot][d], whatever its order."""
    return pool.transpose(1, 2) if case["slots_first"] else pool


def _tables(case, lens, g, spare):
    """Page tables over a shuffled pool: (table, pages of the pool)."""
    per = [-(-c // case["page"]) for c in lens]
    pages = sum(per) + spare
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(lens), max(1, max(per)), dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pages


def _prepare_batch(case, seed):
    st = _State()
    st.case, st.lens = case, _lens(case)
    t = TYPES[case["type"]]
    g = _gen(seed, 1)
    st.table, pages = _tables(case, [c for _, c in st.lens], g, 3)
    starts = [0]
    for r, _ in st.lens:
        starts.append(starts[-1] + r)
    st.n_rows = starts[-1]
    st.row_start, st.ctx_len = _i32(starts), _i32([c for _, c in st.lens])
    st.scale = 1.0 / math.sqrt(case["hd"])
    # keys and values as they leave a norm and a projection: of order one
    st.k = _randn(g, *_pool_shape(case, pages), type=t)
    st.v = _randn(g, *_pool_shape(case, pages), type=t)
    # weights that earlier steps have left: most rows near nothing, a few heavy ones
    st.w = _randn(g, pages, case["nkv"], case["page"]).mul_(2.0).exp_()
    st.pages = pages
    return st, g, t


def prepare(case, seed):
    if case["op"] == "sample":
        return _prepare_sample(case, seed)
    st, g, t = _prepare_batch(case, seed)
    nq, hd = case["nq"], case["hd"]
    if case["op"] in ("attn", "weights"):
        # queries a little larger than the keys, so that some rows attend sharply
        st.q = _randn(g, st.n_rows, nq, hd, type=t, scale=1.5)
        st.lse = torch.empty(st.n_rows, nq, device=DEV)
    if case["op"] == "attn":
        st.out = torch.empty(st.n_rows, nq, hd, dtype=t, device=DEV)
    elif case["op"] == "weights":
        _each_head(st, lambda s, h, p, lse: _put(st.lse, s, h, st, lse))
        st.w_out = st.w.clone()
        st.decay = 0.98
    elif case["op"] == "evict":
        keep = [min(c, case["keep"]) for _, c in st.lens]
        st.dst_table, dst_pages = _tables(case, keep, g, 2)
        shape = _pool_shape(case, dst_pages)
        st.dst_k, st.dst_v = torch.zeros(shape, dtype=t, device=DEV), torch.zeros(shape, dtype=t, device=DEV)
        st.dst_w = torch.zeros(dst_pages, case["nkv"], case["page"], device=DEV)
        st.dst_pages = dst_pages
        st.kept = torch.full((case["seqs"], case["nkv"], case["keep"]), -1, dtype=torch.int32, device=DEV)
        st.new_len = torch.zeros(case["seqs"], dtype=torch.int32, device=DEV)
    else:
        width = (nq + 2 * case["nkv"]) * hd
        it = TYPES[case["in_type"]]
        st.qkv = _randn(g, st.n_rows, width, type=it, scale=1.3)  # the fused projection's output
        st.q_norm = 1 + 0.1 * _randn(g, hd) if case["norm"] else None
        st.k_norm = 1 + 0.1 * _randn(g, hd) if case["norm"] else None
        pos = []
        for r, _ in st.lens:
            pos += list(range(case["pos"] - r, case["pos"]))
        st.positions = _i32(pos)
        st.q_out = torch.empty(st.n_rows, nq, hd, dtype=t, device=DEV)
    if own:
        _plan_batch(st)
    else:
        if case["op"] == "rope":
            st.turns, st.mscale = _turns(case)
            st.turns = torch.tensor(st.turns, dtype=torch.float64, device=DEV)
    return st


def _prepare_sample(case, seed):
    st = _State()
    st.case = case
    n, V = case["n"], case["vocab"]
    g = _gen(seed, 2)
    # a bell of unlikely tokens under a handful of likely ones
    x = _randn(g, n, V, scale=2.2)
    hot = torch.randint(0, V, (n, 24), generator=g, device=DEV)
    x.scatter_add_(1, hot, torch.rand(n, 24, generator=g, device=DEV) * 9 + 3)
    st.x = x.to(TYPES[case["type"]])
    st.u = torch.rand(n, generator=g, device=DEV)
    i = torch.arange(n, device=DEV)
    full = lambda v, t: torch.full((n,), v, dtype=t, device=DEV)
    if case["mixed"]:  # requests of every kind: greedy, top-k, top-p, min-p, all of them, none
        kind = i % 6
        st.t = torch.where(kind == 0, 0.0, 0.5 + torch.rand(n, generator=g, device=DEV))
        st.top_k = torch.where((kind == 1) | (kind == 4), 20 + 37 * (i % 7), 0).to(torch.int32)
        st.top_p = torch.where((kind == 2) | (kind == 4), 0.8 + 0.19 * torch.rand(n, generator=g, device=DEV), 1.0)
        st.min_p = torch.where((kind == 3) | (kind == 4), 0.02, 0.0)
    else:
        st.t, st.top_k = full(case["temperature"], torch.float32), full(case["top_k"], torch.int32)
        st.top_p, st.min_p = full(case["top_p"], torch.float32), full(case["min_p"], torch.float32)
    st.tokens = torch.zeros(n, dtype=torch.int32, device=DEV)
    st.logprobs = torch.zeros(n, device=DEV)
    if own:
        from dpuf_amd import abi
        st.lib = abi.load_engine()
        size = int(st.lib.dpuf_amd_sample_workspace(n, V))
        st.ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    return st


# ---------------------------------------------------------------------------
# the library's entry points
# ---------------------------------------------------------------------------

def _plan_batch(st):
    """The descriptors and workspace that a serving program keeps."""
    from dpuf_amd import abi
    case = st.case
    st.lib = abi.load_engine()

    def pages(k, v, w, n):
        kf = _head_first(case, k)
        return abi.DpufAmdPages(type=TYPE_IDS[case["type"]], n_pages=n, page_size=case["page"],
                                n_kv_heads=case["nkv"], head_dim=case["hd"], page_stride=kf.stride(0),
                                head_stride=kf.stride(1), row_stride=kf.stride(2), k=k.data_ptr(), v=v.data_ptr(),
                                w=w.data_ptr())

    st.b = abi.DpufAmdBatch(n_seqs=case["seqs"], n_rows=st.n_rows, table_stride=st.table.shape[1],
                            max_ctx=case["ctx_hi"], row_start=st.row_start.data_ptr(), ctx_len=st.ctx_len.data_ptr(),
                            page_table=st.table.data_ptr())
    st.p = pages(st.k, st.v, st.w_out if case["op"] == "weights" else st.w, st.pages)
    if case["op"] == "attn":
        size = int(st.lib.dpuf_amd_paged_attn_workspace(C.byref(st.b), C.byref(st.p), case["nq"]))
        st.ws = torch.empty(max(1, size), dtype=torch.uint8, device=DEV)
        st.ws_bytes = size
    elif case["op"] == "evict":
        st.dp = pages(st.dst_k, st.dst_v, st.dst_w, st.dst_pages)
    elif case["op"] == "rope":
        spec = abi.DpufAmdRopeSpec(rot_dim=case["rot"], theta=THETA, scaling=SCALINGS.index(case["scaling"]),
                                   factor=case["factor"], low_freq=1.0, high_freq=4.0, beta_fast=32.0, beta_slow=1.0,
                                   orig_max_pos=ORIG)
        turns, mscale = np.zeros(case["rot"] // 2), C.c_float(0)
        rc = st.lib.dpuf_amd_rope_turns(C.byref(spec), turns.ctypes.data_as(C.c_void_p), C.byref(mscale))
        assert rc == 0, rc
        st.turns = torch.tensor(turns, dtype=torch.float64, device=DEV)
        st.r = abi.DpufAmdRope(turns=st.turns.data_ptr(), rot_dim=case["rot"], interleaved=int(case["interleaved"]),
                               scale=mscale.value)


def _check(rc):
    if rc != 0:
        raise RuntimeError(f"operator returned {rc}")


def _run_own(st):
    case, s = st.case, torch.cuda.current_stream().cuda_stream
    op = case["op"]
    if op == "sample":
        _check(st.lib.dpuf_amd_sample(TYPE_IDS[case["type"]], case["n"], case["vocab"], case["vocab"],
                                      st.x.data_ptr(), st.t.data_ptr(), st.top_k.data_ptr(), st.top_p.data_ptr(),
                                      st.min_p.data_ptr(), st.u.data_ptr(), st.tokens.data_ptr(),
                                      st.logprobs.data_ptr(), st.ws.data_ptr(), st.ws.numel(), s))
        return st.tokens, st.logprobs
    b, p = C.byref(st.b), C.byref(st.p)
    if op == "attn":
        _check(st.lib.dpuf_amd_paged_attn(b, p, case["nq"], st.q.data_ptr(), st.scale, TYPE_IDS[case["type"]],
                                          st.out.data_ptr(), st.lse.data_ptr(), st.ws.data_ptr(), st.ws_bytes, s))
        return st.out, st.lse
    if op == "weights":
        _check(st.lib.dpuf_amd_paged_attn_weights(b, p, case["nq"], st.q.data_ptr(), st.scale, st.lse.data_ptr(),
                                                  st.decay, st.w.data_ptr(), s))
        return st.w_out
    if op == "evict":
        _check(st.lib.dpuf_amd_paged_evict(b, p, case["keep"], case["sink"], case["recent"], C.byref(st.dp),
                                           st.dst_table.data_ptr(), st.dst_table.shape[1], st.kept.data_ptr(),
                                           st.new_len.data_ptr(), s))
        return st.dst_k, st.dst_v, st.dst_w, st.kept, st.new_len
    at, size, width = st.qkv.data_ptr(), st.qkv.element_size(), st.qkv.shape[1]
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    _check(st.lib.dpuf_amd_rope_append(b, p, C.byref(st.r), st.positions.data_ptr(), TYPE_IDS[case["in_type"]], nq,
                                       at, at + nq * hd * size, at + (nq + nkv) * hd * size, width, width, width,
                                       st.q_norm.data_ptr() if case["norm"] else None,
                                       st.k_norm.data_ptr() if case["norm"] else None, EPS, st.q_out.data_ptr(), s))
    return st.q_out, st.k, st.v


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

SCALINGS = ["none", "linear", "llama3", "yarn"]
ORIG = 32768  # positions the model was trained on


def _turns(case):
    """Turns per position of each pair, and the factor on rotated columns."""
    r, f = case["rot"], case["factor"]
    inv = [THETA ** (-2 * j / r) for j in range(r // 2)]
    mscale = 1.0
    if case["scaling"] == "linear":
        inv = [x / f for x in inv]
    elif case["scaling"] == "llama3":
        out = []
        for x in inv:
            waves = ORIG * x / (2 * math.pi)  # turns over the trained range: low 1, high 4
            mix = min(1.0, max(0.0, (waves - 1.0) / (4.0 - 1.0)))
            out.append((1 - mix) * x / f + mix * x)
        inv = out
    elif case["scaling"] == "yarn":
        dim = lambda turns: r * math.log(ORIG / (turns * 2 * math.pi)) / (2 * math.log(THETA))
        lo, hi = max(0, math.floor(dim(32.0))), min(r - 1, math.ceil(dim(1.0)))
        ramp = [min(1.0, max(0.0, (j - lo) / max(hi - lo, 1e-3))) for j in range(r // 2)]
        inv = [x / f * m + x * (1 - m) for x, m in zip(inv, ramp)]
        mscale = 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
    return [x / (2 * math.pi) for x in inv], mscale


def _rows_of(st, pool, s, n):
    """Cached rows [0, n) of sequence s as [kv head][n][...]."""
    per = -(-n // st.case["page"])
    x = pool[st.table[s, :per].long()]          # [pages][kv head][slot]...
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _put(dst, s, h, st, value):
    r0 = sum(r for r, _ in st.lens[:s])
    g = st.case["nq"] // st.case["nkv"]
    dst[r0:r0 + st.lens[s][0], h * g:(h + 1) * g] = value


def _each_head(st, use, keep_p=False, dtype=torch.float32):
    """use(s, kv head, probabilities or None, lse) of every sequence and kv
    head: [rows][group][keys] and [rows][group]."""
    case = st.case
    g = case["nq"] // case["nkv"]
    k_pool, r0 = _head_first(case, st.k), 0
    for s, (r, c) in enumerate(st.lens):
        if r == 0:
            continue
        keys = _rows_of(st, k_pool, s, c).to(dtype)
        mask = torch.arange(c, device=DEV)[None, :] > torch.arange(c - r, c, device=DEV)[:, None]
        for h in range(case["nkv"]):
            q = st.q[r0:r0 + r, h * g:(h + 1) * g].to(dtype).reshape(r * g, -1)
            x = (q @ keys[h].t().contiguous()).mul_(st.scale).view(r, g, c)
            x.masked_fill_(mask[:, None, :], -math.inf)
            top = x.amax(-1, keepdim=True)
            p = x.sub_(top).exp_()
            total = p.sum(-1, keepdim=True)
            use(s, h, p.div_(total) if keep_p else None, (top + total.log()).squeeze(-1))
        r0 += r


def _run_plain(st):
    case = st.case
    op = case["op"]
    if op == "sample":
        return _plain_sample(st)
    if op == "attn":
        v_pool, values = _head_first(case, st.v), {}

        def attend(s, h, p, lse):
            if s not in values:
                values.clear()
                values[s] = _rows_of(st, v_pool, s, st.lens[s][1]).float()
            o = p.flatten(0, 1) @ values[s][h]
            _put(st.out, s, h, st, o.view(*p.shape[:2], -1).to(st.out.dtype))
            _put(st.lse, s, h, st, lse)

        _each_head(st, attend, keep_p=True)
        return st.out, st.lse
    if op == "weights":
        return _plain_weights(st)
    if op == "evict":
        return _plain_evict(st)
    return _plain_rope(st)


def _plain_weights(st):
    case = st.case
    g, r0 = case["nq"] // case["nkv"], 0
    k_pool = _head_first(case, st.k)
    for s, (r, c) in enumerate(st.lens):
        keys, w = _rows_of(st, k_pool, s, c).float(), _rows_of(st, st.w, s, c).clone()
        w *= st.decay
        mask = torch.arange(c, device=DEV)[None, :] > torch.arange(c - r, c, device=DEV)[:, None]
        for h in range(case["nkv"]):
            q = st.q[r0:r0 + r, h * g:(h + 1) * g].float().reshape(r * g, -1)
            x = (q @ keys[h].t().contiguous()).mul_(st.scale).view(r, g, c)
            x.sub_(st.lse[r0:r0 + r, h * g:(h + 1) * g, None]).exp_()
            x.masked_fill_(mask[:, None, :], 0.0)
            w[h] += x.sum((0, 1))
        at = torch.arange(c, device=DEV)
        st.w_out[st.table[s].long()[at // case["page"]], :, at % case["page"]] = w.t()
        r0 += r
    return st.w_out


def _plain_evict(st):
    case = st.case
    page, sink, recent = case["page"], case["sink"], case["recent"]
    k, v = _head_first(case, st.k), _head_first(case, st.v)
    dk, dv = _head_first(case, st.dst_k), _head_first(case, st.dst_v)
    heads = torch.arange(case["nkv"], device=DEV)[:, None]
    for s, (_, c) in enumerate(st.lens):
        n = min(c, case["keep"])
        w = _rows_of(st, st.w, s, c)
        if n == c:
            slots = torch.arange(c, device=DEV).expand(case["nkv"], c)
        else:
            order = w.clone()
            order[:, :sink] = math.inf
            order[:, c - recent:] = math.inf
            slots = order.sort(dim=1, descending=True, stable=True)[1][:, :n].sort(dim=1)[0]
        src, at = st.table[s].long()[slots // page], torch.arange(n, device=DEV)
        dst = st.dst_table[s].long()[at // page][None, :].expand(case["nkv"], n)
        to = (at % page)[None, :].expand(case["nkv"], n)
        dk[dst, heads, to] = k[src, heads, slots % page]
        dv[dst, heads, to] = v[src, heads, slots % page]
        st.dst_w[dst, heads, to] = st.w[src, heads, slots % page]
        st.kept[s, :, :n] = slots.to(torch.int32)
        st.new_len[s:s + 1] = n
    return st.dst_k, st.dst_v, st.dst_w, st.kept, st.new_len


def _plain_rope(st):
    case = st.case
    nq, nkv, hd, rot = case["nq"], case["nkv"], case["hd"], case["rot"]
    x = st.qkv.float().view(st.n_rows, nq + 2 * nkv, hd)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    angle = st.positions.double()[:, None] * st.turns[None, :]
    angle = (angle - angle.round()) * (2 * math.pi)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(y, norm):
        if norm is not None:
            y = y * ((y * y).mean(-1, keepdim=True) + EPS).rsqrt() * norm
        y = y.clone()
        a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if case["interleaved"] else (y[..., :rot // 2], y[..., rot // 2:rot])
        a2, b2 = (a * cos - b * sin) * st.mscale, (a * sin + b * cos) * st.mscale
        a.copy_(a2)
        b.copy_(b2)
        return y

    st.q_out.copy_(turn(q, st.q_norm))
    k = turn(k, st.k_norm)
    pages, slots = [], []
    for s, (r, c) in enumerate(st.lens):
        at = torch.arange(c - r, c, device=DEV)
        pages.append(st.table[s].long()[at // case["page"]])
        slots.append(at % case["page"])
    pages, slots = torch.cat(pages), torch.cat(slots)
    _head_first(case, st.k)[pages, :, slots] = k.to(st.k.dtype)
    _head_first(case, st.v)[pages, :, slots] = v.to(st.v.dtype)
    return st.q_out, st.k, st.v


def _plain_sample(st):
    # in 64 bits: the draw and the top-p border fall between sums of many small terms
    n, V = st.x.shape
    x = st.x.double()
    top = x.amax(1, keepdim=True)
    t = st.t.double()[:, None]
    w = torch.where(t > 0, ((x - top) / t.clamp_min(1e-30)).exp(), torch.zeros_like(x))
    order = x.sort(dim=1, descending=True, stable=True)[1]
    sw = w.gather(1, order)
    rank = torch.arange(V, device=DEV)[None, :]
    k = torch.where((st.top_k <= 0) | (st.top_k > V), V, st.top_k)[:, None]
    sw = torch.where(rank < k, sw, torch.zeros_like(sw))
    before = sw.cumsum(1) - sw
    goal = st.top_p.double()[:, None] * sw.sum(1, keepdim=True)
    keep = (rank < k) & ((st.top_p[:, None] >= 1) | (before < goal) | (rank == 0))
    keep &= (sw >= st.min_p.double()[:, None].clamp(max=1.0)) | (rank == 0)
    kept = torch.zeros(n, V, dtype=torch.bool, device=DEV).scatter_(1, order, keep)
    w = torch.where(kept, w, torch.zeros_like(w))
    run = w.cumsum(1)
    total = run[:, -1:]
    hit = kept & (run > st.u.double()[:, None] * total)
    tok = hit.to(torch.int8).argmax(1)
    greedy = st.t <= 0
    tok = torch.where(greedy, order[:, 0], tok)
    p = w.gather(1, tok[:, None]) / total
    st.tokens.copy_(tok)
    st.logprobs.copy_(torch.where(greedy, torch.zeros_like(p[:, 0]), p[:, 0].log()))
    return st.tokens, st.logprobs


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# the operators' definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    if case["op"] in ("attn", "weights"):
        return _exact_attention(st)
    if case["op"] == "evict":
        return _exact_evict(st)
    return _exact_rope(st)


def _slots(st, s, c):
    at = torch.arange(c, device=DEV)
    return st.table[s].long()[at // st.case["page"]], at % st.case["page"]


def _exact_attention(st):
    case = st.case
    g = case["nq"] // case["nkv"]
    out = torch.zeros(st.n_rows, case["nq"], case["hd"], dtype=torch.float64, device=DEV)
    lses = torch.zeros(st.n_rows, case["nq"], dtype=torch.float64, device=DEV)
    weights = st.w.double()
    row = 0
    for s, (r, c) in enumerate(st.lens):
        pg, sl = _slots(st, s, c)
        k, v = _head_first(case, st.k)[pg, :, sl], _head_first(case, st.v)[pg, :, sl]  # [c][kv head][d]
        fresh = torch.zeros(c, case["nkv"], dtype=torch.float64, device=DEV)
        for i0 in range(0, r, 64):      # 64 rows of every head at a time
            i1 = min(r, i0 + 64)
            seen = torch.arange(c, device=DEV)[None] <= (c - r + torch.arange(i0, i1, device=DEV))[:, None]
            for head in range(case["nq"]):
                score = st.q[row + i0:row + i1, head].double() @ k[:, head // g].double().t().contiguous() * st.scale
                score = torch.where(seen, score, torch.full_like(score, -math.inf))
                if case["op"] == "attn":
                    lse = torch.logsumexp(score, 1)
                    lses[row + i0:row + i1, head] = lse
                    out[row + i0:row + i1, head] = torch.exp(score - lse[:, None]) @ v[:, head // g].double()
                else:
                    lse = st.lse[row + i0:row + i1, head].double()
                    fresh[:, head // g] += torch.exp(score - lse[:, None]).sum(0)
        if case["op"] == "weights":
            weights[pg, :, sl] = st.decay * weights[pg, :, sl] + fresh
        row += r
    return (out, lses) if case["op"] == "attn" else weights


def _exact_evict(st):
    case = st.case
    page, keep = case["page"], case["keep"]
    outs = [_head_first(case, x).cpu().clone() for x in (st.dst_k, st.dst_v)] + [st.dst_w.cpu().clone()]
    pools = [_head_first(case, x).cpu() for x in (st.k, st.v)] + [st.w.cpu()]
    table, dst_table, kept = st.table.cpu().numpy(), st.dst_table.cpu().numpy(), st.kept.cpu().numpy()
    lens = np.zeros(case["seqs"], np.int32)
    for s, (_, c) in enumerate(st.lens):
        n = lens[s] = min(c, keep)
        slot = np.arange(c)
        for h in range(case["nkv"]):
            w = pools[2][table[s, slot // page], h, slot % page].numpy()
            middle = slot[case["sink"]:c - case["recent"]] if n < c else slot[:0]
            best = middle[np.lexsort((middle, -w[middle].astype(np.float64)))][:n - case["sink"] - case["recent"]]
            chosen = np.sort(np.concatenate([slot[:case["sink"]], best, slot[c - case["recent"]:]])) if n < c else slot
            kept[s, h, :n] = chosen
            to = np.arange(n)
            for dst, src in zip(outs, pools):
                dst[dst_table[s, to // page], h, to % page] = src[table[s, chosen // page], h, chosen % page]
    k, v = (_head_first(case, x).contiguous().to(DEV) for x in outs[:2])
    return k, v, outs[2].to(DEV), torch.from_numpy(kept).to(DEV), torch.from_numpy(lens).to(DEV)


def _exact_rope(st):
    case = st.case
    nq, nkv, hd, rot = case["nq"], case["nkv"], case["hd"], case["rot"]
    turns, mscale = _turns(case)
    pairs = torch.tensor(turns, dtype=torch.float64, device=DEV) * (2 * math.pi)
    z = torch.polar(torch.full((st.n_rows, rot // 2), float(mscale), dtype=torch.float64, device=DEV),
                    st.positions.double()[:, None] * pairs)
    heads = st.qkv.double().view(st.n_rows, -1, hd)

    def rotated(y, weight):
        if weight is not None:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / hd + EPS) * weight.double()
        part = y[..., :rot]
        if case["interleaved"]:
            part = torch.view_as_real(torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous()) * z[:, None])
            part = part.flatten(-2)
        else:
            c = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * z[:, None]
            part = torch.cat([c.real, c.imag], -1)
        return torch.cat([part, y[..., rot:]], -1)

    k_pool, v_pool = st.k.double(), st.v.double()
    k, row = rotated(heads[:, nq:nq + nkv], st.k_norm), 0
    for s, (r, c) in enumerate(st.lens):
        pg, sl = _slots(st, s, c)
        _head_first(case, k_pool)[pg[c - r:], :, sl[c - r:]] = k[row:row + r]
        _head_first(case, v_pool)[pg[c - r:], :, sl[c - r:]] = heads[row:row + r, nq + nkv:]
        row += r
    return rotated(heads[:, :nq], st.q_norm), k_pool, v_pool


def _exact_sample(st):
    x, n = st.x.double().cpu().numpy(), st.x.shape[0]
    t, top_k, top_p, min_p, u = (a.double().cpu().numpy() for a in (st.t, st.top_k, st.top_p, st.min_p, st.u))
    tokens, logs = np.zeros(n, np.int32), np.zeros(n)
    for i in range(n):
        row = x[i]
        if t[i] <= 0:
            tokens[i] = int(np.argmax(row))
            continue
        order = np.argsort(-row, kind="stable")
        w = np.exp((row[order] - row[order[0]]) / t[i])
        if 0 < top_k[i] < len(w):
            w = w[:int(top_k[i])]
        if top_p[i] < 1:
            reach = np.cumsum(w)
            w = w[:max(1, int(np.searchsorted(reach, top_p[i] * reach[-1])) + 1)]
        w = w[:max(1, int((w >= min(1.0, min_p[i])).sum()))]
        back = np.argsort(order[:len(w)])
        ids, run_ = order[:len(w)][back], np.cumsum(w[back])
        at = min(int(np.searchsorted(run_, u[i] * run_[-1], side="right")), len(ids) - 1)
        tokens[i] = ids[at]
        logs[i] = math.log(w[back][at] / run_[-1])
    return torch.from_numpy(tokens).to(DEV), torch.from_numpy(logs).to(DEV)
