"""More operators of serving as timed cases: attention over pages with a
sliding window and first tokens that stay visible, RoPE of several position
axes with the append to the cache's pages, and log probabilities of given
tokens with entropy and the largest alternatives.

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


def _window(**kw):
    return _batch("window", **{**dict(window=1024, sink=4, freed=False), **kw})


def _axes(**kw):
    return _batch("axes", **{**dict(in_type="f32", norm=True, interleaved=False, rot=128, sections="24,20,20",
                                    in_turn=True, pos=0, width=32), **kw})


def _logp(**kw):
    return {**dict(op="logp", type="f32", n=1, vocab=VOCAB, extra=0, targets=1, top=20, masked=False), **kw}


def listed():
    return [
        # the small model's reply in an endless conversation, far past its window; old pages long given back
        _window(name="window_token", nq=16, ctx_lo=5203, ctx_hi=5203, window=512, page=16, freed=True),
        # one decode step of a serving batch on a sliding layer: short contexts whole, long ones their window
        _window(name="window_serve", seqs=48, ctx_lo=310, ctx_hi=30000, window=2048, page=16, freed=True),
        # two prompts' chunks scheduled together with decoding sequences
        _window(name="window_mixed", type="f16", seqs=9, chunks=2, rows=131, ctx_lo=700, ctx_hi=9100, window=1024,
                sink=16, page=32, slots_first=True),
        # chunks of eight prompts on a layer of short reach, heads of 64, no first tokens
        _window(name="window_short", seqs=8, chunks=8, rows=64, ctx_lo=900, ctx_hi=7001, window=128, sink=0, nq=64,
                hd=64, page=32),
        # the last call's worth of a long document
        _window(name="window_prompt", rows=512, chunks=1, ctx_lo=16384, ctx_hi=16384, window=4096, page=128),
        # a decode step of eight sessions that talk about pictures, projections in fp32, norms on q and k
        _axes(name="axes_step", seqs=8, ctx_lo=60, ctx_hi=2600, pos=2600),
        # a picture's patches in one full call, time, height and width one after the other in the head
        _axes(name="axes_image", rows=512, chunks=1, ctx_lo=4100, ctx_hi=4100, in_type="bf16", norm=False,
              sections="16,24,24", in_turn=False, pos=4100, page=128),
        # one session's token with its alternatives
        _logp(name="logp_token"),
        # scores of the answers' letters for a batch of questions, an odd vocabulary
        _logp(name="logp_choices", type="f16", n=37, vocab=32003, targets=16, top=1),
        # a decode step of 64 requests, tokens a grammar forbids masked out
        _logp(name="logp_batch", n=64, top=5, masked=True),
        # a prompt call's worth of rows, the perplexity alone
        _logp(name="logp_prompt", n=512, top=0),
        # a long document's rows with alternatives
        _logp(name="logp_document", type="bf16", n=2048),
    ]


_PAIRS = 512 * 4100        # (row, key) pairs of the largest listed attention
_KEYS = 48 * 2048          # cached rows of the largest listed batch
_LOGITS = 2048 * VOCAB     # of the largest listed rows of logits


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def _draw_batch(rng, window):
    nkv, group = rng.choice([2, 4, 8]), rng.choice([1, 2, 4, 5, 8])
    d = dict(type=rng.choice(["bf16", "f16"]), nkv=nkv, nq=min(32, nkv * group) // nkv * nkv,
             hd=rng.choice([64, 128, 128, 128, 256]), page=rng.choice([16, 32, 64, 128, 256]),
             slots_first=rng.random() < 0.3)
    seqs = _log_int(rng, 1, 48)
    rows = 1 if rng.random() < 0.5 else _log_int(rng, 2, 512)
    chunks = 0 if rows == 1 else rng.randint(1, min(seqs, max(1, 512 // rows)))
    heads = max(1.0, d["nq"] * d["hd"] / (32 * 128))
    # what a row sees is bounded by its window, what it costs by that
    reach = int(min(_PAIRS / heads / (max(1, chunks) * rows + seqs), _KEYS / seqs * 8 * 128 / (nkv * d["hd"])))
    reach = max(1, min(window, reach - 16))
    hi = _log_int(rng, rows, 30000 // (1 + seqs // 8))
    return dict(seqs=seqs, chunks=chunks, rows=rows, ctx_lo=_log_int(rng, rows, hi), ctx_hi=hi, **d), reach


def draw(rng):
    op = rng.choice(["window", "window", "axes", "logp"])
    if op == "logp":
        vocab = _log_int(rng, 1000, VOCAB)
        c = _logp(type=rng.choice(["f32", "bf16", "f16"]), vocab=vocab, extra=rng.choice([0, 0, rng.randint(1, 64)]),
                  targets=_log_int(rng, 1, 32), top=rng.choice([0, 1, 5, 20, rng.randint(1, 64)]),
                  masked=rng.random() < 0.3)
        c["n"] = _log_int(rng, 1, min(2048, _LOGITS // (2 if c["type"] == "f32" else 1) // (vocab + c["extra"])))
        return c
    d, reach = _draw_batch(rng, _log_int(rng, 1, 8192))
    if op == "window":
        return _window(window=reach, sink=rng.choice([0, rng.randint(1, 16), rng.randint(1, 64)]),
                       freed=rng.random() < 0.5, **d)
    half = d["hd"] // 2
    rot = rng.choice([2 * half, half, 2 * rng.randint(2, half)])
    n, in_turn = rng.choice([2, 3, 3, 3, 4]), rng.random() < 0.5
    pairs = rot // 2
    if in_turn:      # axis a > 0 takes pairs a, a + n, ... as long as it has some left, the first axis the others
        sizes = [rng.randint(0, (pairs - a + n - 1) // n) if pairs > a else 0 for a in range(1, n)]
        sizes = [pairs - sum(sizes)] + sizes
    else:
        cuts = sorted(rng.randint(0, pairs) for _ in range(n - 1))
        sizes = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
    return _axes(in_type=rng.choice(["f32", d["type"]]), norm=rng.random() < 0.5, interleaved=rng.random() < 0.5,
                 rot=rot, sections=",".join(map(str, sizes)), in_turn=in_turn, pos=_log_int(rng, d["ctx_hi"], 1000000),
                 width=_log_int(rng, 1, 100), **d)


def _lens(case):
    """(new rows, context) of every sequence, chunks first."""
    n, lo, hi = case["seqs"], case["ctx_lo"], case["ctx_hi"]
    ctx = [int(round(hi - (hi - lo) * i / max(1, n - 1))) for i in range(n)]
    return [(min(case["rows"], c) if i < case["chunks"] else min(1, c), c) for i, c in enumerate(ctx)]


def _reach(case, r, c):
    """Cached rows that the last r of c see: the first `a`, and from `b` on."""
    b = max(0, c - r - case["window"] + 1)
    return min(case["sink"], b), b


def work(case):
    op = case["op"]
    if op == "logp":
        size = 4 if case["type"] == "f32" else 2
        # one pass over the logits: a difference, an exponential and two sums each
        return {"bytes": case["n"] * (case["vocab"] * size + 8 * case["targets"] + 8 * case["top"] + 4),
                "flops": 4 * case["n"] * case["vocab"]}
    lens, nq, nkv, hd = _lens(case), case["nq"], case["nkv"], case["hd"]
    rows = sum(r for r, _ in lens)
    if op == "window":
        w, sink = case["window"], case["sink"]
        ends = [_reach(case, r, c) + (c,) for r, c in lens]
        keys = sum(a + c - b for a, b, c in ends)
        table = 4 * sum(-(-a // case["page"]) + -(-(c - b) // case["page"]) for a, b, c in ends)
        pairs = sum(min(p, w) + min(sink, max(0, p - w)) for r, c in lens for p in range(c - r + 1, c + 1))
        return {"bytes": 2 * (2 * keys * nkv * hd + 2 * rows * nq * hd) + 4 * rows * nq + table,
                "flops": 4 * hd * nq * pairs}
    size = 4 if case["in_type"] == "f32" else 2
    width = (nq + 2 * nkv) * hd
    return {"bytes": rows * (width * (size + 2) + 4 + 4 * len(case["sections"].split(","))),
            "flops": rows * width * (6 if case["norm"] else 3)}


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


def _head_first(case, pool):
    """A pool as [page][kv head][slot][d], whatever its order."""
    return pool.transpose(1, 2) if case["slots_first"] else pool


def _prepare_batch(case, seed):
    st = _State()
    st.case, st.lens = case, _lens(case)
    g, t, page = _gen(seed, 3), TYPES[case["type"]], case["page"]
    # page tables over a shuffled pool; pages that no later row sees either may have been given back
    held = []
    for r, c in st.lens:
        n = -(-c // page)
        if case["op"] == "window" and case["freed"]:
            a, b = _reach(case, r, c)
            held.append([i for i in range(n) if i * page < a or (i + 1) * page > b])
        elif case["op"] == "axes":       # the append writes the last rows alone
            held.append(list(range((c - r) // page, n)))
        else:
            held.append(list(range(n)))
    st.pages = sum(map(len, held)) + 3
    order = torch.randperm(st.pages, generator=g, device=DEV).tolist()
    table = np.full((len(held), max(-(-c // page) for _, c in st.lens)), -1, np.int32)
    for s, ids in enumerate(held):
        table[s, ids] = [order.pop() for _ in ids]
    st.table = torch.from_numpy(table).to(DEV)
    starts = [0]
    for r, _ in st.lens:
        starts.append(starts[-1] + r)
    st.n_rows = starts[-1]
    st.row_start, st.ctx_len = _i32(starts), _i32([c for _, c in st.lens])
    # keys and values as they leave a norm and a projection: of order one
    inner = (page, case["nkv"]) if case["slots_first"] else (case["nkv"], page)
    st.k = _randn(g, st.pages, *inner, case["hd"], type=t)
    st.v = _randn(g, st.pages, *inner, case["hd"], type=t)
    return st, g, t


def prepare(case, seed):
    if case["op"] == "logp":
        return _prepare_logp(case, seed)
    st, g, t = _prepare_batch(case, seed)
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    if case["op"] == "window":
        # queries a little larger than the keys, so that some rows attend sharply
        st.q = _randn(g, st.n_rows, nq, hd, type=t, scale=1.5)
        st.scale = 1.0 / math.sqrt(hd)
        st.out = torch.empty(st.n_rows, nq, hd, dtype=t, device=DEV)
        st.lse = torch.empty(st.n_rows, nq, device=DEV)
    else:
        # the fused projection's output
        st.qkv = _randn(g, st.n_rows, (nq + 2 * nkv) * hd, type=TYPES[case["in_type"]], scale=1.3)
        st.q_norm = 1 + 0.1 * _randn(g, hd) if case["norm"] else None
        st.k_norm = 1 + 0.1 * _randn(g, hd) if case["norm"] else None
        # a chunk is a picture of `width` patches a line, or the frames of a film; single tokens are text
        st.sections = [int(x) for x in case["sections"].split(",")]
        axes = len(st.sections)
        pos, w = [[] for _ in range(axes)], case["width"]
        for r, _ in st.lens:
            base = case["pos"] - r
            for i in range(r):
                at = [base + i // (w * 64), base + i // w, base + i % w, base + i % 7] if r > 1 else [base] * 4
                for a in range(axes):
                    pos[a].append(at[a])
        st.positions = _i32(pos)
        st.q_out = torch.empty(st.n_rows, nq, hd, dtype=t, device=DEV)
        st.turns = torch.tensor([THETA ** (-2 * j / case["rot"]) / (2 * math.pi) for j in range(case["rot"] // 2)],
                                dtype=torch.float64, device=DEV)
    if own:
        _plan_batch(st)
    elif case["op"] == "axes":
        st.axis = _axis_of(case, st.sections)
    return st


def _prepare_logp(case, seed):
    st = _State()
    st.case = case
    n, V = case["n"], case["vocab"]
    g = _gen(seed, 4)
    st.rows = torch.empty(n, V + case["extra"], dtype=TYPES[case["type"]], device=DEV)
    st.x = st.rows[:, :V]
    st.targets = torch.randint(0, V, (n, case["targets"]), generator=g, device=DEV, dtype=torch.int32)
    for r0 in range(0, n, 256):
        x = _randn(g, min(256, n - r0), V + case["extra"], scale=2.2)
        # a bell of unlikely tokens under a handful of likely ones, some of which are asked for
        hot = torch.randint(0, V, (x.shape[0], 24), generator=g, device=DEV)
        x.scatter_add_(1, hot, torch.rand(x.shape[0], 24, generator=g, device=DEV) * 9 + 3)
        if case["masked"]:
            x[:, 2::3] = -math.inf
        st.rows[r0:r0 + 256] = x.to(st.rows.dtype)
        st.targets[r0:r0 + 256, ::2] = hot[:, :(case["targets"] + 1) // 2].to(torch.int32)
    st.logp = torch.empty(n, case["targets"], device=DEV)
    st.entropy = torch.empty(n, device=DEV)
    st.top = torch.empty(n, case["top"], dtype=torch.int32, device=DEV)
    st.top_logp = torch.empty(n, case["top"], device=DEV)
    if own:
        from dpuf_amd import abi
        st.lib = abi.load_engine()
        st.ws_bytes = int(st.lib.dpuf_amd_logprobs_workspace(n, V, case["top"]))
        st.ws = torch.empty(max(1, st.ws_bytes), dtype=torch.uint8, device=DEV)
    return st


# ---------------------------------------------------------------------------
# the library's entry points
# ---------------------------------------------------------------------------

def _plan_batch(st):
    """The descriptors and workspace that a serving program keeps."""
    from dpuf_amd import abi
    case = st.case
    st.lib = abi.load_engine()
    kf = _head_first(case, st.k)
    st.p = abi.DpufAmdPages(type=TYPE_IDS[case["type"]], n_pages=st.pages, page_size=case["page"],
                            n_kv_heads=case["nkv"], head_dim=case["hd"], page_stride=kf.stride(0),
                            head_stride=kf.stride(1), row_stride=kf.stride(2), k=st.k.data_ptr(), v=st.v.data_ptr(),
                            w=None)
    st.b = abi.DpufAmdBatch(n_seqs=case["seqs"], n_rows=st.n_rows, table_stride=st.table.shape[1],
                            max_ctx=case["ctx_hi"], row_start=st.row_start.data_ptr(), ctx_len=st.ctx_len.data_ptr(),
                            page_table=st.table.data_ptr())
    if case["op"] == "window":
        st.ws_bytes = int(st.lib.dpuf_amd_paged_attn_window_workspace(C.byref(st.b), C.byref(st.p), case["nq"],
                                                                      case["window"], case["sink"]))
        st.ws = torch.empty(max(1, st.ws_bytes), dtype=torch.uint8, device=DEV)
    else:
        st.r = abi.DpufAmdRope(turns=st.turns.data_ptr(), rot_dim=case["rot"], interleaved=int(case["interleaved"]),
                               scale=1.0)
        sizes = st.sections + [0] * (4 - len(st.sections))
        st.a = abi.DpufAmdRopeAxes(n_axes=len(st.sections), sections=(C.c_int32 * 4)(*sizes),
                                   in_turn=int(case["in_turn"]))


def _check(rc):
    if rc != 0:
        raise RuntimeError(f"operator returned {rc}")


def _run_own(st):
    case, s = st.case, torch.cuda.current_stream().cuda_stream
    if case["op"] == "logp":
        _check(st.lib.dpuf_amd_logprobs(TYPE_IDS[case["type"]], case["n"], case["vocab"], st.rows.shape[1],
                                        st.x.data_ptr(), case["targets"], st.targets.data_ptr(), case["top"],
                                        st.logp.data_ptr(), st.entropy.data_ptr(),
                                        st.top.data_ptr() if case["top"] else None,
                                        st.top_logp.data_ptr() if case["top"] else None, st.ws.data_ptr(), st.ws_bytes,
                                        s))
        return st.logp, st.entropy, st.top, st.top_logp
    b, p = C.byref(st.b), C.byref(st.p)
    if case["op"] == "window":
        _check(st.lib.dpuf_amd_paged_attn_window(b, p, case["nq"], st.q.data_ptr(), st.scale, case["window"],
                                                 case["sink"], TYPE_IDS[case["type"]], st.out.data_ptr(),
                                                 st.lse.data_ptr(), st.ws.data_ptr(), st.ws_bytes, s))
        return st.out, st.lse
    at, size, width = st.qkv.data_ptr(), st.qkv.element_size(), st.qkv.shape[1]
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    _check(st.lib.dpuf_amd_rope_append_axes(b, p, C.byref(st.r), C.byref(st.a), st.positions.data_ptr(),
                                            st.positions.stride(0), TYPE_IDS[case["in_type"]], nq, at,
                                            at + nq * hd * size, at + (nq + nkv) * hd * size, width, width, width,
                                            st.q_norm.data_ptr() if case["norm"] else None,
                                            st.k_norm.data_ptr() if case["norm"] else None, EPS, st.q_out.data_ptr(),
                                            s))
    return st.q_out, st.k, st.v


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _run_plain(st):
    if st.case["op"] == "logp":
        return _plain_logp(st)
    return _plain_window(st) if st.case["op"] == "window" else _plain_axes(st)


def _plain_window(st):
    case = st.case
    page, w, sink, g = case["page"], case["window"], case["sink"], case["nq"] // case["nkv"]
    kp, vp, r0 = _head_first(case, st.k), _head_first(case, st.v), 0
    for s, (r, c) in enumerate(st.lens):
        a, b = _reach(case, r, c)
        at = torch.cat([torch.arange(a, device=DEV), torch.arange(b, c, device=DEV)])
        pg, sl = st.table[s].long()[at // page], at % page
        place = torch.arange(c - r, c, device=DEV)[:, None]
        hidden = (at[None] > place) | ((at[None] <= place - w) & (at[None] >= sink))
        for h in range(case["nkv"]):
            keys, values = kp[pg, h, sl].float(), vp[pg, h, sl].float()
            q = st.q[r0:r0 + r, h * g:(h + 1) * g].float().reshape(r * g, -1)
            x = (q @ keys.t().contiguous()).mul_(st.scale).view(r, g, -1)
            x.masked_fill_(hidden[:, None, :], -math.inf)
            top = x.amax(-1, keepdim=True)
            p = x.sub_(top).exp_()
            total = p.sum(-1, keepdim=True)
            o = p.div_(total).flatten(0, 1) @ values
            st.out[r0:r0 + r, h * g:(h + 1) * g] = o.view(r, g, -1).to(st.out.dtype)
            st.lse[r0:r0 + r, h * g:(h + 1) * g] = (top + total.log()).squeeze(-1)
        r0 += r
    return st.out, st.lse


def _axis_of(case, sections):
    """Axis of each pair of rotated columns."""
    n, pairs = len(sections), case["rot"] // 2
    if case["in_turn"]:
        axis = [j % n if j < n * sections[j % n] else 0 for j in range(pairs)]
    else:
        axis = [a for a in range(n) for _ in range(sections[a])]
    return torch.tensor(axis, device=DEV)


def _plain_axes(st):
    case = st.case
    nq, nkv, hd, rot = case["nq"], case["nkv"], case["hd"], case["rot"]
    x = st.qkv.float().view(st.n_rows, nq + 2 * nkv, hd)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    angle = st.positions[st.axis].t().double() * st.turns[None, :]
    angle = (angle - angle.round()) * (2 * math.pi)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(y, norm):
        if norm is not None:
            y = y * ((y * y).mean(-1, keepdim=True) + EPS).rsqrt() * norm
        y = y.clone()
        a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if case["interleaved"] else (y[..., :rot // 2], y[..., rot // 2:rot])
        a2, b2 = a * cos - b * sin, a * sin + b * cos
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


def _plain_logp(st):
    case = st.case
    for r0 in range(0, case["n"], 512):
        r1 = min(case["n"], r0 + 512)
        x = st.x[r0:r1].float()
        d = x - x.amax(1, keepdim=True)
        e = d.exp()
        total = e.sum(1, keepdim=True)
        log_total = total.log()
        e.div_(total)
        st.entropy[r0:r1] = log_total.squeeze(1) - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1)
        st.logp[r0:r1] = d.gather(1, st.targets[r0:r1].long()) - log_total
        if case["top"]:
            order = x.sort(dim=1, descending=True, stable=True)[1][:, :case["top"]]
            st.top[r0:r1] = order.to(torch.int32)
            st.top_logp[r0:r1] = d.gather(1, order) - log_total
    return st.logp, st.entropy, st.top, st.top_logp


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# the operators' definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logp":
        return _exact_logp(st)
    return _exact_window(st) if case["op"] == "window" else _exact_axes(st)


def _exact_window(st):
    case = st.case
    g, w, page = case["nq"] // case["nkv"], case["window"], case["page"]
    out = torch.zeros(st.n_rows, case["nq"], case["hd"], dtype=torch.float64, device=DEV)
    lse = torch.zeros(st.n_rows, case["nq"], dtype=torch.float64, device=DEV)
    row = 0
    for s, (r, c) in enumerate(st.lens):
        for i0 in range(0, r, 64):      # 64 rows of every head at a time
            i1 = min(r, i0 + 64)
            first, last = c - r + i0, c - r + i1 - 1          # their places
            lo = max(0, first - w + 1)
            near = torch.arange(lo, last + 1, device=DEV)
            far = torch.arange(0, min(lo, case["sink"]), device=DEV)
            t = torch.cat([far, near])
            pg = st.table[s][torch.div(t, page, rounding_mode="floor")].long()
            k, v = _head_first(case, st.k)[pg, :, t % page].double(), _head_first(case, st.v)[pg, :, t % page].double()
            p = torch.arange(first, last + 1, device=DEV)[:, None]
            seen = (t <= p) & ((t > p - w) | (t < case["sink"]))
            for head in range(case["nq"]):
                score = st.q[row + i0:row + i1, head].double() @ k[:, head // g].t().contiguous() * st.scale
                score = torch.where(seen, score, torch.full_like(score, -math.inf))
                z = torch.logsumexp(score, 1)
                lse[row + i0:row + i1, head] = z
                out[row + i0:row + i1, head] = torch.exp(score - z[:, None]) @ v[:, head // g]
        row += r
    return out, lse


def _exact_axes(st):
    case = st.case
    nq, nkv, hd, rot, n = case["nq"], case["nkv"], case["hd"], case["rot"], len(st.sections)
    pairs = rot // 2
    # the pairs of each axis, listed
    if case["in_turn"]:
        of = {a: list(range(a, n * st.sections[a], n)) for a in range(1, n)}
        of[0] = sorted(set(range(pairs)) - {j for js in of.values() for j in js})
    else:
        at = np.cumsum([0] + st.sections)
        of = {a: list(range(at[a], at[a + 1])) for a in range(n)}
    angle = torch.zeros(st.n_rows, pairs, dtype=torch.float64, device=DEV)
    for a, js in of.items():
        freq = torch.tensor([THETA ** (-2.0 * j / rot) for j in js], dtype=torch.float64, device=DEV)
        angle[:, js] = st.positions[a].double()[:, None] * freq
    z = torch.polar(torch.ones_like(angle), angle)
    heads = st.qkv.double().view(st.n_rows, -1, hd)

    def rotated(y, weight):
        if weight is not None:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / hd + EPS) * weight.double()
        part = y[..., :rot]
        if case["interleaved"]:
            part = torch.view_as_real(torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous()) * z[:, None])
            part = part.flatten(-2)
        else:
            c = torch.complex(part[..., :pairs].contiguous(), part[..., pairs:].contiguous()) * z[:, None]
            part = torch.cat([c.real, c.imag], -1)
        return torch.cat([part, y[..., rot:]], -1)

    k_pool, v_pool = st.k.double(), st.v.double()
    k, row = rotated(heads[:, nq:nq + nkv], st.k_norm), 0
    for s, (r, c) in enumerate(st.lens):
        t = torch.arange(c - r, c, device=DEV)
        pg = st.table[s].long()[torch.div(t, case["page"], rounding_mode="floor")]
        _head_first(case, k_pool)[pg, :, t % case["page"]] = k[row:row + r]
        _head_first(case, v_pool)[pg, :, t % case["page"]] = heads[row:row + r, nq + nkv:]
        row += r
    return rotated(heads[:, :nq], st.q_norm), k_pool, v_pool


def _exact_logp(st):
    case, n, V = st.case, st.case["n"], st.case["vocab"]
    logp = torch.zeros(n, case["targets"], dtype=torch.float64, device=DEV)
    entropy = torch.zeros(n, dtype=torch.float64, device=DEV)
    top = torch.zeros(n, case["top"], dtype=torch.int32, device=DEV)
    top_logp = torch.zeros(n, case["top"], dtype=torch.float64, device=DEV)
    for r in range(0, n, 128):
        x = st.x[r:r + 128].double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        entropy[r:r + 128] = -torch.xlogy(lp.exp(), lp.exp()).sum(1)
        logp[r:r + 128] = torch.take_along_dim(lp, st.targets[r:r + 128].long(), 1)
        if case["top"]:
            # the largest one at a time; argmax of "is it the largest" finds its first place
            left = x.clone()
            for i in range(case["top"]):
                first = (left == left.amax(1, keepdim=True)).to(torch.uint8).argmax(1, keepdim=True)
                top[r:r + 128, i] = first.squeeze(1).to(torch.int32)
                top_logp[r:r + 128, i] = lp.gather(1, first).squeeze(1)
                left.scatter_(1, first, -math.inf)
    return logp, entropy, top, top_logp
