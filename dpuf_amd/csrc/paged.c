/*
 * paged.c -- entry points of the paged-serving operators (include/dpuf_amd.h):
 * every argument is checked here, on the host, before a kernel that relies on
 * it is launched; what only the device knows (lengths, page numbers) the
 * kernels clamp or mask themselves.
 */
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "../../include/dpuf_amd.h"
#include "hip_layer.h"

#define MAX_SEQS 16384
#define MAX_ROWS 65536
#define MAX_ROW_STRIDE ((int64_t)1 << 26) /* the kernels hold 16 rows' offsets in 32 bits */

static int aligned(const void* p, uintptr_t n) { return p && ((uintptr_t)p & (n - 1)) == 0; }

/* The device all of the n non-NULL pointers are on, or -1. */
static int32_t device_of(const void* const* p, int n) {
    int32_t dev = -1;
    for (int i = 0; i < n; i++) {
        if (!p[i]) continue;
        const int32_t d = dpuf_hip_ptr_device(p[i]);
        if (d < 0 || (dev >= 0 && d != dev)) return -1;
        dev = d;
    }
    return dev;
}

/* Memory that a call reads or writes. */
typedef struct {
    const void* p;
    uint64_t n;
} Span;

static int overlap(Span a, Span b) {
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    return a.p && b.p && a.n && b.n && x < y + b.n && y < x + a.n;
}

/* Whether any of the n spans at a shares memory with any of the m at b. */
static int any_overlap(const Span* a, int n, const Span* b, int m) {
    for (int i = 0; i < n; i++)
        for (int j = 0; j < m; j++)
            if (overlap(a[i], b[j])) return 1;
    return 0;
}
/* Whether any two of the n spans do. */
static int overlap_within(const Span* a, int n) {
    for (int i = 1; i < n; i++)
        if (any_overlap(a + i, 1, a, i)) return 1;
    return 0;
}
#define COUNT(a) ((int)(sizeof(a) / sizeof((a)[0])))

static int32_t check_pages(const DpufAmdPages* p) {
    if (!p) return -1;
    if (p->type != DPUF_AMD_BF16 && p->type != DPUF_AMD_F16) return -5;
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return -5;
    if (p->n_pages < 1 || p->n_kv_heads < 1 || p->n_kv_heads > 256) return -2;
    if (p->page_size < 16 || p->page_size > 1024 || (p->page_size & (p->page_size - 1))) return -2;
    const int64_t s[3] = {p->page_stride, p->head_stride, p->row_stride};
    for (int i = 0; i < 3; i++)
        if (s[i] < p->head_dim || s[i] % 8 != 0) return -4;
    if (p->row_stride > MAX_ROW_STRIDE) return -4;
    if (!aligned(p->k, 16) || !aligned(p->v, 16)) return -1;
    return 0;
}

static int32_t check_batch(const DpufAmdBatch* b, const DpufAmdPages* p) {
    if (!b || !aligned(b->row_start, 4) || !aligned(b->ctx_len, 4) || !aligned(b->page_table, 4)) return -1;
    if (b->n_seqs < 1 || b->n_seqs > MAX_SEQS || b->n_rows < 0 || b->n_rows > MAX_ROWS || b->table_stride < 1 ||
        (int64_t)b->table_stride * p->page_size > (int64_t)1 << 30)
        return -2;
    return 0;
}

static int32_t check_heads(const DpufAmdPages* p, int32_t nq) {
    return nq < 1 || nq % p->n_kv_heads != 0 || nq / p->n_kv_heads > 32 ? -2 : 0;
}

static int64_t type_size(int32_t t) { return t == DPUF_AMD_F32 ? 4 : 2; }

/* n elements of `size` bytes, n rows of `cols` of them, and what strides of any
 * size span: more than an address space holds counts as all of it. */
static Span run(const void* p, int64_t n, int64_t size) {
    const Span s = {p, (uint64_t)(n * size)};
    return s;
}
static Span bounded(const void* p, unsigned __int128 n, int64_t size) {
    const uint64_t most = UINT64_MAX / 2 - (uintptr_t)p / 2;
    const Span s = {p, n > most / (uint64_t)size ? most : (uint64_t)n * (uint64_t)size};
    return s;
}
static Span rows_of(const void* p, int64_t n, int64_t stride, int64_t cols, int64_t size) {
    return bounded(p, n > 0 ? (unsigned __int128)(n - 1) * (uint64_t)stride + (uint64_t)cols : 0, size);
}
/* The batch's three arrays. */
static void batch_spans(const DpufAmdBatch* b, Span* s) {
    s[0] = run(b->row_start, b->n_seqs + 1, 4);
    s[1] = run(b->ctx_len, b->n_seqs, 4);
    s[2] = run(b->page_table, (int64_t)b->n_seqs * b->table_stride, 4);
}
/* The pages' k or v from its first row to its last, and w. */
static Span pool_span(const DpufAmdPages* p, const void* at) {
    const unsigned __int128 n = (unsigned __int128)(p->n_pages - 1) * (uint64_t)p->page_stride +
                                (unsigned __int128)(p->n_kv_heads - 1) * (uint64_t)p->head_stride +
                                (unsigned __int128)(p->page_size - 1) * (uint64_t)p->row_stride + (uint64_t)p->head_dim;
    return bounded(at, n, 2);
}
static Span weight_span(const DpufAmdPages* p, const void* at) {
    return run(at, (int64_t)p->n_pages * p->n_kv_heads * p->page_size, 4);
}

/* Runs `call` with the pointers' device current. */
#define ON_DEVICE(dev, call)                               \
    do {                                                   \
        const int32_t back_ = dpuf_hip_device_enter(dev);  \
        if (dpuf_hip_ok()) call;                           \
        dpuf_hip_device_leave(back_);                      \
        return dpuf_hip_ok() ? 0 : -6;                     \
    } while (0)

DPUF_EXPORT int32_t dpuf_amd_rope_turns(const DpufAmdRopeSpec* spec, double* turns, float* scale) {
    if (!spec || !turns || !scale) return -1;
    const int32_t r = spec->rot_dim;
    const double theta = spec->theta, f = spec->factor, two_pi = 6.283185307179586476925;
    const double orig = spec->orig_max_pos;
    if (r < 2 || r > 256 || (r & 1) || !(theta > 1.0) || !isfinite(theta)) return -2;
    if (spec->scaling < DPUF_AMD_ROPE_PLAIN || spec->scaling > DPUF_AMD_ROPE_YARN) return -2;
    if (spec->scaling != DPUF_AMD_ROPE_PLAIN && !(f >= 1.0 && isfinite(f))) return -2;
    if (spec->scaling >= DPUF_AMD_ROPE_LLAMA3 && spec->orig_max_pos < 1) return -2;
    if (spec->scaling == DPUF_AMD_ROPE_LLAMA3 &&
        !(spec->low_freq > 0.0f && spec->high_freq > spec->low_freq && isfinite(spec->high_freq)))
        return -2;
    if (spec->scaling == DPUF_AMD_ROPE_YARN &&
        !(spec->beta_slow > 0.0f && spec->beta_fast > spec->beta_slow && isfinite(spec->beta_fast)))
        return -2;
    double lo = 0.0, hi = 0.0;
    *scale = 1.0f;
    if (spec->scaling == DPUF_AMD_ROPE_YARN) {
        /* dims whose pair makes beta turns over the trained positions */
        lo = floor(r * log(orig / (spec->beta_fast * two_pi)) / (2.0 * log(theta)));
        hi = ceil(r * log(orig / (spec->beta_slow * two_pi)) / (2.0 * log(theta)));
        if (lo < 0.0) lo = 0.0;
        if (hi > r - 1) hi = r - 1;
        *scale = (float)(f > 1.0 ? 0.1 * log(f) + 1.0 : 1.0);
    }
    for (int32_t j = 0; j < r / 2; j++) {
        double t = pow(theta, -2.0 * j / r) / two_pi;
        double keep = 1.0; /* share of the frequency left as it is */
        if (spec->scaling == DPUF_AMD_ROPE_LINEAR) keep = 0.0;
        if (spec->scaling == DPUF_AMD_ROPE_LLAMA3)
            keep = (orig * t - spec->low_freq) / ((double)spec->high_freq - spec->low_freq);
        if (spec->scaling == DPUF_AMD_ROPE_YARN) keep = 1.0 - (j - lo) / (hi - lo > 1e-3 ? hi - lo : 1e-3);
        keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        turns[j] = t * keep + (1.0 - keep) * (keep < 1.0 ? t / f : 0.0);
    }
    return 0;
}

/* Axis a > 0 takes pairs a, a + n, ... of `pairs` in turn, as many as it says. */
static int32_t check_axes(const DpufAmdRopeAxes* x, int32_t pairs) {
    if (!x) return -1;
    if (x->n_axes < 1 || x->n_axes > 4) return -2;
    int64_t sum = 0;
    for (int32_t a = 0; a < x->n_axes; a++) {
        if (x->sections[a] < 0 || x->sections[a] > pairs) return -2;
        if (x->in_turn && a > 0 && x->sections[a] > 0 && a + x->n_axes * (x->sections[a] - 1) >= pairs) return -2;
        sum += x->sections[a];
    }
    return sum == pairs ? 0 : -2;
}

/* axes NULL: one axis. */
static int32_t rope_append(const DpufAmdBatch* batch, const DpufAmdPages* pages, const DpufAmdRope* rope,
                           const DpufAmdRopeAxes* axes, const int32_t* d_positions, int64_t pos_stride,
                           int32_t in_type, int32_t n_q_heads, const void* d_q, const void* d_k, const void* d_v,
                           int64_t q_stride, int64_t k_stride, int64_t v_stride, const float* d_q_norm,
                           const float* d_k_norm, float eps, void* d_q_out, void* hip_stream) {
    dpuf_hip_clear_error();
    int32_t rc = check_pages(pages);
    if (rc == 0) rc = check_batch(batch, pages);
    if (rc != 0) return rc;
    if (in_type != DPUF_AMD_F32 && in_type != DPUF_AMD_BF16 && in_type != DPUF_AMD_F16) return -5;
    if (!rope || !aligned(rope->turns, 8)) return -1;
    const int64_t hd = pages->head_dim, nkv = pages->n_kv_heads, es = type_size(in_type);
    if (rope->rot_dim < 2 || (rope->rot_dim & 1) || rope->rot_dim > hd || !isfinite(rope->scale)) return -2;
    const int32_t n_axes = axes ? axes->n_axes : 1;
    rc = axes ? check_axes(axes, rope->rot_dim / 2) : 0;
    if (rc != 0) return rc;
    if (n_axes > 1 && pos_stride < batch->n_rows) return -4;
    if (n_q_heads < 0 || n_q_heads > 32 * nkv) return -2;
    if ((n_q_heads == 0) != (d_q == NULL) || (n_q_heads == 0) != (d_q_out == NULL)) return -1;
    if (batch->n_rows == 0) return 0;
    if (!aligned(d_positions, 4) || !aligned(d_k, 16) || !aligned(d_v, 16)) return -1;
    if (n_q_heads && (!aligned(d_q, 16) || !aligned(d_q_out, 16))) return -1;
    if ((d_q_norm && !aligned(d_q_norm, 4)) || (d_k_norm && !aligned(d_k_norm, 4))) return -1;
    if ((d_q_norm || d_k_norm) && !(eps >= 0.0f && isfinite(eps))) return -2;
    const int64_t st[3] = {q_stride, k_stride, v_stride}, need[3] = {n_q_heads * hd, nkv * hd, nkv * hd};
    for (int i = n_q_heads ? 0 : 1; i < 3; i++)
        if (st[i] < need[i] || st[i] % 8 != 0) return -4;
    const int in_place = d_q && d_q_out == d_q && in_type == pages->type && q_stride == need[0];
    Span in[9] = {rows_of(d_k, batch->n_rows, k_stride, need[1], es), rows_of(d_v, batch->n_rows, v_stride, need[2], es),
                  rows_of(d_positions, n_axes, n_axes > 1 ? pos_stride : 0, batch->n_rows, 4),
                  run(rope->turns, rope->rot_dim / 2, 8), run(d_q_norm, hd, 4), run(d_k_norm, hd, 4)};
    batch_spans(batch, in + 6);
    const Span q = rows_of(d_q, batch->n_rows, q_stride, need[0], es);
    /* k and v may lie interleaved in one allocation */
    const Span out[] = {run(d_q_out, batch->n_rows * need[0], 2), pool_span(pages, pages->k), pool_span(pages, pages->v),
                        weight_span(pages, pages->w)};
    if (any_overlap(out, 4, in, COUNT(in)) || any_overlap(out + 1, 3, &q, 1) || (!in_place && overlap(out[0], q)) ||
        any_overlap(out, 1, out + 1, 3) || any_overlap(out + 1, 2, out + 3, 1))
        return -1;
    const void* ps[] = {pages->k, pages->v, pages->w, batch->row_start, batch->ctx_len, batch->page_table, rope->turns,
                        d_positions, d_q, d_k, d_v, d_q_norm, d_k_norm, d_q_out};
    const int32_t dev = device_of(ps, (int)(sizeof ps / sizeof ps[0]));
    if (dev < 0) return -1;
    ON_DEVICE(dev, dpuf_hip_rope_append(hip_stream, batch, pages, rope, axes, d_positions, pos_stride, in_type,
                                        n_q_heads, d_q, d_k, d_v, q_stride, k_stride, v_stride, d_q_norm, d_k_norm, eps,
                                        d_q_out));
}

DPUF_EXPORT int32_t dpuf_amd_rope_append(const DpufAmdBatch* batch, const DpufAmdPages* pages,
                                         const DpufAmdRope* rope, const int32_t* d_positions, int32_t in_type,
                                         int32_t n_q_heads, const void* d_q, const void* d_k, const void* d_v,
                                         int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                         const float* d_q_norm, const float* d_k_norm, float eps, void* d_q_out,
                                         void* hip_stream) {
    return rope_append(batch, pages, rope, NULL, d_positions, 0, in_type, n_q_heads, d_q, d_k, d_v, q_stride, k_stride,
                       v_stride, d_q_norm, d_k_norm, eps, d_q_out, hip_stream);
}

DPUF_EXPORT int32_t dpuf_amd_rope_append_axes(const DpufAmdBatch* batch, const DpufAmdPages* pages,
                                              const DpufAmdRope* rope, const DpufAmdRopeAxes* axes,
                                              const int32_t* d_positions, int64_t pos_stride, int32_t in_type,
                                              int32_t n_q_heads, const void* d_q, const void* d_k, const void* d_v,
                                              int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                              const float* d_q_norm, const float* d_k_norm, float eps, void* d_q_out,
                                              void* hip_stream) {
    if (!axes) return -1;
    return rope_append(batch, pages, rope, axes, d_positions, pos_stride, in_type, n_q_heads, d_q, d_k, d_v, q_stride,
                       k_stride, v_stride, d_q_norm, d_k_norm, eps, d_q_out, hip_stream);
}

DPUF_EXPORT size_t dpuf_amd_paged_attn_workspace(const DpufAmdBatch* batch, const DpufAmdPages* pages,
                                                 int32_t n_q_heads) {
    if (check_pages(pages) != 0 || check_batch(batch, pages) != 0 || check_heads(pages, n_q_heads) != 0) return 0;
    return dpuf_hip_paged_attn_workspace(batch, pages, n_q_heads, 0, 0);
}

static int window_ok(int32_t window, int32_t sink) {
    return window >= 1 && window <= 1 << 30 && sink >= 0 && sink <= 1 << 30;
}

DPUF_EXPORT size_t dpuf_amd_paged_attn_window_workspace(const DpufAmdBatch* batch, const DpufAmdPages* pages,
                                                        int32_t n_q_heads, int32_t window, int32_t sink) {
    if (check_pages(pages) != 0 || check_batch(batch, pages) != 0 || check_heads(pages, n_q_heads) != 0 ||
        !window_ok(window, sink))
        return 0;
    return dpuf_hip_paged_attn_workspace(batch, pages, n_q_heads, window, sink);
}

/* window 0: none. */
static int32_t paged_attn(const DpufAmdBatch* batch, const DpufAmdPages* pages, int32_t n_q_heads, const void* d_q,
                          float scale, int32_t window, int32_t sink, int32_t out_type, void* d_out, float* d_lse,
                          void* d_workspace, size_t workspace_bytes, void* hip_stream) {
    dpuf_hip_clear_error();
    int32_t rc = check_pages(pages);
    if (rc == 0) rc = check_batch(batch, pages);
    if (rc == 0) rc = check_heads(pages, n_q_heads);
    if (rc != 0) return rc;
    if (out_type != DPUF_AMD_F32 && out_type != pages->type) return -5;
    if (!(scale > 0.0f) || !isfinite(scale)) return -2;
    if (batch->n_rows == 0) return 0;
    if (!aligned(d_q, 16) || !aligned(d_out, 16) || (d_lse && !aligned(d_lse, 4))) return -1;
    const size_t ws = dpuf_hip_paged_attn_workspace(batch, pages, n_q_heads, window, sink);
    if (ws > 0 && !aligned(d_workspace, 16)) return -1;
    if (workspace_bytes < ws) return -7;
    const int64_t nr = (int64_t)batch->n_rows * n_q_heads, n = nr * pages->head_dim;
    Span in[6] = {run(d_q, n, 2), pool_span(pages, pages->k), pool_span(pages, pages->v)};
    batch_spans(batch, in + 3);
    const Span out[] = {run(d_out, n, type_size(out_type)), run(d_lse, nr, 4), run(d_workspace, (int64_t)ws, 1)};
    if (any_overlap(out, 3, in, COUNT(in)) || overlap_within(out, 3)) return -1;
    const void* ps[] = {pages->k, pages->v, batch->row_start, batch->ctx_len, batch->page_table, d_q, d_out, d_lse,
                        ws > 0 ? d_workspace : NULL};
    const int32_t dev = device_of(ps, (int)(sizeof ps / sizeof ps[0]));
    if (dev < 0) return -1;
    ON_DEVICE(dev, dpuf_hip_paged_attn(hip_stream, batch, pages, n_q_heads, d_q, scale, window, sink,
                                       out_type == DPUF_AMD_F32, d_out, d_lse, ws > 0 ? d_workspace : NULL));
}

DPUF_EXPORT int32_t dpuf_amd_paged_attn(const DpufAmdBatch* batch, const DpufAmdPages* pages, int32_t n_q_heads,
                                        const void* d_q, float scale, int32_t out_type, void* d_out, float* d_lse,
                                        void* d_workspace, size_t workspace_bytes, void* hip_stream) {
    return paged_attn(batch, pages, n_q_heads, d_q, scale, 0, 0, out_type, d_out, d_lse, d_workspace, workspace_bytes,
                      hip_stream);
}

DPUF_EXPORT int32_t dpuf_amd_paged_attn_window(const DpufAmdBatch* batch, const DpufAmdPages* pages, int32_t n_q_heads,
                                               const void* d_q, float scale, int32_t window, int32_t sink,
                                               int32_t out_type, void* d_out, float* d_lse, void* d_workspace,
                                               size_t workspace_bytes, void* hip_stream) {
    if (!window_ok(window, sink)) return -2;
    return paged_attn(batch, pages, n_q_heads, d_q, scale, window, sink, out_type, d_out, d_lse, d_workspace,
                      workspace_bytes, hip_stream);
}

DPUF_EXPORT int32_t dpuf_amd_paged_attn_weights(const DpufAmdBatch* batch, const DpufAmdPages* pages,
                                                int32_t n_q_heads, const void* d_q, float scale, const float* d_lse,
                                                float decay, const float* d_w_in, void* hip_stream) {
    dpuf_hip_clear_error();
    int32_t rc = check_pages(pages);
    if (rc == 0) rc = check_batch(batch, pages);
    if (rc == 0) rc = check_heads(pages, n_q_heads);
    if (rc != 0) return rc;
    if (!(scale > 0.0f) || !isfinite(scale) || !isfinite(decay)) return -2;
    if (!aligned(pages->w, 4) || (d_w_in && !aligned(d_w_in, 4))) return -1;
    if (batch->n_rows > 0 && (!aligned(d_q, 16) || !aligned(d_lse, 4))) return -1;
    const int64_t nr = (int64_t)batch->n_rows * n_q_heads;
    Span in[6] = {run(d_q, nr * pages->head_dim, 2), run(d_lse, nr, 4), pool_span(pages, pages->k)};
    batch_spans(batch, in + 3);
    const Span w = weight_span(pages, pages->w), w_in = weight_span(pages, d_w_in);
    if (any_overlap(&w, 1, in, COUNT(in)) || (d_w_in != pages->w && overlap(w, w_in))) return -1;
    const void* ps[] = {pages->k, pages->w, batch->row_start, batch->ctx_len, batch->page_table, d_w_in,
                        batch->n_rows > 0 ? d_q : NULL, batch->n_rows > 0 ? (const void*)d_lse : NULL};
    const int32_t dev = device_of(ps, (int)(sizeof ps / sizeof ps[0]));
    if (dev < 0) return -1;
    ON_DEVICE(dev, dpuf_hip_paged_attn_weights(hip_stream, batch, pages, n_q_heads, d_q, scale, d_lse, decay, d_w_in));
}

DPUF_EXPORT int32_t dpuf_amd_paged_evict(const DpufAmdBatch* batch, const DpufAmdPages* pages, int32_t keep,
                                         int32_t sink, int32_t recent, const DpufAmdPages* dst,
                                         const int32_t* d_dst_table, int32_t dst_table_stride, int32_t* d_kept,
                                         int32_t* d_new_len, void* hip_stream) {
    dpuf_hip_clear_error();
    int32_t rc = check_pages(pages);
    if (rc == 0) rc = check_pages(dst);
    if (rc == 0 && !batch) rc = -1;
    if (rc != 0) return rc;
    DpufAmdBatch b = *batch;    /* without new rows */
    b.row_start = b.ctx_len;
    b.n_rows = 0;
    rc = check_batch(&b, pages);
    if (rc != 0) return rc;
    if (dst->type != pages->type || dst->head_dim != pages->head_dim) return -5;
    if (dst->n_kv_heads != pages->n_kv_heads) return -2;
    if (keep < 1 || sink < 0 || recent < 0 || (int64_t)sink + recent > keep) return -2;
    if (dst_table_stride < 1 || (int64_t)dst_table_stride * dst->page_size > (int64_t)1 << 30 ||
        keep > (int64_t)dst_table_stride * dst->page_size)
        return -2;
    if (!aligned(pages->w, 4) || !aligned(dst->w, 4) || !aligned(d_dst_table, 4) || !aligned(d_kept, 4) ||
        !aligned(d_new_len, 4))
        return -1;
    const int64_t ns = batch->n_seqs;
    const Span in[] = {run(batch->ctx_len, ns, 4), run(batch->page_table, ns * batch->table_stride, 4),
                       run(d_dst_table, ns * dst_table_stride, 4)};
    const Span lists[] = {run(d_kept, ns * pages->n_kv_heads * keep, 4), run(d_new_len, ns, 4)};
    /* dst may be other pages of the same pool */
    const Span from[] = {pool_span(pages, pages->k), pool_span(pages, pages->v), weight_span(pages, pages->w)};
    const Span to[] = {pool_span(dst, dst->k), pool_span(dst, dst->v), weight_span(dst, dst->w)};
    if (any_overlap(lists, 2, in, 3) || overlap(lists[0], lists[1]) || any_overlap(lists, 2, from, 3) ||
        any_overlap(lists, 2, to, 3) || any_overlap(to, 3, in, 3) || any_overlap(to, 2, from + 2, 1) ||
        any_overlap(to + 2, 1, from, 2) || any_overlap(to, 2, to + 2, 1))
        return -1;
    const void* ps[] = {pages->k, pages->v, pages->w, dst->k, dst->v, dst->w, batch->ctx_len, batch->page_table,
                        d_dst_table, d_kept, d_new_len};
    const int32_t dev = device_of(ps, (int)(sizeof ps / sizeof ps[0]));
    if (dev < 0) return -1;
    ON_DEVICE(dev, dpuf_hip_paged_evict(hip_stream, &b, pages, keep, sink, recent, dst, d_dst_table,
                                        dst_table_stride, d_kept, d_new_len));
}

DPUF_EXPORT size_t dpuf_amd_sample_workspace(int32_t n, int32_t V) {
    if (n < 1 || n > MAX_ROWS || V < 1 || V > DPUF_AMD_SAMPLE_MAX_VOCAB) return 0;
    return dpuf_hip_sample_workspace(n, V);
}

DPUF_EXPORT int32_t dpuf_amd_sample(int32_t type, int32_t n, int32_t V, int64_t row_stride, const void* d_logits,
                                    const float* d_temperature, const int32_t* d_top_k, const float* d_top_p,
                                    const float* d_min_p, const float* d_u, int32_t* d_tokens, float* d_logprobs,
                                    void* d_workspace, size_t workspace_bytes, void* hip_stream) {
    dpuf_hip_clear_error();
    if (type != DPUF_AMD_F32 && type != DPUF_AMD_BF16 && type != DPUF_AMD_F16) return -5;
    if (n < 1 || n > MAX_ROWS || V < 1 || V > DPUF_AMD_SAMPLE_MAX_VOCAB) return -2;
    if (row_stride < V) return -4;
    if (!aligned(d_logits, (uintptr_t)type_size(type)) || !aligned(d_u, 4) || !aligned(d_tokens, 4)) return -1;
    const void* opt[] = {d_temperature, d_top_k, d_top_p, d_min_p, d_logprobs};
    for (int i = 0; i < 5; i++)
        if (opt[i] && !aligned(opt[i], 4)) return -1;
    const size_t ws = dpuf_hip_sample_workspace(n, V);
    if (ws > 0 && !aligned(d_workspace, 16)) return -1;
    if (workspace_bytes < ws) return -7;
    const Span in[] = {rows_of(d_logits, n, row_stride, V, type_size(type)), run(d_temperature, n, 4), run(d_top_k, n, 4),
                       run(d_top_p, n, 4), run(d_min_p, n, 4), run(d_u, n, 4)};
    const Span out[] = {run(d_tokens, n, 4), run(d_logprobs, n, 4), run(d_workspace, (int64_t)ws, 1)};
    if (any_overlap(out, 3, in, COUNT(in)) || overlap_within(out, 3)) return -1;
    const void* ps[] = {d_logits, d_temperature, d_top_k, d_top_p, d_min_p, d_u, d_tokens, d_logprobs,
                        ws > 0 ? d_workspace : NULL};
    const int32_t dev = device_of(ps, (int)(sizeof ps / sizeof ps[0]));
    if (dev < 0) return -1;
    ON_DEVICE(dev, dpuf_hip_sample(hip_stream, type, n, V, row_stride, d_logits, d_temperature, d_top_k, d_top_p,
                                   d_min_p, d_u, d_tokens, d_logprobs, d_workspace));
}

DPUF_EXPORT size_t dpuf_amd_logprobs_workspace(int32_t n, int32_t V, int32_t n_top) {
    if (n < 1 || n > MAX_ROWS || V < 1 || V > DPUF_AMD_SAMPLE_MAX_VOCAB || n_top < 0 ||
        n_top > DPUF_AMD_LOGPROBS_MAX_TOP)
        return 0;
    return dpuf_hip_logprobs_workspace(n, V, n_top);
}

DPUF_EXPORT int32_t dpuf_amd_logprobs(int32_t type, int32_t n, int32_t V, int64_t row_stride, const void* d_logits,
                                      int32_t n_targets, const int32_t* d_targets, int32_t n_top, float* d_logprobs,
                                      float* d_entropy, int32_t* d_top_tokens, float* d_top_logprobs,
                                      void* d_workspace, size_t workspace_bytes, void* hip_stream) {
    dpuf_hip_clear_error();
    if (type != DPUF_AMD_F32 && type != DPUF_AMD_BF16 && type != DPUF_AMD_F16) return -5;
    if (n < 1 || n > MAX_ROWS || V < 1 || V > DPUF_AMD_SAMPLE_MAX_VOCAB || n_targets < 0 ||
        n_targets > DPUF_AMD_LOGPROBS_MAX_TARGETS || n_top < 0 || n_top > DPUF_AMD_LOGPROBS_MAX_TOP)
        return -2;
    if (row_stride < V) return -4;
    if ((n_targets == 0) != (d_targets == NULL) || (n_targets == 0) != (d_logprobs == NULL) ||
        (n_top == 0) != (d_top_tokens == NULL) || (n_top == 0) != (d_top_logprobs == NULL) ||
        (n_targets == 0 && n_top == 0 && !d_entropy))
        return -1;
    if (!aligned(d_logits, (uintptr_t)type_size(type))) return -1;
    const void* opt[] = {d_targets, d_logprobs, d_entropy, d_top_tokens, d_top_logprobs};
    for (int i = 0; i < COUNT(opt); i++)
        if (opt[i] && !aligned(opt[i], 4)) return -1;
    const size_t ws = dpuf_hip_logprobs_workspace(n, V, n_top);
    if (ws > 0 && !aligned(d_workspace, 16)) return -1;
    if (workspace_bytes < ws) return -7;
    const Span in[] = {rows_of(d_logits, n, row_stride, V, type_size(type)), run(d_targets, (int64_t)n * n_targets, 4)};
    const Span out[] = {run(d_logprobs, (int64_t)n * n_targets, 4), run(d_entropy, n, 4),
                        run(d_top_tokens, (int64_t)n * n_top, 4), run(d_top_logprobs, (int64_t)n * n_top, 4),
                        run(d_workspace, (int64_t)ws, 1)};
    if (any_overlap(out, COUNT(out), in, COUNT(in)) || overlap_within(out, COUNT(out))) return -1;
    const void* ps[] = {d_logits, d_targets, d_logprobs, d_entropy, d_top_tokens, d_top_logprobs,
                        ws > 0 ? d_workspace : NULL};
    const int32_t dev = device_of(ps, COUNT(ps));
    if (dev < 0) return -1;
    ON_DEVICE(dev, dpuf_hip_logprobs(hip_stream, type, n, V, row_stride, d_logits, n_targets, d_targets, n_top,
                                     d_logprobs, d_entropy, d_top_tokens, d_top_logprobs, ws > 0 ? d_workspace : NULL));
}
