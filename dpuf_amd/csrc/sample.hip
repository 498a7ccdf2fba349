// sample.hip -- one token from a row of logits with temperature, top-k, top-p
// and min-p, drawn with a given uniform number.
//
// With M the row's largest logit, the weight of token i is
//     w_i = rint(2^S exp((x_i - M) / T)),  S = 62 - ceil(log2 V),
// a 64-bit integer: the V weights of a row sum below 2^63, sums of them are
// the same in any order (LDS atomics included), and a token whose weight
// rounds to 0 has less than 2^-38 of the largest token's.  Such tokens can
// never be drawn, so they are dropped at once: what is left lies within
// A = (S + 1) ln 2 temperatures of M.
//
// The order "larger logit first, then lower index" is that of the integers
// c_i = (order-preserving bits of x_i) << 32 | (2^32 - 1 - i).  Top-k, top-p
// and min-p each keep a prefix of it, so together they keep the shortest.
//
// A row is cut into chunks, one workgroup each, in three launches:
//   k_smp_max   the chunks' largest logits;
//   k_smp_hist  tokens and weight in each of NB bins of (M - x) / T per chunk
//               (only the sum where neither top-k nor top-p is on); the
//               workgroup that ends last adds the chunks' bins up and finds
//               the bins in which the prefixes end;
//   k_smp_pick  collects the tokens that decide: all of the prefix's where
//               they fit, else those of the bins the borders lie in; the
//               workgroup that ends last sorts them, finds the border and
//               draws, from the list or, in index order, from the chunk in
//               which the running sum passes the draw.
// Rows whose border bin alone holds more tokens than can be sorted (long runs
// of equal logits) are left to one workgroup that splits the bin further.
//
// The last workgroup is found with a counter per row; what it reads from the
// others was stored past the L2 of their XCD (agent scope) and acknowledged
// before they counted, and it reads past its own.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hip_internal.h"
#include "paged.h"

namespace {

constexpr int NT = 256;          // threads of a workgroup
constexpr int NW = NT / 64;
constexpr int NB = 1024;         // bins
constexpr int CAP = 2048;        // tokens sorted in LDS
constexpr int ROWS = 1024;       // rows of one set of launches
constexpr int MAX_CHUNKS = 64;   // a wave's lanes take a row's chunks

enum { SM_DONE = 0, SM_PLAIN, SM_LIST, SM_BINS, SM_SPLIT };

struct SmState {
    unsigned tick[2], n_list;
    int mode;
    int by_k, by_p, by_m;        // settings that cut something
    int last;                    // SM_LIST: the last bin whose tokens are listed
    int bk, pl, ph, ml, mh;      // border bins: top-k's, top-p's and min-p's first and last
    unsigned rk;                 // tokens of bin bk that top-k keeps
    unsigned long long wk, wp;   // weight in the bins above bk, above pl
    unsigned long long total;    // weight of the whole row
};

struct SmArgs {
    const void* x;
    int64_t stride;
    int V, S, vec, chunk, chunks;
    const float* temp;
    const int* top_k;
    const float *top_p, *min_p, *u;
    int* tok;
    float* logp;
    uint64_t *best, *csum, *wsum, *list;
    uint32_t* count;
    SmState* state;
};

struct F32L {
    static constexpr int VE = 4, SIZE = 4;
    static DEV float one(const void* p, int64_t i) { return ((const float*)p)[i]; }
    static DEV void many(const void* p, int64_t i, float* o) {
        const float4 v = *(const float4*)((const float*)p + i);
        o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
    }
};
template <typename T> struct H16L {
    static constexpr int VE = 8, SIZE = 2;
    static DEV float one(const void* p, int64_t i) { return (float)((const typename T::e*)p)[i]; }
    static DEV void many(const void* p, int64_t i, float* o) {
        const typename T::v8 v = vec_of<typename T::v8>(*(const u32x4*)((const uint16_t*)p + i));
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (float)v[e];
    }
};

DEV void put_agent(uint64_t* p, uint64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DEV uint64_t get_agent(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

DEV uint32_t order_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);      // -0 and +0 are one value
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
DEV float from_bits(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
DEV uint64_t comp_of(float x, int i) { return (uint64_t)order_bits(x) << 32 | (0xffffffffu - (uint32_t)i); }
DEV float logit_of(uint64_t c) { return from_bits((uint32_t)(c >> 32)); }
DEV int index_of(uint64_t c) { return (int)(0xffffffffu - (uint32_t)c); }

// 2^s exp(-a) for 0 <= a < 64: exp(-a) = 2^-n exp(r) with n = rint(a / ln 2) and
// r = n ln 2 - a, by the Taylor series of exp up to r^13 / 13! (|r| <= ln 2 / 2:
// what is left out is below 2^-56).
DEV double exp_neg(double a, int s) {
    const double n = rint(a * 1.4426950408889634074);
    // ln 2 in two parts, the first of 40 bits: n times it is exact
    double r = fma(n, 0x1.62e42fefa2000p-1, -a);
    r = fma(n, 0x1.9ef35793c7673p-41, r);
    double e = 1.0 / 6227020800.0;
    e = fma(e, r, 1.0 / 479001600.0);
    e = fma(e, r, 1.0 / 39916800.0);
    e = fma(e, r, 1.0 / 3628800.0);
    e = fma(e, r, 1.0 / 362880.0);
    e = fma(e, r, 1.0 / 40320.0);
    e = fma(e, r, 1.0 / 5040.0);
    e = fma(e, r, 1.0 / 720.0);
    e = fma(e, r, 1.0 / 120.0);
    e = fma(e, r, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    return ldexp(e, s - (int)n);
}

// f(token, logit) for the tokens [lo, hi) of a row, in no particular order; lo
// is a multiple of 8.
template <typename L, typename F> DEV void each(const void* p, int vec, int lo, int hi, F f) {
    constexpr int VE = L::VE, U = 16 / VE;
    int done = lo;
    if (vec) {
        const int v1 = hi / VE;
        for (int v0 = lo / VE + threadIdx.x; v0 < v1; v0 += NT * U) {
            float x[U][VE];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = v0 + u * NT;
                L::many(p, (int64_t)(v < v1 ? v : v0) * VE, x[u]);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = v0 + u * NT;
                if (v < v1)
#pragma unroll
                    for (int e = 0; e < VE; e++) f(v * VE + e, x[u][e]);
            }
        }
        done = v1 * VE > lo ? v1 * VE : lo;
    }
    for (int i = done + threadIdx.x; i < hi; i += NT) f(i, L::one(p, i));
}

// A row with its settings.
template <typename L> struct Row {
    const void* p;
    int V, S, vec;
    float M;
    double invT, A, p_goal;
    float bins;                  // bins per temperature
    int k, by_k, by_p, by_m;
    double min_p, edge;          // min_p and -ln min_p

    // (M - x) / T, or infinity for tokens that cannot be drawn
    DEV double depth(float x) const {
        const double d = (double)M - (double)x;
        return x == M ? 0.0 : d < __builtin_huge_val() ? d * invT : __builtin_huge_val();
    }
    DEV uint64_t weight(double a) const { return a < A ? (uint64_t)(exp_neg(a, S) + 0.5) : 0; }
    DEV uint64_t weight_of(uint64_t c) const { return weight(depth(logit_of(c))); }
    DEV int bin(double a) const {
        const int b = (int)((float)a * bins);
        return b < NB - 1 ? b : NB - 1;
    }
    // a token with a weight: only the last bin's need the exponential to tell
    DEV bool alive(double a, int b) const { return a < A && (b < NB - 1 || weight(a) != 0); }
    DEV bool above_min(double a) const { return !by_m || exp_neg(a, 0) >= min_p; }

    DEV void open(const SmArgs& a, int r) {
        p = (const char*)a.x + r * a.stride * L::SIZE;
        V = a.V;
        S = a.S;
        vec = a.vec;
    }
    // The settings of row r with largest logit m; false where the row needs
    // no weights (nothing above -infinity, or greedy).
    DEV bool set(const SmArgs& a, int r, uint64_t best) {
        M = logit_of(best);
        const float T = a.temp ? a.temp[r] : 1.0f;
        if (best == 0 || M == -__builtin_huge_valf() || !(T > 0.0f)) return false;
        invT = 1.0 / (double)T;
        A = (S + 1) * 0.69314718055994530942;
        bins = (float)(NB / A);
        k = a.top_k ? a.top_k[r] : 0;
        by_k = k > 0 && k < V;
        const float tp = a.top_p ? a.top_p[r] : 1.0f, mp = a.min_p ? a.min_p[r] : 0.0f;
        by_p = tp < 1.0f;
        p_goal = tp > 0.0f ? (double)tp : 0.0;
        min_p = mp > 1.0f ? 1.0 : mp > 0.0f ? (double)mp : 0.0;
        edge = min_p > 0.0 ? -log(min_p) : 0.0;
        by_m = min_p > 0.0 && edge < A;
        return true;
    }
    // Top-p's goal for a total: one token at least.
    DEV double goal(uint64_t total) const { return fmax(p_goal * (double)total, 0.5); }
};

// The row's largest composite from its chunks'.
DEV uint64_t row_best(const SmArgs& a, int r) {
    const int lane = threadIdx.x & 63;
    uint64_t b = lane < a.chunks ? a.best[(size_t)r * a.chunks + lane] : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)b, d), hi = __shfl_xor((uint32_t)(b >> 32), d);
        const uint64_t o = (uint64_t)hi << 32 | lo;
        b = o > b ? o : b;
    }
    return b;
}

DEV uint64_t shfl_up64(uint64_t v, int d) {
    const uint32_t lo = __shfl_up((uint32_t)v, d), hi = __shfl_up((uint32_t)(v >> 32), d);
    return (uint64_t)hi << 32 | lo;
}

// Inclusive sum over the workgroup's threads; *total gets the sum of all.
DEV uint64_t scan64(uint64_t* red, uint64_t v, uint64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = shfl_up64(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 63) red[wave] = v;
    __syncthreads();
    uint64_t base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
        if (w == wave) base = all;
        all += red[w];
    }
    *total = all;
    return v + base;
}

// Whether this workgroup is the last of `of` to get here; what the others
// stored with put_agent before can then be read with get_agent.
DEV bool last_here(unsigned* tick, int of, int* sh) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this thread's stores are acknowledged
    __syncthreads();
    if (threadIdx.x == 0)
        *sh = of == 1 || __hip_atomic_fetch_add(tick, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1u;
    __syncthreads();
    return *sh != 0;
}

// Draw number of a row: the token whose running sum passes it.
DEV uint64_t aim_of(float u, uint64_t total) {
    const uint64_t t = u > 0.0f ? (uint64_t)((double)(u < 1.0f ? u : 1.0f) * (double)total) : 0;
    return t < total ? t : total - 1;
}
template <typename L> DEV void answer(const SmArgs& a, const Row<L>& row, int r, int tok, float x, uint64_t total) {
    a.tok[r] = tok;
    if (a.logp) a.logp[r] = (float)(-row.depth(x) - log((double)total / (double)(1ull << row.S)));
}

// ---------------------------------------------------------------------------
template <typename L> __global__ __launch_bounds__(NT) void k_smp_max(SmArgs a) {
    __shared__ uint64_t red[NW];
    const int r = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
    Row<L> row;
    row.open(a, r);
    if (c == 0 && t == 0) {
        a.state[r].tick[0] = a.state[r].tick[1] = 0;
        a.state[r].n_list = 0;
    }
    float m = -__builtin_huge_valf();
    int at = -1;
    each<L>(row.p, row.vec, c * a.chunk, min(a.V, (c + 1) * a.chunk), [&](int i, float x) {
        if (x > m) {
            m = x;
            at = i;
        }
    });
    uint64_t b = at >= 0 ? comp_of(m, at) : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)b, d), hi = __shfl_xor((uint32_t)(b >> 32), d);
        const uint64_t o = (uint64_t)hi << 32 | lo;
        b = o > b ? o : b;
    }
    if ((t & 63) == 0) red[t >> 6] = b;
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < NW; w++) b = red[w] > b ? red[w] : b;
        a.best[(size_t)r * a.chunks + c] = b;
    }
}

// ---------------------------------------------------------------------------
struct HistShared {
    unsigned long long wsum[NB];
    uint32_t count[NB];
    uint64_t red[NW];
    uint64_t v0, v1;
    int flag, b;
};

// Finds the border bins from the row's bins (in sh, all chunks added up).
template <typename L> DEV void find_borders(const SmArgs& a, HistShared& sh, const Row<L>& row, SmState* st) {
    constexpr int PER = NB / NT;
    const int t = threadIdx.x;
    uint64_t c = 0, w = 0, tc, tw;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        c += sh.count[PER * t + e];
        w += sh.wsum[PER * t + e];
    }
    const uint64_t c0 = scan64(sh.red, c, &tc) - c, w0 = scan64(sh.red, w, &tw) - w;
    __shared__ int bk, pl, ph;
    __shared__ uint64_t nk, wk, wp;
    if (t == 0) {
        bk = pl = ph = -1;
        nk = wk = wp = 0;
    }
    __syncthreads();
    if (row.by_k) {
        uint64_t n = c0, s = w0;
#pragma unroll
        for (int e = 0; e < PER; e++) {
            const int b = PER * t + e;
            if (n < (uint64_t)row.k && n + sh.count[b] >= (uint64_t)row.k) {
                bk = b;
                nk = n;
                wk = s;
            }
            n += sh.count[b];
            s += sh.wsum[b];
        }
    }
    __syncthreads();
    const bool by_k = bk >= 0;       // fewer tokens than k: all stay
    if (row.by_p) {
        // the weight that top-k leaves lies between these
        const double g0 = row.goal(by_k ? wk : tw), g1 = row.goal(by_k ? wk + sh.wsum[bk] : tw);
        uint64_t s = w0;
#pragma unroll
        for (int e = 0; e < PER; e++) {
            const int b = PER * t + e;
            const uint64_t s1 = s + sh.wsum[b];
            if ((double)s < g0 && (double)s1 >= g0) {
                pl = b;
                wp = s;
            }
            if ((double)s < g1 && (double)s1 >= g1) ph = b;
            s = s1;
        }
    }
    __syncthreads();
    const bool by_p = pl >= 0 && ph >= 0;
    const int ml = row.by_m ? row.bin(row.edge * (1.0 - 1e-9)) : -1, mh = row.by_m ? row.bin(row.edge * (1.0 + 1e-9)) : -1;
    const int last = by_k ? bk : by_p ? ph : NB - 1;
    uint64_t n_up = 0, n_s = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int b = PER * t + e;
        if (b <= last) n_up += sh.count[b];
        if ((by_k && b == bk) || (by_p && b >= pl && b <= ph) || (row.by_m && b >= ml && b <= mh)) n_s += sh.count[b];
    }
    uint64_t a_up, a_s;
    scan64(sh.red, n_up, &a_up);
    scan64(sh.red, n_s, &a_s);
    if (t == 0) {
        st->by_k = by_k;
        st->by_p = by_p;
        st->by_m = row.by_m;
        st->last = last;
        st->bk = bk;
        st->pl = pl;
        st->ph = ph;
        st->ml = ml;
        st->mh = mh;
        st->rk = by_k ? (unsigned)((uint64_t)row.k - nk) : 0;
        st->wk = wk;
        st->wp = wp;
        st->total = tw;
        st->mode = a_up <= CAP ? SM_LIST : a_s <= CAP ? SM_BINS : SM_SPLIT;
    }
}

template <typename L> __global__ __launch_bounds__(NT) void k_smp_hist(SmArgs a) {
    __shared__ HistShared sh;
    const int r = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
    SmState* st = a.state + r;
    Row<L> row;
    row.open(a, r);
    const uint64_t best = row_best(a, r);
    if (!row.set(a, r, best)) {
        if (c == 0 && t == 0) {
            const bool none = best == 0 || logit_of(best) == -__builtin_huge_valf();
            a.tok[r] = none ? -1 : index_of(best);
            if (a.logp) a.logp[r] = none ? -__builtin_huge_valf() : 0.0f;
            st->mode = SM_DONE;
        }
        return;
    }
    const int lo = c * a.chunk, hi = min(a.V, lo + a.chunk);
    if (!row.by_k && !row.by_p) {
        uint64_t s = 0, all;
        each<L>(row.p, row.vec, lo, hi, [&](int, float x) {
            const double d = row.depth(x);
            if (row.above_min(d)) s += row.weight(d);
        });
        scan64(sh.red, s, &all);
        if (t == 0) {
            a.csum[(size_t)r * a.chunks + c] = all;
            if (c == 0) st->mode = SM_PLAIN;
        }
        return;
    }
    for (int b = t; b < NB; b += NT) {
        sh.count[b] = 0;
        sh.wsum[b] = 0;
    }
    __syncthreads();
    each<L>(row.p, row.vec, lo, hi, [&](int, float x) {
        const double d = row.depth(x);
        const uint64_t w = row.weight(d);
        if (w) {
            const int b = row.bin(d);
            atomicAdd(&sh.count[b], 1u);
            atomicAdd(&sh.wsum[b], (unsigned long long)w);
        }
    });
    __syncthreads();
    const size_t at = ((size_t)r * a.chunks + c) * NB;
    for (int b = t; b < NB; b += NT) put_agent(a.wsum + at + b, sh.wsum[b]);
    for (int b = t; b < NB / 2; b += NT)
        put_agent((uint64_t*)(a.count + at) + b, (uint64_t)sh.count[2 * b + 1] << 32 | sh.count[2 * b]);
    if (!last_here(&st->tick[0], a.chunks, &sh.flag)) return;
    if (a.chunks > 1) {
        constexpr int PER = NB / NT;
        const uint64_t* cp = (const uint64_t*)(a.count + (size_t)r * a.chunks * NB) + PER / 2 * t;
        const uint64_t* wp = a.wsum + (size_t)r * a.chunks * NB + PER * t;
        uint64_t n[PER / 2] = {}, w[PER] = {};
#pragma unroll 4
        for (int k = 0; k < a.chunks; k++) {
            // two 32-bit sums in one word: a row has at most 2^24 tokens
#pragma unroll
            for (int e = 0; e < PER / 2; e++) n[e] += get_agent(cp + (size_t)k * (NB / 2) + e);
#pragma unroll
            for (int e = 0; e < PER; e++) w[e] += get_agent(wp + (size_t)k * NB + e);
        }
#pragma unroll
        for (int e = 0; e < PER; e++) {
            sh.count[PER * t + e] = (uint32_t)(n[e / 2] >> (32 * (e & 1)));
            sh.wsum[PER * t + e] = w[e];
        }
        __syncthreads();
    }
    find_borders(a, sh, row, st);
}

// ---------------------------------------------------------------------------
struct PickShared {
    uint64_t list[CAP], lw[CAP];
    unsigned long long wsum[NB];
    uint32_t count[NB];
    uint64_t red[NW];
    uint64_t b0, b1;
    int i0, i1, flag;
    uint32_t n_list;
};

// Descending sort of sh.list[0, n): short lists by counting the larger ones
// (the composites differ), longer ones bitonic.
DEV void sort_desc(PickShared& sh, int n) {
    __syncthreads();
    if (n <= 2 * NT) {
        uint64_t v[2];
        int rank[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 2; e++) v[e] = threadIdx.x + e * NT < n ? sh.list[threadIdx.x + e * NT] : 0;
        for (int j = 0; j < n; j++) {
            const uint64_t o = sh.list[j];
            rank[0] += o > v[0];
            rank[1] += o > v[1];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; e++)
            if (threadIdx.x + e * NT < n) sh.list[rank[e]] = v[e];
        __syncthreads();
        return;
    }
    int n2 = 1;
    while (n2 < n) n2 <<= 1;
    for (int i = n + threadIdx.x; i < n2; i += NT) sh.list[i] = 0;
    for (int k = 2; k <= n2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < n2 / 2; i += NT) {
                const int x = (i & ~(j - 1)) << 1 | (i & (j - 1)), y = x | j;
                const uint64_t p = sh.list[x], q = sh.list[y];
                if ((p < q) == !(x & k)) {
                    sh.list[x] = q;
                    sh.list[y] = p;
                }
            }
        }
    __syncthreads();
}

// What a prefix search looks for: the first `count` tokens, or the shortest
// prefix whose weights reach `goal`.
struct Want {
    uint64_t count;
    double goal;
    bool by_weight;
    DEV bool met(uint64_t n, uint64_t w) const { return by_weight ? (double)w >= goal : n >= count; }
};

// Position in sh.list[i0, i1) (sorted) at which a prefix with n0 tokens and w0
// weight before it meets `want`, and *sum the weight up to and with it; i1 - 1
// where it does not.
template <typename L>
DEV int walk(PickShared& sh, const Row<L>& row, const Want& want, int i0, int i1, uint64_t n0, uint64_t w0,
             uint64_t* sum) {
    constexpr int PER = CAP / NT;
    const int t = threadIdx.x;
    uint64_t w[PER], tot = 0, all;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int at = i0 + PER * t + e;
        w[e] = at < i1 ? row.weight_of(sh.list[at]) : 0;
        tot += w[e];
    }
    uint64_t s = scan64(sh.red, tot, &all) - tot + w0;
    if (t == 0) {
        sh.i0 = i1 - 1;
        sh.b0 = w0 + all;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int at = i0 + PER * t + e;
        const uint64_t n = n0 + PER * t + e;
        if (at < i1 && !want.met(n, s) && want.met(n + 1, s + w[e])) {
            sh.i0 = at;
            sh.b0 = s + w[e];
        }
        s += w[e];
    }
    __syncthreads();
    const int at = sh.i0;
    *sum = sh.b0;
    __syncthreads();
    return at;
}

// Draws from the sorted list's first m tokens, in index order.
template <typename L> DEV void draw_list(const SmArgs& a, PickShared& sh, const Row<L>& row, int r, int m) {
    const int t = threadIdx.x;
    uint64_t own = 0, total;
    for (int i = t; i < m; i += NT) {
        sh.lw[i] = row.weight_of(sh.list[i]);
        own += sh.lw[i];
    }
    scan64(sh.red, own, &total);
    __syncthreads();
    const uint64_t aim = aim_of(a.u[r], total);
    if (m <= 2 * NT) {
        // a token's running sum: the weights of the kept ones before it
        for (int i = t; i < m; i += NT) {
            const uint32_t me = (uint32_t)sh.list[i];       // larger for earlier tokens
            uint64_t before = 0;
            for (int j = 0; j < m; j++) before += (uint32_t)sh.list[j] > me ? sh.lw[j] : 0;
            if (before <= aim && aim < before + sh.lw[i])
                answer(a, row, r, index_of(sh.list[i]), logit_of(sh.list[i]), total);
        }
        return;
    }
    for (int i = t; i < m; i += NT) sh.list[i] = sh.list[i] << 32 | sh.list[i] >> 32;
    sort_desc(sh, m);
    constexpr int PER = CAP / NT;
    uint64_t w[PER], tot = 0, all;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int at = PER * t + e;
        w[e] = at < m ? row.weight(row.depth(from_bits((uint32_t)sh.list[at]))) : 0;
        tot += w[e];
    }
    uint64_t s = scan64(sh.red, tot, &all) - tot;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int at = PER * t + e;
        if (s <= aim && aim < s + w[e])
            answer(a, row, r, index_of(sh.list[at] >> 32), from_bits((uint32_t)sh.list[at]), total);
        s += w[e];
    }
}

// The token of [lo, hi) whose running sum of kept(token, logit), `base` before
// lo, passes aim: every wave sums a run, then all walk the run that holds it.
template <typename L, typename F>
DEV void draw_range(const SmArgs& a, PickShared& sh, const Row<L>& row, int r, int lo, int hi, uint64_t base,
                    uint64_t aim, uint64_t total, F kept) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int run = (hi - lo + NW - 1) / NW, r0 = lo + wave * run, r1 = min(r0 + run, hi);
    uint64_t s = 0;
    for (int i = r0 + lane; i < r1; i += 64) s += kept(i, L::one(row.p, i));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = shfl_up64(s, d);
        if (lane >= d) s += o;
    }
    __syncthreads();
    if (lane == 63) sh.red[wave] = s;
    __syncthreads();
    int w0 = 0;
    while (w0 < NW - 1 && base + sh.red[w0] <= aim) base += sh.red[w0++];
    const int s0 = lo + w0 * run, s1 = min(s0 + run, hi);
    const int per = (run + NT - 1) / NT, i0 = min(s0 + t * per, s1), i1 = min(i0 + per, s1);
    uint64_t own = 0, all;
    for (int i = i0; i < i1; i++) own += kept(i, L::one(row.p, i));
    const uint64_t end = scan64(sh.red, own, &all) + base;
    if (own && end > aim && end - own <= aim) {
        uint64_t at = end - own;
        for (int i = i0; i < i1; i++) {
            const float x = L::one(row.p, i);
            at += kept(i, x);
            if (at > aim) {
                answer(a, row, r, i, x, total);
                break;
            }
        }
    }
}

// The chunk in which the running sum of the chunks' sums (lane c: chunk c's)
// passes the draw.
DEV int pick_chunk(uint64_t sum, float u, uint64_t* base, uint64_t* aim, uint64_t* total) {
    const int lane = threadIdx.x & 63;
    uint64_t s = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = shfl_up64(s, d);
        if (lane >= d) s += o;
    }
    const uint32_t lo = __shfl((uint32_t)s, 63), hi = __shfl((uint32_t)(s >> 32), 63);
    *total = (uint64_t)hi << 32 | lo;
    *aim = aim_of(u, *total);
    const int c = __ffsll((unsigned long long)__ballot(s > *aim)) - 1;
    const uint64_t b = s - sum;
    *base = (uint64_t)__shfl((uint32_t)(b >> 32), c) << 32 | __shfl((uint32_t)b, c);
    return c;
}

// ---------------------------------------------------------------------------
// A row by one workgroup, for borders in runs too long to sort: the bin's
// composites, which differ, are split into NB ranges until one fits.
// ---------------------------------------------------------------------------
DEV bool find_bin(PickShared& sh, const Want& want, uint64_t n0, uint64_t w0, int* bin, uint64_t* bn, uint64_t* bw) {
    constexpr int PER = NB / NT;
    const int t = threadIdx.x;
    uint64_t c = 0, w = 0, tc, tw;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        c += sh.count[PER * t + e];
        w += sh.wsum[PER * t + e];
    }
    uint64_t n = scan64(sh.red, c, &tc) - c + n0, s = scan64(sh.red, w, &tw) - w + w0;
    if (t == 0) sh.i0 = -1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int b = PER * t + e;
        const uint64_t n1 = n + sh.count[b], s1 = s + sh.wsum[b];
        if (want.met(n1, s1) && !want.met(n, s)) {
            sh.i0 = b;
            sh.b0 = n;
            sh.b1 = s;
        }
        n = n1;
        s = s1;
    }
    __syncthreads();
    *bin = sh.i0;
    *bn = sh.b0;
    *bw = sh.b1;
    __syncthreads();
    return *bin >= 0;
}

// Composite of the last token of the prefix that `want` asks for among the
// tokens with composites of at least `least`; *sum gets the prefix's weight.
template <typename L>
DEV uint64_t split_cut(PickShared& sh, const Row<L>& row, const Want& want, uint64_t least, uint64_t* sum) {
    const int t = threadIdx.x;
    uint64_t lo = least, hi = ~0ull, bn = 0, bw = 0;
    for (;;) {
        int sf = 0;
        while (((hi - lo) >> sf) >= NB) sf++;
        __syncthreads();
        for (int b = t; b < NB; b += NT) {
            sh.count[b] = 0;
            sh.wsum[b] = 0;
        }
        __syncthreads();
        each<L>(row.p, row.vec, 0, row.V, [&](int i, float x) {
            const uint64_t w = row.weight(row.depth(x)), c = comp_of(x, i);
            if (w && c >= lo && c <= hi) {
                atomicAdd(&sh.count[(hi - c) >> sf], 1u);
                atomicAdd(&sh.wsum[(hi - c) >> sf], (unsigned long long)w);
            }
        });
        __syncthreads();
        int b;
        uint64_t n1, w1;
        if (!find_bin(sh, want, bn, bw, &b, &n1, &w1)) break;     // all of them: only at the first turn
        const uint32_t in = sh.count[b];
        bn = n1;
        bw = w1;
        hi -= (uint64_t)b << sf;
        const uint64_t width = (1ull << sf) - 1;
        lo = hi - lo > width ? hi - width : lo;
        __syncthreads();
        if (in > CAP) continue;
        if (t == 0) sh.n_list = 0;
        __syncthreads();
        each<L>(row.p, row.vec, 0, row.V, [&](int i, float x) {
            const uint64_t c = comp_of(x, i);
            if (c >= lo && c <= hi && row.weight(row.depth(x))) {
                const uint32_t at = atomicAdd(&sh.n_list, 1u);
                if (at < CAP) sh.list[at] = c;
            }
        });
        __syncthreads();
        const int n = min((int)sh.n_list, CAP);
        sort_desc(sh, n);
        const int at = walk(sh, row, want, 0, n, bn, bw, sum);
        return sh.list[at];
    }
    return least;
}

template <typename L> DEV void split_row(const SmArgs& a, PickShared& sh, const Row<L>& row, const SmState& st, int r) {
    uint64_t cut = 0, total = st.total;
    if (st.by_k) cut = split_cut(sh, row, Want{(uint64_t)row.k, 0.0, false}, 0, &total);
    if (st.by_p) {
        uint64_t s;
        const uint64_t c = split_cut(sh, row, Want{0, row.goal(total), true}, cut, &s);
        cut = c > cut ? c : cut;
    }
    auto kept = [&](int i, float x) -> uint64_t {
        const double d = row.depth(x);
        return comp_of(x, i) >= cut && row.above_min(d) ? row.weight(d) : 0;
    };
    uint64_t own = 0;
    each<L>(row.p, row.vec, 0, row.V, [&](int i, float x) { own += kept(i, x); });
    scan64(sh.red, own, &total);
    draw_range(a, sh, row, r, 0, row.V, 0, aim_of(a.u[r], total), total, kept);
}

template <typename L> __global__ __launch_bounds__(NT) void k_smp_pick(SmArgs a) {
    __shared__ PickShared sh;
    const int r = blockIdx.y, c = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    SmState* sp = a.state + r;
    const int mode = sp->mode;
    if (mode == SM_DONE || ((mode == SM_PLAIN || mode == SM_SPLIT) && c != 0)) return;
    Row<L> row;
    row.open(a, r);
    row.set(a, r, row_best(a, r));
    if (mode == SM_PLAIN) {
        uint64_t base, aim, total;
        const int at = pick_chunk(lane < a.chunks ? a.csum[(size_t)r * a.chunks + lane] : 0, a.u[r], &base, &aim, &total);
        draw_range(a, sh, row, r, at * a.chunk, min(a.V, (at + 1) * a.chunk), base, aim, total,
                   [&](int, float x) -> uint64_t {
                       const double d = row.depth(x);
                       return row.above_min(d) ? row.weight(d) : 0;
                   });
        return;
    }
    const SmState st = *sp;
    if (mode == SM_SPLIT) {
        split_row(a, sh, row, st, r);
        return;
    }
    // the tokens that decide
    if (t == 0) sh.n_list = 0;
    __syncthreads();
    each<L>(row.p, row.vec, c * a.chunk, min(a.V, (c + 1) * a.chunk), [&](int i, float x) {
        const double d = row.depth(x);
        if (!(d < row.A)) return;
        const int b = row.bin(d);
        const bool in = mode == SM_LIST ? b <= st.last
                                        : (st.by_k && b == st.bk) || (st.by_p && b >= st.pl && b <= st.ph) ||
                                              (st.by_m && b >= st.ml && b <= st.mh);
        if (in && row.alive(d, b)) {
            const uint32_t at = atomicAdd(&sh.n_list, 1u);
            if (at < CAP) sh.list[at] = comp_of(x, i);
        }
    });
    __syncthreads();
    int n = min((int)sh.n_list, CAP);
    uint64_t* list = a.list + (size_t)r * CAP;
    if (a.chunks > 1) {
        if (t == 0 && n > 0)
            sh.i0 = (int)__hip_atomic_fetch_add(&sp->n_list, (unsigned)n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        for (int i = t; i < n; i += NT)
            if (sh.i0 + i < CAP) put_agent(list + sh.i0 + i, sh.list[i]);
        if (!last_here(&sp->tick[1], a.chunks, &sh.flag)) return;
        n = min((int)__hip_atomic_load(&sp->n_list, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), CAP);
        __syncthreads();
        for (int i = t; i < n; i += NT) sh.list[i] = get_agent(list + i);
    }
    sort_desc(sh, n);
    uint64_t sum = st.total;
    if (mode == SM_LIST) {
        // the list holds everything top-k or top-p could keep
        int m = n;
        if (st.by_k) {
            m = walk(sh, row, Want{(uint64_t)row.k, 0.0, false}, 0, n, 0, 0, &sum) + 1;
        }
        if (st.by_p) {
            uint64_t s;
            m = min(m, walk(sh, row, Want{0, row.goal(sum), true}, 0, n, 0, 0, &s) + 1);
        }
        if (st.by_m) {
            if (t == 0) sh.i1 = 0;
            __syncthreads();
            for (int i = t; i < m; i += NT)
                if (row.above_min(row.depth(logit_of(sh.list[i])))) atomicMax(&sh.i1, i + 1);
            __syncthreads();
            m = max(1, min(m, sh.i1));
        }
        draw_list(a, sh, row, r, m);
        return;
    }
    // first list entry of a bin, or n: bins ascend along the sorted list
    auto first_of = [&](int b) -> int {
        if (t == 0) sh.i1 = n;
        __syncthreads();
        for (int i = t; i < n; i += NT)
            if (row.bin(row.depth(logit_of(sh.list[i]))) >= b) atomicMin(&sh.i1, i);
        __syncthreads();
        const int at = sh.i1;
        __syncthreads();
        return at;
    };
    int cb = NB;               // the border: bins above cb stay, and of it the composites from cc
    uint64_t cc = 0;
    auto cut_at = [&](int b, uint64_t comp) {
        if (b < cb || (b == cb && comp > cc)) {
            cb = b;
            cc = comp;
        }
    };
    if (st.by_k) {
        const int i0 = first_of(st.bk), i1 = first_of(st.bk + 1);
        const int at = walk(sh, row, Want{st.rk, 0.0, false}, i0, i1, 0, st.wk, &sum);
        cut_at(st.bk, sh.list[at]);
    }
    if (st.by_p) {
        const int i0 = first_of(st.pl), i1 = first_of(st.ph + 1);
        uint64_t s;
        const int at = walk(sh, row, Want{0, row.goal(sum), true}, i0, i1, 0, st.wp, &s);
        cut_at(row.bin(row.depth(logit_of(sh.list[at]))), sh.list[at]);
    }
    if (st.by_m) {
        const int i0 = first_of(st.ml), i1 = first_of(st.mh + 1);
        if (t == 0) sh.i0 = -1;
        __syncthreads();
        for (int i = i0 + t; i < i1; i += NT)
            if (row.above_min(row.depth(logit_of(sh.list[i])))) atomicMax(&sh.i0, i);
        __syncthreads();
        const int at = sh.i0;
        __syncthreads();
        if (at < 0) cut_at(st.ml, ~0ull);
        else cut_at(row.bin(row.depth(logit_of(sh.list[at]))), sh.list[at]);
    }
    // the chunks' sums: bins above the border, and what stays of its own
    for (int k = wave; k < a.chunks; k += NW) {
        const uint64_t* w = a.wsum + ((size_t)r * a.chunks + k) * NB;
        uint64_t s = 0;
        for (int b = lane; b < cb; b += 64) s += get_agent(w + b);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t o = shfl_up64(s, d);
            if (lane >= d) s += o;
        }
        if (lane == 63) sh.lw[k] = s;
    }
    __syncthreads();
    for (int i = t; i < n; i += NT)
        if (sh.list[i] >= cc && row.bin(row.depth(logit_of(sh.list[i]))) == cb)
            atomicAdd((unsigned long long*)&sh.lw[index_of(sh.list[i]) / a.chunk],
                      (unsigned long long)row.weight_of(sh.list[i]));
    __syncthreads();
    uint64_t base, aim, total;
    const int at = pick_chunk(lane < a.chunks ? sh.lw[lane] : 0, a.u[r], &base, &aim, &total);
    draw_range(a, sh, row, r, at * a.chunk, min(a.V, (at + 1) * a.chunk), base, aim, total,
               [&](int i, float x) -> uint64_t {
                   const double d = row.depth(x);
                   if (!(d < row.A)) return 0;
                   const int b = row.bin(d);
                   return b < cb || (b == cb && comp_of(x, i) >= cc) ? row.weight(d) : 0;
               });
}

struct SmPlan {
    int rows, chunk, chunks;
    size_t best, csum, wsum, list, count, state, bytes;
};

// Chunks of at least 4 096 tokens, as many as give about four workgroups a CU
// over all rows, 64 at most.
SmPlan plan(int n, int V) {
    SmPlan p;
    p.rows = n < ROWS ? n : ROWS;
    int c = (ROWS + p.rows - 1) / p.rows;
    if (c > MAX_CHUNKS) c = MAX_CHUNKS;
    p.chunk = ((V + c - 1) / c + 7) & ~7;
    if (p.chunk < 4096) p.chunk = 4096;
    p.chunks = (V + p.chunk - 1) / p.chunk;
    const size_t k = (size_t)p.rows * p.chunks;
    p.best = 0;
    p.csum = p.best + k * 8;
    p.wsum = p.csum + k * 8;
    p.list = p.wsum + k * NB * 8;
    p.count = p.list + (size_t)p.rows * CAP * 8;
    p.state = p.count + k * NB * 4;
    p.bytes = p.state + (size_t)p.rows * sizeof(SmState);
    return p;
}

template <typename L> void launch(const SmArgs& a, int rows, hipStream_t st) {
    const dim3 g(a.chunks, rows);
    hipLaunchKernelGGL(k_smp_max<L>, g, dim3(NT), 0, st, a);
    hipLaunchKernelGGL(k_smp_hist<L>, g, dim3(NT), 0, st, a);
    hipLaunchKernelGGL(k_smp_pick<L>, g, dim3(NT), 0, st, a);
    LAUNCHED("k_smp_max/hist/pick");
}

}  // namespace

extern "C" {

size_t dpuf_hip_sample_workspace(int32_t n, int32_t V) { return plan(n, V).bytes; }

void dpuf_hip_sample(void* s, int32_t type, int32_t n, int32_t V, int64_t stride, const void* x, const float* temp,
                     const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* tok,
                     float* logp, void* ws) {
    const SmPlan pl = plan(n, V);
    const int es = type == DPUF_AMD_F32 ? 4 : 2;
    SmArgs a;
    a.stride = stride;
    a.V = V;
    int lg = 0;
    while ((1 << lg) < V) lg++;
    a.S = 62 - lg;
    a.vec = ((uintptr_t)x & 15) == 0 && (stride * es) % 16 == 0;
    a.chunk = pl.chunk;
    a.chunks = pl.chunks;
    char* w = (char*)ws;
    a.best = (uint64_t*)(w + pl.best);
    a.csum = (uint64_t*)(w + pl.csum);
    a.wsum = (uint64_t*)(w + pl.wsum);
    a.list = (uint64_t*)(w + pl.list);
    a.count = (uint32_t*)(w + pl.count);
    a.state = (SmState*)(w + pl.state);
    for (int32_t r0 = 0; r0 < n; r0 += ROWS) {
        a.x = (const char*)x + r0 * stride * es;
        a.temp = temp ? temp + r0 : nullptr;
        a.top_k = top_k ? top_k + r0 : nullptr;
        a.top_p = top_p ? top_p + r0 : nullptr;
        a.min_p = min_p ? min_p + r0 : nullptr;
        a.u = u + r0;
        a.tok = tok + r0;
        a.logp = logp ? logp + r0 : nullptr;
        const int rows = n - r0 < ROWS ? n - r0 : ROWS;
        if (type == DPUF_AMD_F32) launch<F32L>(a, rows, ST(s));
        else if (type == DPUF_AMD_BF16) launch<H16L<Bf16>>(a, rows, ST(s));
        else launch<H16L<Fp16>>(a, rows, ST(s));
    }
}

}  // extern "C"
