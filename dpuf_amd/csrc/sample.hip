// sample.hip -- one token from a row of logits with temperature, top-k, top-p
// and min-p, drawn with a given uniform number.
//
// With M the row's largest logit, the weight of token i is
//     w_i = rint(2^S exp((x_i - M) / T)),  S = min(51, 62 - ceil(log2 V)),
// a 64-bit integer: the V weights of a row sum below 2^63, sums of them are
// the same in any order (LDS atomics included), and a token whose weight
// rounds to 0 has less than 2^-38 of the largest token's.  Such tokens can
// never be drawn, so they are dropped at once: what is left lies within
// (S + 1) ln 2 temperatures of M.
//
// The order "larger logit first, then lower index" is that of the integers
// c_i = (order-preserving bits of x_i) << 32 | (2^32 - 1 - i).  Top-k, top-p
// and min-p each keep a prefix of it, so together they keep the shortest.
//
// A row is cut into chunks, one workgroup each, in three launches:
//   k_smp_max   the chunks' largest and least logits;
//   k_smp_hist  tokens and weight in each of NB bins of M - x per chunk
//               (only the sum where neither top-k nor top-p is on); the
//               workgroup that ends last adds the chunks' bins up, groups of
//               16 first, and finds the bins in which the prefixes end;
//   k_smp_pick  collects the tokens that decide: all of the prefix's where
//               they are at most LISTED, else those of the bins the
//               borders lie in; the workgroup that ends last finds the borders
//               among them and draws, from the list or, in index order, from
//               the chunk in which the running sum passes the draw.
// Rows whose border bin alone holds more tokens than the list (long runs of
// equal logits) are left to one workgroup that splits the bin further.
//
// 64 rows of 151 936 fp32 logits with settings of every kind: 9.1, 21 and 25 us
// (bytes; 64-bit exponentials and LDS atomics; one more read, then the slowest
// row's last workgroup, about 15 us of dependent steps); one row with top-k 50
// and top-p 0.95: 3.3, 9 and 7.7, all latency, most of it loads of what other
// XCDs stored.
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
constexpr int FULL = 1000;       // of them for the tokens that surely have a weight
constexpr int GB = 16;           // bins of a group
constexpr int NG = NB / GB;      // groups: a wave's lanes
constexpr int CAP = 2048;        // tokens listed in LDS
constexpr int LISTED = 256;      // tokens ranked as they are
constexpr int ROWS = 1024;       // rows of one set of launches
constexpr int MAX_CHUNKS = 64;   // a wave's lanes take a row's chunks

enum { SM_DONE = 0, SM_PLAIN, SM_LIST, SM_BINS, SM_SPLIT };

// A row's settings.
struct Settings {
    float M;                     // the largest logit; 0 where that is infinite (then only its like are left)
    float bins;                  // bins per logit
    int inf, k, by_k, by_p, by_m;
    double invT, p_goal;
    double min_w, edge, blur;    // 2^S min_p (0: off), -T ln min_p, 2^-48 T
};

struct SmState {
    Settings set;
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
    // csum: weight of each chunk's quarters; gsum: weight, tokens of each group of bins
    uint64_t *best, *csum, *wsum, *gsum, *list;
    uint32_t* count;
    float* least;
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

// 2^S exp(-a) = 2^(S - y / 16) exp(r) with y = rint(16 a / ln 2) and r = y ln 2 /
// 16 - a: the sixteenth powers from a table, exp(r) by its Taylor series up to
// r^6 / 6! (|r| <= ln 2 / 32: what is left out is below 2^-50; the rounding of
// ln 2 / 16 times y, at most 1 024 for a weight, below 2^-48).
__device__ const double SIXTEENTHS[16] = {
    0x1.0000000000000p+0, 0x1.ea4afa2a490dap-1, 0x1.d5818dcfba487p-1, 0x1.c199bdd85529cp-1,
    0x1.ae89f995ad3adp-1, 0x1.9c49182a3f090p-1, 0x1.8ace5422aa0dbp-1, 0x1.7a11473eb0187p-1,
    0x1.6a09e667f3bcdp-1, 0x1.5ab07dd485429p-1, 0x1.4bfdad5362a27p-1, 0x1.3dea64c123422p-1,
    0x1.306fe0a31b715p-1, 0x1.2387a6e756238p-1, 0x1.172b83c7d517bp-1, 0x1.0b5586cf9890fp-1,
};
DEV double exp_neg(const double* table, double a, int S) {
    // the sum's last bits are the rounded integer
    const double t = fma(a, 0x1.71547652b82fep+4, 0x1.8p52);
    const int y = (int)(uint32_t)__builtin_bit_cast(uint64_t, t);
    const double r = fma(t - 0x1.8p52, 0x1.62e42fefa39efp-5, -a);
    double e = fma(r, 1.0 / 720.0, 1.0 / 120.0);
    e = fma(e, r, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    // the power of two goes into the table entry's exponent
    const uint64_t p = __builtin_bit_cast(uint64_t, table[y & 15]) + ((uint64_t)(uint32_t)(S - (y >> 4)) << 52);
    return e * __builtin_bit_cast(double, p);
}
// rint(e) for 0 <= e <= 2^51: the sum's last bit is worth one
DEV uint64_t to_int(double e) {
    return __builtin_bit_cast(uint64_t, e + 0x1p52) - __builtin_bit_cast(uint64_t, 0x1p52);
}

// f(token, logit) for the tokens [lo, hi) of a row, in no particular order; lo
// a multiple of 8; by N threads: the workgroup's, or a wave's lanes.
template <typename L, int N = NT, typename F> DEV void each(const void* p, int vec, int lo, int hi, F f) {
    constexpr int VE = L::VE, U = 16 / VE;
    const int t = threadIdx.x % N;
    int done = lo;
    if (vec) {
        const int v1 = hi / VE;
        for (int v0 = lo / VE + t; v0 < v1; v0 += N * U) {
            float x[U][VE];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = v0 + u * N;
                L::many(p, (int64_t)(v < v1 ? v : v0) * VE, x[u]);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = v0 + u * N;
                if (v < v1)
#pragma unroll
                    for (int e = 0; e < VE; e++) f(v * VE + e, x[u][e]);
            }
        }
        done = v1 * VE > lo ? v1 * VE : lo;
    }
    for (int i = done + t; i < hi; i += N) f(i, L::one(p, i));
}

template <typename L> struct Row : Settings {
    const void* p;
    const double* table;         // SIXTEENTHS in LDS
    int V, S, vec;

    DEV double below(float x) const {      // the largest logit less x
        if (inf) x = x == __builtin_huge_valf() ? 0.0f : -__builtin_huge_valf();
        return (double)M - (double)x;
    }
    // 2^S exp(-d / T); 64 temperatures are far past the last weight
    DEV double exp_of(double d) const { return exp_neg(table, fmin(d * invT, 64.0), S); }
    DEV uint64_t weight(double d) const { return to_int(exp_of(d)); }
    DEV uint64_t weight_of(uint64_t c) const { return weight(below(logit_of(c))); }
    // with min_p's say
    DEV uint64_t weight_min(float x) const {
        const double e = exp_of(below(x));
        return e >= min_w ? to_int(e) : 0;
    }
    DEV int bin(double d) const { return min((int)((float)d * bins), NB - 1); }
    DEV int bin_of(uint64_t c) const { return bin(below(logit_of(c))); }

    DEV void open(const SmArgs& a, int r, const double* powers) {
        table = powers;
        p = (const char*)a.x + r * a.stride * L::SIZE;
        V = a.V;
        S = a.S;
        vec = a.vec;
    }
    // The settings of row r with its largest and its least logit above
    // -infinity; false where the row needs no weights (there is none, or
    // greedy).
    DEV bool set(const SmArgs& a, int r, uint64_t best, float least) {
        M = logit_of(best);
        const float T = a.temp ? a.temp[r] : 1.0f;
        if (best == 0 || M == -__builtin_huge_valf() || !(T > 0.0f)) return false;
        inf = M == __builtin_huge_valf();
        // FULL bins over the row's logits, or over those with a weight
        const float span = fminf(M - least, T * ((float)(S + 1) * 0.6931472f));
        bins = (float)FULL / fmaxf(span, 1e-30f);
        if (inf) M = 0.0f;
        invT = 1.0 / (double)T;
        k = a.top_k ? a.top_k[r] : 0;
        by_k = k > 0 && k < V;
        const float tp = a.top_p ? a.top_p[r] : 1.0f, mp = a.min_p ? a.min_p[r] : 0.0f;
        by_p = tp < 1.0f;
        p_goal = tp > 0.0f ? (double)tp : 0.0;
        const double min_p = mp > 1.0f ? 1.0 : mp > 0.0f ? (double)mp : 0.0;
        edge = min_p > 0.0 ? -log(min_p) : 0.0;
        by_m = min_p > 0.0 && edge < (S + 1) * 0.69314718055994530942;
        edge = edge > 0.0 ? edge * (double)T : 0.0;      // (an infinite T among them)
        blur = 0x1p-48 * (double)T;
        min_w = by_m ? ldexp(min_p, S) : 0.0;
        return true;
    }
    // Top-p's goal for a total: one token at least.
    DEV double goal(uint64_t total) const { return fmax(p_goal * (double)total, 0.5); }
};

// SIXTEENTHS into LDS; a barrier follows before it is read.
DEV void load_table(double* table) {
    if (threadIdx.x < 16) table[threadIdx.x] = SIXTEENTHS[threadIdx.x];
}

// The row's largest composite and least logit from its chunks'.
DEV uint64_t row_best(const SmArgs& a, int r, float* least) {
    const int lane = threadIdx.x & 63;
    const size_t at = (size_t)r * a.chunks + min(lane, a.chunks - 1);
    uint64_t b = a.best[at];
    float m = a.least[at];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)b, d), hi = __shfl_xor((uint32_t)(b >> 32), d);
        const uint64_t o = (uint64_t)hi << 32 | lo;
        b = o > b ? o : b;
        m = fminf(m, __shfl_xor(m, d));
    }
    *least = m;
    return b;
}

template <int CTRL, int ROWS> DEV uint64_t dpp64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
    return (uint64_t)hi << 32 | lo;
}
// Inclusive sum over a wave's lanes: within rows of 16 (shifts by 1, 2, 4, 8),
// then the last lane of a row, and of the lower half, to those after it.
DEV uint64_t wave_scan64(uint64_t v) {
    v += dpp64<0x111, 0xF>(v);
    v += dpp64<0x112, 0xF>(v);
    v += dpp64<0x114, 0xF>(v);
    v += dpp64<0x118, 0xF>(v);
    v += dpp64<0x142, 0xA>(v);
    v += dpp64<0x143, 0xC>(v);
    return v;
}
DEV uint64_t lane_of(uint64_t v, int l) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}

// Inclusive sum over the workgroup's threads; *total gets the sum of all.
DEV uint64_t scan64(uint64_t* red, uint64_t v, uint64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan64(v);
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
// The same of two sums at once.
DEV void scan64x2(uint64_t* red, uint64_t& x, uint64_t& y) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    x = wave_scan64(x);
    y = wave_scan64(y);
    __syncthreads();
    if (lane == 63) {
        red[wave] = x;
        red[NW + wave] = y;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW - 1; w++)
        if (w < wave) {
            x += red[w];
            y += red[NW + w];
        }
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
    if (a.logp) a.logp[r] = (float)(-row.below(x) * row.invT - log((double)total / (double)(1ull << row.S)));
}

// ---------------------------------------------------------------------------
template <typename L> __global__ __launch_bounds__(NT) void k_smp_max(SmArgs a) {
    __shared__ uint64_t red[NW];
    __shared__ float red_min[NW];
    const int r = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
    Row<L> row;
    row.open(a, r, nullptr);
    if (c == 0 && t == 0) {
        a.state[r].tick[0] = a.state[r].tick[1] = 0;
        a.state[r].n_list = 0;
    }
    float m = -__builtin_huge_valf(), least = -m;
    int at = -1;
    each<L>(row.p, row.vec, c * a.chunk, min(a.V, (c + 1) * a.chunk), [&](int i, float x) {
        if (x > m) {
            m = x;
            at = i;
        }
        if (x > -__builtin_huge_valf()) least = fminf(least, x);
    });
    uint64_t b = at >= 0 ? comp_of(m, at) : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)b, d), hi = __shfl_xor((uint32_t)(b >> 32), d);
        const uint64_t o = (uint64_t)hi << 32 | lo;
        b = o > b ? o : b;
        least = fminf(least, __shfl_xor(least, d));
    }
    if ((t & 63) == 0) {
        red[t >> 6] = b;
        red_min[t >> 6] = least;
    }
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < NW; w++) {
            b = red[w] > b ? red[w] : b;
            least = fminf(least, red_min[w]);
        }
        a.best[(size_t)r * a.chunks + c] = b;
        a.least[(size_t)r * a.chunks + c] = least;
    }
}

// ---------------------------------------------------------------------------
struct HistShared {
    unsigned long long wsum[NB];
    uint32_t count[NB];
    unsigned long long gw[NG], fw[GB];     // a group's, a fine bin's weight over all chunks
    uint32_t gc[NG], fc[GB];
    uint64_t red[2 * NW];
    double table[16];
    int flag;
};

// What a prefix search looks for: the first `count` tokens, or the shortest
// prefix whose weights reach `goal`.
enum { BY_COUNT, BY_GOAL };
struct Want {
    int by;
    uint64_t count;
    double goal;
    DEV bool met(uint64_t n, uint64_t w) const {
        return by == BY_COUNT ? n >= count : (double)w >= goal;
    }
};

// A bin with the tokens and weight above it and in it.
struct Border {
    int bin;               // -1: the search's end lies past the last bin
    uint64_t n, w, n_in, w_in;
};

// The first of `lanes` lanes' (count, weight) pairs at which a prefix with n
// tokens and w weight before them meets `want` (-1: none); every wave alike.
DEV int cross(const Want& want, int lanes, uint64_t c, uint64_t v, uint64_t* n, uint64_t* w) {
    const int lane = threadIdx.x & 63;
    const uint64_t ic = wave_scan64(lane < lanes ? c : 0), iv = wave_scan64(lane < lanes ? v : 0);
    const uint64_t hit = __ballot(lane < lanes && want.met(*n + ic, *w + iv));
    if (!hit) return -1;
    const int at = __ffsll((unsigned long long)hit) - 1;
    *n += lane_of(ic - c, at);
    *w += lane_of(iv - v, at);
    return at;
}

// The 16 bins of group g over all chunks, into sh.fc / sh.fw.
DEV void load_group(const SmArgs& a, HistShared& sh, int r, int g) {
    const int t = threadIdx.x, b = t & (GB - 1);
    __syncthreads();
    if (t < GB) {
        sh.fc[t] = 0;
        sh.fw[t] = 0;
    }
    __syncthreads();
    if (a.chunks == 1) {
        if (t < GB) {
            sh.fc[t] = sh.count[g * GB + t];
            sh.fw[t] = sh.wsum[g * GB + t];
        }
    } else {
        constexpr int KG = NT / GB;        // threads of a bin
        uint64_t v[MAX_CHUNKS / KG];
        uint32_t c[MAX_CHUNKS / KG];
        const size_t at = (size_t)r * a.chunks * NB + g * GB + b;
#pragma unroll
        for (int i = 0; i < MAX_CHUNKS / KG; i++) {
            const int k = t / GB + i * KG;
            const size_t x = at + (size_t)min(k, a.chunks - 1) * NB;
            v[i] = get_agent(a.wsum + x);
            c[i] = __hip_atomic_load(a.count + x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (k >= a.chunks) v[i] = c[i] = 0;
        }
        for (int i = 1; i < MAX_CHUNKS / KG; i++) {
            v[0] += v[i];
            c[0] += c[i];
        }
        if (c[0]) {
            atomicAdd(&sh.fc[b], c[0]);
            atomicAdd(&sh.fw[b], (unsigned long long)v[0]);
        }
    }
    __syncthreads();
}

DEV Border find_border(const SmArgs& a, HistShared& sh, int r, const Want& want, int* loaded) {
    const int lane = threadIdx.x & 63;
    Border o = {-1, 0, 0, 0, 0};
    const int g = cross(want, NG, sh.gc[lane], sh.gw[lane], &o.n, &o.w);
    if (g < 0) return o;
    if (*loaded != g) load_group(a, sh, r, g);
    *loaded = g;
    const uint64_t c = sh.fc[lane & (GB - 1)], w = sh.fw[lane & (GB - 1)];
    const int f = cross(want, GB, c, w, &o.n, &o.w);
    if (f < 0) return o;
    o.bin = g * GB + f;
    o.n_in = lane_of(c, f);
    o.w_in = lane_of(w, f);
    return o;
}

// Finds the border bins from the groups' sums.
template <typename L> DEV void find_borders(const SmArgs& a, HistShared& sh, const Row<L>& row, SmState* st, int r) {
    const int t = threadIdx.x, lane = t & 63;
    const uint64_t tn = lane_of(wave_scan64(sh.gc[lane]), 63), tw = lane_of(wave_scan64(sh.gw[lane]), 63);
    // a list of whole groups, where that is short enough, needs no bins (each
    // group's take a microsecond or two to load: top-k 50 and top-p 0.95 of one
    // row 8.8 us for the launch against 12.4)
    {
        uint64_t n = 0, w = 0, gk = 0;
        const int g = row.by_k ? cross(Want{BY_COUNT, (uint64_t)row.k, 0.0}, NG, sh.gc[lane], sh.gw[lane], &n, &w) : -1;
        int last = g;
        if (g < 0) {         // all tokens stay, or top-p's
            n = w = 0;
            last = row.by_p ? cross(Want{BY_GOAL, 0, row.goal(tw)}, NG, sh.gc[lane], sh.gw[lane], &n, &w) : -1;
        }
        if (last < 0) {
            n = 0;
            gk = tn;
            last = NG - 1;
        } else {
            gk = sh.gc[last];
        }
        if (n + gk <= LISTED) {
            if (t == 0) {
                st->by_k = g >= 0;
                st->by_p = row.by_p;
                st->by_m = row.by_m;
                st->last = last * GB + GB - 1;
                st->total = tw;
                st->mode = SM_LIST;
            }
            return;
        }
    }
    int loaded = -1;
    Border k = {-1, 0, 0, 0, 0}, p0 = k, p1 = k;
    if (row.by_k) k = find_border(a, sh, r, Want{BY_COUNT, (uint64_t)row.k, 0.0}, &loaded);
    const bool by_k = k.bin >= 0;        // fewer tokens than k: all stay
    if (row.by_p) {
        // the weight that top-k leaves lies between these
        p0 = find_border(a, sh, r, Want{BY_GOAL, 0, row.goal(by_k ? k.w : tw)}, &loaded);
        p1 = by_k ? find_border(a, sh, r, Want{BY_GOAL, 0, row.goal(k.w + k.w_in)}, &loaded) : p0;
    }
    const bool by_p = p0.bin >= 0 && p1.bin >= 0;
    const int last = by_k ? k.bin : by_p ? p1.bin : NB - 1;
    const uint64_t upto = by_k ? k.n + k.n_in : by_p ? p1.n + p1.n_in : tn;
    // min-p's border cuts something only where it lies within top-k's and
    // top-p's prefix: behind `last` its bins, however many tokens they hold,
    // are not listed.  So a list has at most in_s tokens, and at most upto
    // (of the border's distance 1e-6 on either side, and 2^-48 temperatures:
    // what rounding moves a weight's distance by)
    const int ml = row.by_m ? row.bin(fmax(row.edge * (1.0 - 1e-6) - row.blur, 0.0)) : NB;
    const int mh = row.by_m ? min(row.bin(row.edge * (1.0 + 1e-6) + row.blur), last) : -1;
    uint64_t in_s = (by_k ? k.n_in : 0) + (by_p ? p1.n + p1.n_in - p0.n : 0);
    if (upto > CAP)
        for (int b = ml; b <= mh; b++) {
            if (loaded != b / GB) load_group(a, sh, r, b / GB);
            loaded = b / GB;
            in_s += sh.fc[b % GB];
        }
    if (t == 0) {
        st->by_k = by_k;
        st->by_p = by_p;
        st->by_m = ml <= last;
        st->last = last;
        st->bk = k.bin;
        st->pl = p0.bin;
        st->ph = p1.bin;
        st->ml = ml;
        st->mh = mh;
        st->rk = by_k ? (unsigned)((uint64_t)row.k - k.n) : 0;
        st->wk = k.w;
        st->wp = p0.w;
        st->total = tw;
        st->mode = upto <= LISTED ? SM_LIST : in_s <= CAP || upto <= CAP ? SM_BINS : SM_SPLIT;
    }
}

template <typename L> __global__ __launch_bounds__(NT) void k_smp_hist(SmArgs a) {
    __shared__ HistShared sh;
    const int r = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
    SmState* st = a.state + r;
    Row<L> row;
    row.open(a, r, sh.table);
    load_table(sh.table);
    float least;
    const uint64_t best = row_best(a, r, &least);
    if (!row.set(a, r, best, least)) {
        if (c == 0 && t == 0) {
            const bool none = best == 0 || logit_of(best) == -__builtin_huge_valf();
            a.tok[r] = none ? -1 : index_of(best);
            if (a.logp) a.logp[r] = none ? -__builtin_huge_valf() : 0.0f;
            st->mode = SM_DONE;
        }
        return;
    }
    if (c == 0 && t == 0) st->set = row;
    const int lo = c * a.chunk, hi = min(a.V, lo + a.chunk);
    if (!row.by_k && !row.by_p) {
        // a sum for each wave's quarter of the chunk
        __syncthreads();
        const int q = a.chunk / NW, q0 = lo + (t >> 6) * q;
        uint64_t s = 0;
        each<L, 64>(row.p, row.vec, q0, min(hi, q0 + q), [&](int, float x) { s += row.weight_min(x); });
        s = wave_scan64(s);
        if ((t & 63) == 63) a.csum[((size_t)r * a.chunks + c) * NW + (t >> 6)] = s;
        if (c == 0 && t == 0) st->mode = SM_PLAIN;
        return;
    }
    for (int b = t; b < NB; b += NT) {
        sh.count[b] = 0;
        sh.wsum[b] = 0;
    }
    __syncthreads();
    each<L>(row.p, row.vec, lo, hi, [&](int, float x) {
        const double d = row.below(x);
        const uint64_t w = row.weight(d);
        if (w) {
            const int b = row.bin(d);
            atomicAdd(&sh.count[b], 1u);
            atomicAdd(&sh.wsum[b], (unsigned long long)w);
        }
    });
    __syncthreads();
    // the groups' sums, four threads a group
    {
        constexpr int Q = GB / (NT / NG);
        uint32_t n = 0;
        uint64_t w = 0;
#pragma unroll
        for (int e = 0; e < Q; e++) {
            n += sh.count[Q * t + e];
            w += sh.wsum[Q * t + e];
        }
#pragma unroll
        for (int d = 1; d < NT / NG; d <<= 1) {
            n += __shfl_xor(n, d);
            w += (uint64_t)__shfl_xor((uint32_t)(w >> 32), d) << 32 | __shfl_xor((uint32_t)w, d);
        }
        if (t % (NT / NG) == 0) {
            sh.gc[t / (NT / NG)] = n;
            sh.gw[t / (NT / NG)] = w;
        }
    }
    __syncthreads();
    if (a.chunks == 1) {
        for (int b = t; b < NB; b += NT) a.wsum[(size_t)r * NB + b] = sh.wsum[b];
    } else {
        const size_t at = ((size_t)r * a.chunks + c) * NB, ag = ((size_t)r * a.chunks + c) * NG;
        for (int b = t; b < NB; b += NT) put_agent(a.wsum + at + b, sh.wsum[b]);
        for (int b = t; b < NB / 2; b += NT)
            put_agent((uint64_t*)(a.count + at) + b, (uint64_t)sh.count[2 * b + 1] << 32 | sh.count[2 * b]);
        if (t < NG) {
            put_agent(a.gsum + 2 * (ag + t), sh.gw[t]);
            put_agent(a.gsum + 2 * (ag + t) + 1, sh.gc[t]);
        }
        if (!last_here(&st->tick[0], a.chunks, &sh.flag)) return;
        // a load of another XCD's store takes a microsecond or two: all of
        // the groups' at a time, a group by each wave's lane, the chunks by
        // the four waves in turn
        uint64_t w[MAX_CHUNKS / NW], n[MAX_CHUNKS / NW];
        const uint64_t* gp = a.gsum + 2 * ((size_t)r * a.chunks * NG + (t & 63));
#pragma unroll
        for (int i = 0; i < MAX_CHUNKS / NW; i++) {
            const int k = min((t >> 6) + i * NW, a.chunks - 1);
            w[i] = get_agent(gp + 2 * (size_t)k * NG);
            n[i] = get_agent(gp + 2 * (size_t)k * NG + 1);
        }
        if (t < NG) {
            sh.gc[t] = 0;
            sh.gw[t] = 0;
        }
        __syncthreads();
        uint64_t sw = 0, sn = 0;
#pragma unroll
        for (int i = 0; i < MAX_CHUNKS / NW; i++)
            if ((t >> 6) + i * NW < a.chunks) {
                sw += w[i];
                sn += n[i];
            }
        if (sn) {
            atomicAdd(&sh.gc[t & 63], (uint32_t)sn);
            atomicAdd(&sh.gw[t & 63], (unsigned long long)sw);
        }
        __syncthreads();
    }
    find_borders(a, sh, row, st, r);
}

// ---------------------------------------------------------------------------
struct PickShared {
    uint64_t list[CAP];
    union {
        uint64_t lw[CAP];        // the list's weights
        struct {                 // split_cut's bins: before there is a list
            unsigned long long wsum[NB];
            uint32_t count[NB];
        } bins;
    };
    unsigned long long wsum[NT];
    uint32_t count[NT];
    uint64_t red[2 * NW];
    double table[16];
    uint64_t b0, b1;
    int i0, i1, flag;
    uint32_t n_list;
};

// Entry of sh.list[0, n) (weights in sh.lw) at which a prefix in descending
// order of key(entry) (distinct integers) meets `want`, n0 tokens and w0
// weight before it, among the entries that in(entry) takes; *sum the weight up
// to and with it.  -1: none does.  Radix selection, 8 bits at a time from the
// highest bit in which two keys differ, until one entry is left.
template <typename K, typename I>
DEV int select(PickShared& sh, int n, const Want& want, uint64_t n0, uint64_t w0, K key, I in, uint64_t* sum) {
    const int t = threadIdx.x;
    // the bits in which keys differ: or and and of all
    uint64_t any = 0, all = ~0ull;
    for (int i = t; i < n; i += NT)
        if (in(i)) {
            any |= key(i);
            all &= key(i);
        }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        any |= (uint64_t)__shfl_xor((uint32_t)(any >> 32), d) << 32 | __shfl_xor((uint32_t)any, d);
        all &= (uint64_t)__shfl_xor((uint32_t)(all >> 32), d) << 32 | __shfl_xor((uint32_t)all, d);
    }
    __syncthreads();
    if ((t & 63) == 0) {
        sh.wsum[t >> 6] = any;
        sh.wsum[NW + (t >> 6)] = all;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) {
        any |= sh.wsum[w];
        all &= sh.wsum[NW + w];
    }
    const uint64_t differ = any & ~all;
    int top = differ ? 64 - __clzll((long long)differ) : 1;      // keys agree from this bit up
    uint64_t known = top < 64 ? all >> top << top : 0;
    for (;;) {
        const int low = top > 8 ? top - 8 : 0, mask = (1 << (top - low)) - 1;
        __syncthreads();
        sh.count[t] = 0;
        sh.wsum[t] = 0;
        if (t == 0) sh.i0 = -1;
        __syncthreads();
        for (int i = t; i < n; i += NT)
            if (in(i)) {
                const uint64_t k = key(i);
                if (top == 64 || k >> top == known >> top) {
                    const int b = mask - (int)(k >> low & mask);
                    atomicAdd(&sh.count[b], 1u);
                    atomicAdd(&sh.wsum[b], (unsigned long long)sh.lw[i]);
                }
            }
        __syncthreads();
        const uint64_t c = sh.count[t], w = sh.wsum[t];
        uint64_t n1 = c, w1 = w;
        scan64x2(sh.red, n1, w1);
        n1 += n0;
        w1 += w0;
        if (want.met(n1, w1) && !want.met(n1 - c, w1 - w)) {
            sh.i0 = t;
            sh.i1 = (int)c;
            sh.b0 = n1 - c;
            sh.b1 = w1 - w;
        }
        __syncthreads();
        const int b = sh.i0;
        if (b < 0) return -1;
        n0 = sh.b0;
        w0 = sh.b1;
        const int left = sh.i1;
        known |= (uint64_t)(mask - b) << low;
        top = low;
        if (left == 1 || top == 0) break;
    }
    __syncthreads();
    for (int i = t; i < n; i += NT)
        if (in(i) && key(i) >> top == known >> top) sh.i0 = i;
    __syncthreads();
    const int at = sh.i0;
    *sum = w0 + sh.lw[at];
    __syncthreads();
    return at;
}

// The token of [lo, hi) whose running sum of kept(token, logit), `base` before
// lo, passes aim: by tiles of TE consecutive tokens a thread, the next tile's
// loads ahead of the current one's sums.
template <typename L, typename F>
DEV void draw_range(const SmArgs& a, PickShared& sh, const Row<L>& row, int r, int lo, int hi, uint64_t base,
                    uint64_t aim, uint64_t total, F kept) {
    constexpr int TE = 8;
    const int t = threadIdx.x;
    auto load = [&](int i0, float* x) {
        if (row.vec && i0 + TE <= hi) {       // lo and the tiles are multiples of 8
#pragma unroll
            for (int e = 0; e < TE; e += L::VE) L::many(row.p, i0 + e, x + e);
        } else {
#pragma unroll
            for (int e = 0; e < TE; e++) x[e] = i0 + e < hi ? L::one(row.p, i0 + e) : -__builtin_huge_valf();
        }
    };
    float x[TE], nx[TE];
    load(lo + t * TE, x);
    for (int i0 = lo + t * TE; i0 - t * TE < hi; i0 += NT * TE) {
        if (i0 - t * TE + NT * TE < hi) load(i0 + NT * TE, nx);
        uint64_t w[TE], own = 0, all;
#pragma unroll
        for (int e = 0; e < TE; e++) {
            w[e] = i0 + e < hi ? kept(i0 + e, x[e]) : 0;
            own += w[e];
        }
        uint64_t s = scan64(sh.red, own, &all) - own + base;
        if (base + all > aim) {
#pragma unroll
            for (int e = 0; e < TE; e++) {
                if (s <= aim && aim < s + w[e]) answer(a, row, r, i0 + e, x[e], total);
                s += w[e];
            }
            return;
        }
        base += all;
#pragma unroll
        for (int e = 0; e < TE; e++) x[e] = nx[e];
    }
}

// The lane at which a running sum of the lanes' sums passes aim, base before
// the first; *base gets the sum before it.
DEV int pick_lane(uint64_t sum, uint64_t aim, uint64_t* base) {
    const uint64_t s = wave_scan64(sum) + *base;
    const int l = __ffsll((unsigned long long)__ballot(s > aim)) - 1;
    *base = lane_of(s - sum, l);
    return l;
}

// ---------------------------------------------------------------------------
// A row by one workgroup, for borders in runs too long to sort: the bin's
// composites, which differ, are split into NB ranges until one fits.
// ---------------------------------------------------------------------------
DEV bool find_bin(PickShared& sh, const Want& want, uint64_t n0, uint64_t w0, int* bin, uint64_t* bn, uint64_t* bw) {
    constexpr int PER = NB / NT;
    const int t = threadIdx.x;
    uint64_t c = 0, w = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        c += sh.bins.count[PER * t + e];
        w += sh.bins.wsum[PER * t + e];
    }
    uint64_t n = c, s = w;
    scan64x2(sh.red, n, s);
    n += n0 - c;
    s += w0 - w;
    if (t == 0) sh.i0 = -1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int b = PER * t + e;
        const uint64_t n1 = n + sh.bins.count[b], s1 = s + sh.bins.wsum[b];
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
            sh.bins.count[b] = 0;
            sh.bins.wsum[b] = 0;
        }
        __syncthreads();
        each<L>(row.p, row.vec, 0, row.V, [&](int i, float x) {
            const uint64_t w = row.weight(row.below(x)), c = comp_of(x, i);
            if (w && c >= lo && c <= hi) {
                atomicAdd(&sh.bins.count[(hi - c) >> sf], 1u);
                atomicAdd(&sh.bins.wsum[(hi - c) >> sf], (unsigned long long)w);
            }
        });
        __syncthreads();
        int b;
        uint64_t n1, w1;
        if (!find_bin(sh, want, bn, bw, &b, &n1, &w1)) break;     // all of them: only at the first turn
        const uint32_t in = sh.bins.count[b];
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
            if (c >= lo && c <= hi && row.weight(row.below(x))) {
                const uint32_t at = atomicAdd(&sh.n_list, 1u);
                if (at < CAP) sh.list[at] = c;
            }
        });
        __syncthreads();
        const int n = min((int)sh.n_list, CAP);
        for (int i = t; i < n; i += NT) sh.lw[i] = row.weight_of(sh.list[i]);
        __syncthreads();
        const int at = select(sh, n, want, bn, bw, [&](int i) { return sh.list[i]; }, [](int) { return true; }, sum);
        return at < 0 ? least : sh.list[at];
    }
    return least;
}

template <typename L> DEV void split_row(const SmArgs& a, PickShared& sh, const Row<L>& row, const SmState& st, int r) {
    uint64_t cut = 0, total = st.total;
    if (st.by_k) cut = split_cut(sh, row, Want{BY_COUNT, (uint64_t)row.k, 0.0}, 0, &total);
    if (st.by_p) {
        uint64_t s;
        const uint64_t c = split_cut(sh, row, Want{BY_GOAL, 0, row.goal(total)}, cut, &s);
        cut = c > cut ? c : cut;
    }
    auto kept = [&](int i, float x) -> uint64_t {
        return comp_of(x, i) >= cut ? row.weight_min(x) : 0;
    };
    uint64_t own = 0;
    each<L>(row.p, row.vec, 0, row.V, [&](int i, float x) { own += kept(i, x); });
    scan64(sh.red, own, &total);
    draw_range(a, sh, row, r, 0, row.V, 0, aim_of(a.u[r], total), total, kept);
}

// Of a list of at most LISTED tokens, for token t < n of sh.list: how many lie
// above it (kABOVE: in descending order of composites, else in index order)
// and their weight.  A quarter of the list by each wave for E tokens a lane, n
// at most 64 E; *total gets the whole list's weight.
template <bool kABOVE, int E>
DEV void ranks_of(PickShared& sh, int n, uint64_t* above, uint64_t* before, uint64_t* total) {
    static_assert(64 * E <= LISTED && CAP >= LISTED + NW * LISTED, "the parts lie behind the list");
    const int t = threadIdx.x, lane = t & 63, part = t >> 6;
    uint64_t *pn = sh.list + LISTED, *pw = sh.lw + LISTED;       // [NW][LISTED]
    uint64_t c[E], na[E] = {}, wa[E] = {}, sum = 0;
#pragma unroll
    for (int e = 0; e < E; e++) c[e] = sh.list[lane + 64 * e];   // behind the list's end: not looked at
#pragma unroll 4
    for (int j = part; j < n; j += NW) {
        const uint64_t cj = sh.list[j], wj = sh.lw[j];
        sum += wj;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const bool up = kABOVE ? cj > c[e] : (uint32_t)cj > (uint32_t)c[e];      // larger: a lower index
            if (kABOVE) na[e] += up;
            wa[e] += up ? wj : 0;
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (kABOVE) pn[part * LISTED + lane + 64 * e] = na[e];
        pw[part * LISTED + lane + 64 * e] = wa[e];
    }
    if (lane == 0) sh.red[part] = sum;
    __syncthreads();
    *above = *before = *total = 0;
#pragma unroll
    for (int e = 0; e < NW; e++) {
        *total += sh.red[e];
        if (t < n) {
            if (kABOVE) *above += pn[e * LISTED + t];
            *before += pw[e * LISTED + t];
        }
    }
    __syncthreads();
}

template <bool kABOVE> DEV void ranks(PickShared& sh, int n, uint64_t* above, uint64_t* before, uint64_t* total) {
    if (n <= 128) ranks_of<kABOVE, 2>(sh, n, above, before, total);
    else ranks_of<kABOVE, LISTED / 64>(sh, n, above, before, total);
}

// The draw from such a list that holds the whole prefix, without selection (50
// to 100 tokens of one row of 151 936: 7.7 us for the launch, 14 by selection).
template <typename L>
DEV void answer_few(const SmArgs& a, PickShared& sh, const Row<L>& row, const SmState& st, int r, int n) {
    const int t = threadIdx.x;
    const uint64_t c = t < n ? sh.list[t] : 0, w = t < n ? sh.lw[t] : 0;
    uint64_t above, before, total;
    if (t == 0) {
        sh.b0 = sh.b1 = 0;
        sh.red[NW] = st.total;
    }
    ranks<true>(sh, n, &above, &before, &total);
    if (st.by_k && t < n && above == (uint64_t)row.k - 1) {
        sh.b0 = c;
        sh.red[NW] = before + w;
    }
    __syncthreads();
    const double goal = row.goal(sh.red[NW]);
    if (st.by_p && t < n && (double)before < goal && (double)(before + w) >= goal) sh.b1 = c;
    __syncthreads();
    const uint64_t cut = sh.b1 > sh.b0 ? sh.b1 : sh.b0;
    const uint64_t left = c >= cut && t < n && (!st.by_m || row.weight_min(logit_of(c))) ? w : 0;
    if (t < n) sh.lw[t] = left;
    __syncthreads();
    ranks<false>(sh, n, &above, &before, &total);
    const uint64_t aim = aim_of(a.u[r], total);
    if (t < n && before <= aim && aim < before + left) answer(a, row, r, index_of(c), logit_of(c), total);
}
// The borders in such a list of bins: what of it lies above a border's first
// bin is above all of that bin's tokens.
template <typename L> DEV uint64_t cut_few(PickShared& sh, const Row<L>& row, const SmState& st, int n) {
    const int t = threadIdx.x;
    const uint64_t c = t < n ? sh.list[t] : 0, w = t < n ? sh.lw[t] : 0;
    const int b = t < n ? row.bin_of(c) : NB;
    uint64_t above, before, total;
    if (t == 0) {
        sh.b0 = sh.b1 = 0;
        sh.red[NW] = st.total;
        sh.count[0] = 0;
        sh.wsum[0] = sh.wsum[1] = 0;
    }
    __syncthreads();
    if (st.by_k && b < st.bk) {
        atomicAdd(&sh.count[0], 1u);
        atomicAdd(&sh.wsum[0], (unsigned long long)w);
    }
    if (st.by_p && b < st.pl) atomicAdd(&sh.wsum[1], (unsigned long long)w);
    ranks<true>(sh, n, &above, &before, &total);
    if (st.by_k && b == st.bk && above - sh.count[0] + 1 == st.rk) {
        sh.b0 = c;
        sh.red[NW] = st.wk + before - sh.wsum[0] + w;
    }
    __syncthreads();
    const double goal = row.goal(sh.red[NW]);
    before += st.wp - sh.wsum[1];
    if (st.by_p && b >= st.pl && b <= st.ph && (double)before < goal && (double)(before + w) >= goal) sh.b1 = c;
    __syncthreads();
    return sh.b1 > sh.b0 ? sh.b1 : sh.b0;
}

template <typename L> __global__ __launch_bounds__(NT) void k_smp_pick(SmArgs a) {
    __shared__ PickShared sh;
    const int r = blockIdx.y, c = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    SmState* sp = a.state + r;
    const int mode = sp->mode;
    if (mode == SM_DONE || ((mode == SM_PLAIN || mode == SM_SPLIT) && c != 0)) return;
    Row<L> row;
    row.open(a, r, sh.table);
    load_table(sh.table);
    (Settings&)row = sp->set;
    if (t == 0) sh.n_list = 0;
    __syncthreads();
    if (mode == SM_PLAIN) {
        // the chunk, then the quarter of it
        uint64_t sums[NW] = {}, own = 0, base = 0;
        if (lane < a.chunks)
#pragma unroll
            for (int w = 0; w < NW; w++) sums[w] = a.csum[((size_t)r * a.chunks + lane) * NW + w];
#pragma unroll
        for (int w = 0; w < NW; w++) own += sums[w];
        const uint64_t total = lane_of(wave_scan64(own), 63), aim = aim_of(a.u[r], total);
        const int at = pick_lane(own, aim, &base);
        int w = 0;
        uint64_t here = lane_of(sums[0], at);
#pragma unroll
        for (int e = 1; e < NW; e++)
            if (w == e - 1 && base + here <= aim) {
                base += here;
                here = lane_of(sums[e], at);
                w = e;
            }
        const int q = a.chunk / NW, lo = at * a.chunk + w * q;
        draw_range(a, sh, row, r, lo, min(a.V, lo + q), base, aim, total,
                   [&](int, float x) -> uint64_t { return row.weight_min(x); });
        return;
    }
    const SmState st = *sp;
    if (mode == SM_SPLIT) {
        split_row(a, sh, row, st, r);
        return;
    }
    // the tokens that decide; most are told by their logit alone
    int b_lo = NB, b_hi = -1;
    if (mode == SM_LIST) {
        b_lo = 0;
        b_hi = st.last;
    } else {
        if (st.by_k) b_lo = min(b_lo, st.bk), b_hi = max(b_hi, st.bk);
        if (st.by_p) b_lo = min(b_lo, st.pl), b_hi = max(b_hi, st.ph);
        if (st.by_m) b_lo = min(b_lo, st.ml), b_hi = max(b_hi, st.mh);
    }
    // (with a bin of slack for the rounding of differences and products)
    const float inf = __builtin_huge_valf();
    const double per = 1.0 / (double)row.bins, slack = 1e-6 * fabs((double)row.M);
    const float x_lo = row.inf || b_hi >= NB - 1 ? -inf : (float)((double)row.M - (b_hi + 2) * per - slack);
    const float x_hi = row.inf || b_lo < 2 ? inf : (float)((double)row.M - (b_lo - 2) * per + slack);
    each<L>(row.p, row.vec, c * a.chunk, min(a.V, (c + 1) * a.chunk), [&](int i, float x) {
        if (!(x >= x_lo && x <= x_hi)) return;
        const double d = row.below(x);
        const int b = row.bin(d);
        const bool in = mode == SM_LIST ? b <= st.last
                                        : (st.by_k && b == st.bk) || (st.by_p && b >= st.pl && b <= st.ph) ||
                                              (st.by_m && b >= st.ml && b <= st.mh);
        if (in && row.weight(d) != 0) {
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
        // (the first tokens before their number is known)
        const uint64_t early = get_agent(list + t);
        n = min((int)__hip_atomic_load(&sp->n_list, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), CAP);
        __syncthreads();
        if (t < n) sh.list[t] = early;
        for (int i = t + NT; i < n; i += NT) sh.list[i] = get_agent(list + i);
    }
    __syncthreads();
    for (int i = t; i < n; i += NT) sh.lw[i] = row.weight_of(sh.list[i]);
    __syncthreads();
    if (mode == SM_LIST) {
        answer_few(a, sh, row, st, r, n);
        return;
    }
    auto comp = [&](int i) { return sh.list[i]; };
    auto bin_of = [&](int i) { return row.bin_of(sh.list[i]); };
    uint64_t sum = st.total, cut = 0;      // composites below cut are out
    const bool few = n <= LISTED;
    if (few) cut = cut_few(sh, row, st, n);
    if (!few && st.by_k) {
        const int at = select(sh, n, Want{BY_COUNT, st.rk, 0.0}, 0, st.wk, comp,
                              [&](int i) { return bin_of(i) == st.bk; }, &sum);
        if (at >= 0) cut = sh.list[at];
    }
    if (!few && st.by_p) {
        uint64_t s;
        const int at = select(sh, n, Want{BY_GOAL, 0, row.goal(sum)}, 0, st.wp, comp,
                              [&](int i) {
                                  if (!st.by_k && !st.by_m) return true;     // a list of top-p's bins alone
                                  const int b = bin_of(i);
                                  return b >= st.pl && b <= st.ph;
                              },
                              &s);
        if (at >= 0 && sh.list[at] > cut) cut = sh.list[at];
    }
    // what stays of the list
    for (int i = t; i < n; i += NT)
        if (sh.list[i] < cut || (st.by_m && row.weight_min(logit_of(sh.list[i])) == 0)) sh.lw[i] = 0;
    __syncthreads();
    // the chunks' sums: the bins above the highest border, and what stays of
    // the list from there on
    const int cb = min(cut ? row.bin_of(cut) : NB, st.by_m ? st.ml : NB), g = cb / GB;
    if (a.chunks == 1) {
        uint64_t own = 0;
        if (wave == 0)
            for (int b = lane; b < cb; b += 64) own += a.wsum[(size_t)r * NB + b];
        own = wave_scan64(own);
        if (t == 63) sh.wsum[0] = own;
    } else {
        // a chunk a wave, the loads of CS at a time, all of them before any is waited for
        constexpr int CS = 12;
        const int fine = min(g * GB + (lane & (GB - 1)), NB - 1);
        for (int k0 = wave; k0 < a.chunks; k0 += CS * NW) {
            uint64_t sg[CS], sf[CS];
#pragma unroll
            for (int e = 0; e < CS; e++) {
                const size_t at = (size_t)r * a.chunks + min(k0 + e * NW, a.chunks - 1);
                sg[e] = get_agent(a.gsum + 2 * (at * NG + lane));
                sf[e] = get_agent(a.wsum + at * NB + fine);
            }
#pragma unroll
            for (int e = 0; e < CS; e++) {
                const uint64_t own = wave_scan64((lane < g ? sg[e] : 0) + (lane < cb - g * GB ? sf[e] : 0));
                if (lane == 63 && k0 + e * NW < a.chunks) sh.wsum[k0 + e * NW] = own;
            }
        }
    }
    __syncthreads();
    for (int i = t; i < n; i += NT)
        if (sh.lw[i] && bin_of(i) >= cb)
            atomicAdd(&sh.wsum[index_of(sh.list[i]) / a.chunk], (unsigned long long)sh.lw[i]);
    __syncthreads();
    const uint64_t mine = lane < a.chunks ? sh.wsum[lane] : 0;
    const uint64_t total = lane_of(wave_scan64(mine), 63), aim = aim_of(a.u[r], total);
    uint64_t base = 0;
    const int at = pick_lane(mine, aim, &base);
    draw_range(a, sh, row, r, at * a.chunk, min(a.V, (at + 1) * a.chunk), base, aim, total,
               [&](int i, float x) -> uint64_t { return comp_of(x, i) >= cut ? row.weight_min(x) : 0; });
}

struct SmPlan {
    int rows, chunk, chunks;
    size_t best, csum, wsum, gsum, list, count, least, state, bytes;
};

// Chunks of 4 096 tokens, or a multiple where that would be more than about
// four workgroups a CU over all rows, or more than 64 chunks a row.
SmPlan plan(int n, int V) {
    SmPlan p;
    p.rows = n < ROWS ? n : ROWS;
    int c = (ROWS + p.rows - 1) / p.rows;
    if (c > MAX_CHUNKS) c = MAX_CHUNKS;
    p.chunk = ((V + c - 1) / c + 4095) / 4096 * 4096;
    if (p.chunk > 4096 && V / (p.chunk - 4096) < (c > 1 ? MAX_CHUNKS : 1)) p.chunk -= 4096;
    p.chunks = (V + p.chunk - 1) / p.chunk;
    const size_t k = (size_t)p.rows * p.chunks;
    p.best = 0;
    p.csum = p.best + k * 8;
    p.wsum = p.csum + k * NW * 8;
    p.gsum = p.wsum + k * NB * 8;
    p.list = p.gsum + k * NG * 16;
    p.count = p.list + (size_t)p.rows * CAP * 8;
    p.least = p.count + k * NB * 4;
    p.state = (p.least + k * 4 + 7) / 8 * 8;
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
    a.S = 62 - lg < 51 ? 62 - lg : 51;
    a.vec = ((uintptr_t)x & 15) == 0 && (stride * es) % 16 == 0;
    a.chunk = pl.chunk;
    a.chunks = pl.chunks;
    char* w = (char*)ws;
    a.best = (uint64_t*)(w + pl.best);
    a.csum = (uint64_t*)(w + pl.csum);
    a.wsum = (uint64_t*)(w + pl.wsum);
    a.gsum = (uint64_t*)(w + pl.gsum);
    a.list = (uint64_t*)(w + pl.list);
    a.count = (uint32_t*)(w + pl.count);
    a.least = (float*)(w + pl.least);
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
