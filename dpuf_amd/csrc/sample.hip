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
// c_i = (order-preserving bits of x_i) << 32 | (2^32 - 1 - i).  Top-k and
// top-p both keep a prefix of it: the tokens with c_i >= cut.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hip_internal.h"
#include "paged.h"

namespace {

constexpr int NT = 512;          // threads of a row's workgroup
constexpr int NB = 2048;         // bins
constexpr int CAP = 4096;        // tokens sorted in LDS

struct SmArgs {
    const void* x;
    int64_t stride;
    int n, V, S, vec;
    const float* temp;
    const int* top_k;
    const float *top_p, *min_p, *u;
    int* tok;
    float* logp;
};

struct F32L {
    static constexpr int VE = 4;
    static DEV float one(const void* p, int64_t i) { return ((const float*)p)[i]; }
    static DEV void many(const void* p, int64_t i, float* o) {
        const float4 v = *(const float4*)((const float*)p + i);
        o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
    }
};
template <typename T> struct H16L {
    static constexpr int VE = 8;
    static DEV float one(const void* p, int64_t i) { return (float)((const typename T::e*)p)[i]; }
    static DEV void many(const void* p, int64_t i, float* o) {
        const typename T::v8 v = vec_of<typename T::v8>(*(const u32x4*)((const uint16_t*)p + i));
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (float)v[e];
    }
};

DEV uint32_t order_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);      // -0 and +0 are one value
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
DEV float from_bits(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
DEV uint64_t comp_of(float x, int i) { return (uint64_t)order_bits(x) << 32 | (0xffffffffu - (uint32_t)i); }

// 2^s exp(-a) for 0 <= a < 64: exp(-a) = 2^-n exp(r) with n = rint(a / ln 2) and
// r = n ln 2 - a, by the Taylor series of exp up to r^13 / 13! (|r| <= ln 2 / 2: what is left
// out is below 2^-56).
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

struct Shared {
    unsigned long long wsum[NB];
    uint32_t count[NB];
    uint64_t list[CAP];
    uint64_t lw[CAP];
    uint64_t red[NT / 64];
    uint64_t b0, b1;
    int i0, i1;
    uint32_t n_list;
};

DEV uint64_t shfl_up64(uint64_t v, int d) {
    const uint32_t lo = __shfl_up((uint32_t)v, d), hi = __shfl_up((uint32_t)(v >> 32), d);
    return (uint64_t)hi << 32 | lo;
}

// Inclusive sum over the workgroup's threads; *total gets the sum of all.
DEV uint64_t scan64(Shared& sh, uint64_t v, uint64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = shfl_up64(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 63) sh.red[wave] = v;
    __syncthreads();
    uint64_t base = 0, all = 0;
    for (int w = 0; w < NT / 64; w++) {
        if (w == wave) base = all;
        all += sh.red[w];
    }
    *total = all;
    return v + base;
}

// Descending bitonic sort of sh.list[0, n), n a power of two.
DEV void sort_desc(Shared& sh, int n) {
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < n / 2; i += NT) {
                const int a = (i & ~(j - 1)) << 1 | (i & (j - 1)), b = a | j;
                const uint64_t x = sh.list[a], y = sh.list[b];
                const bool desc = !(a & k);
                if ((x < y) == desc) {
                    sh.list[a] = y;
                    sh.list[b] = x;
                }
            }
        }
    __syncthreads();
}

// One row in the workgroup's hands.
template <typename L>
struct Row {
    const void* p;      // the row's first logit
    int V, S, vec;
    float M;
    double invT, A, scale, min_p;
    float bins;         // bins per temperature

    // (M - x) / T, or infinity for tokens that cannot be drawn
    DEV double depth(float x) const {
        const double d = (double)M - (double)x;
        return x == M ? 0.0 : d < __builtin_huge_val() ? d * invT : __builtin_huge_val();
    }
    DEV uint64_t weight(double a) const { return a < A ? (uint64_t)(exp_neg(a, S) + 0.5) : 0; }
    DEV int bin(double a) const {
        const int b = (int)((float)a * bins);
        return b < NB - 1 ? b : NB - 1;
    }
    // f(token, logit) for every token of the row, in no particular order
    template <typename F> DEV void each(F f) const {
        constexpr int VE = L::VE, U = 16 / VE;
        int done = 0;
        if (vec) {
            const int nv = V / VE;
            for (int v0 = threadIdx.x; v0 < nv; v0 += NT * U) {
                float x[U][VE];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int v = v0 + u * NT;
                    L::many(p, (int64_t)(v < nv ? v : v0) * VE, x[u]);
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int v = v0 + u * NT;
                    if (v < nv)
#pragma unroll
                        for (int e = 0; e < VE; e++) f(v * VE + e, x[u][e]);
                }
            }
            done = nv * VE;
        }
        for (int i = done + threadIdx.x; i < V; i += NT) f(i, L::one(p, i));
    }
};

// What a prefix search looks for: the first `count` tokens, or the shortest
// prefix whose weights reach `goal`.
struct Want {
    uint64_t count;
    double goal;
    bool by_weight;
};

// The bin in which a prefix ends: bins descend from 0.  before_n, before_w:
// tokens and weight in the bins above it.  False when the whole set is short
// of it (then everything stays).
DEV bool find_bin(Shared& sh, const Want& w, uint64_t n0, uint64_t w0, int* bin, uint64_t* bn, uint64_t* bw) {
    constexpr int PER = NB / NT;
    uint64_t c = 0, ws = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        c += sh.count[PER * threadIdx.x + e];
        ws += sh.wsum[PER * threadIdx.x + e];
    }
    uint64_t tc, tw;
    uint64_t ic = scan64(sh, c, &tc) - c + n0, iw = scan64(sh, ws, &tw) - ws + w0;
    if (threadIdx.x == 0) sh.i0 = -1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int b = PER * threadIdx.x + e;
        const uint64_t nc = ic + sh.count[b], nw = iw + sh.wsum[b];
        const bool was = w.by_weight ? (double)iw >= w.goal : ic >= w.count;
        const bool is = w.by_weight ? (double)nw >= w.goal : nc >= w.count;
        if (is && !was) {
            sh.i0 = b;
            sh.b0 = ic;
            sh.b1 = iw;
        }
        ic = nc;
        iw = nw;
    }
    __syncthreads();
    const int r = sh.i0;
    *bin = r;
    *bn = sh.b0;
    *bw = sh.b1;
    __syncthreads();
    return r >= 0;
}

DEV void clear_bins(Shared& sh) {
    __syncthreads();
    for (int b = threadIdx.x; b < NB; b += NT) {
        sh.count[b] = 0;
        sh.wsum[b] = 0;
    }
    __syncthreads();
}

// Cut of the prefix that `want` asks for, its tokens lying in the bin `b` of
// the row's first histogram with bn tokens and bw weight above it and n_in in
// it: the composite of the prefix's last token; *sum gets the prefix's weight.
template <typename L>
DEV uint64_t resolve(Shared& sh, const Row<L>& row, const Want& want, int b, uint64_t bn, uint64_t bw, uint64_t n_in,
                     uint64_t* sum) {
    uint64_t lo = 0, hi = ~0ull;
    // more tokens in the bin than can be sorted: split the range of their
    // composites until they fit (they are distinct, so this ends)
    while (n_in > CAP) {
        int sh_ = 0;
        while (((hi - lo) >> sh_) >= NB) sh_++;
        clear_bins(sh);
        row.each([&](int i, float x) {
            const double a = row.depth(x);
            const uint64_t w = row.weight(a);
            if (w && row.bin(a) == b) {
                const uint64_t c = comp_of(x, i);
                if (c >= lo && c <= hi) {
                    atomicAdd(&sh.count[(hi - c) >> sh_], 1u);
                    atomicAdd(&sh.wsum[(hi - c) >> sh_], (unsigned long long)w);
                }
            }
        });
        __syncthreads();
        int sb;
        uint64_t n2, w2;
        if (!find_bin(sh, want, bn, bw, &sb, &n2, &w2)) break;
        n_in = sh.count[sb];
        bn = n2;
        bw = w2;
        hi -= (uint64_t)sb << sh_;
        const uint64_t width = (1ull << sh_) - 1;
        lo = hi - lo > width ? hi - width : lo;
        __syncthreads();
    }
    if (threadIdx.x == 0) sh.n_list = 0;
    __syncthreads();
    row.each([&](int i, float x) {
        const double a = row.depth(x);
        if (row.weight(a) && row.bin(a) == b) {
            const uint64_t c = comp_of(x, i);
            if (c >= lo && c <= hi) {
                const uint32_t at = atomicAdd(&sh.n_list, 1u);
                if (at < CAP) sh.list[at] = c;
            }
        }
    });
    __syncthreads();
    const int n = min((int)sh.n_list, CAP);
    int n2 = 1;
    while (n2 < n) n2 <<= 1;
    for (int i = n + threadIdx.x; i < n2; i += NT) sh.list[i] = 0;
    sort_desc(sh, n2);
    // walk the sorted tokens, PER a thread
    constexpr int PER = CAP / NT;
    uint64_t w[PER], tot = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int at = PER * threadIdx.x + e;
        w[e] = at < n ? row.weight(row.depth(from_bits((uint32_t)(sh.list[at] >> 32)))) : 0;
        tot += w[e];
    }
    uint64_t all;
    uint64_t iw = scan64(sh, tot, &all) - tot + bw;
    if (threadIdx.x == 0) {       // short of it by rounding of the goal: the last one
        sh.i0 = n - 1;
        sh.b1 = bw + all;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int at = PER * threadIdx.x + e;
        const uint64_t nw = iw + w[e];
        const bool was = want.by_weight ? (double)iw >= want.goal : bn + at >= want.count;
        const bool is = want.by_weight ? (double)nw >= want.goal : bn + at + 1 >= want.count;
        if (at < n && is && !was) {
            sh.i0 = at;
            sh.b1 = nw;
        }
        iw = nw;
    }
    __syncthreads();
    const uint64_t cut = n > 0 ? sh.list[sh.i0] : 0;
    *sum = sh.b1;
    __syncthreads();
    return cut;
}

template <typename L>
__global__ __launch_bounds__(NT) void k_sample(SmArgs a) {
    __shared__ Shared sh;
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    Row<L> row;
    row.p = (const char*)a.x + r * a.stride * (L::VE == 4 ? 4 : 2);
    row.V = a.V;
    row.S = a.S;
    row.vec = a.vec;

    // the largest logit and its first index
    uint64_t best = 0;
    row.each([&](int i, float x) {
        const uint64_t c = comp_of(x, i);
        if (x == x && c > best) best = c;
    });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)best, d), hi = __shfl_xor((uint32_t)(best >> 32), d);
        const uint64_t o = (uint64_t)hi << 32 | lo;
        if (o > best) best = o;
    }
    if (lane == 0) sh.red[wave] = best;
    __syncthreads();
    for (int w = 0; w < NT / 64; w++)
        if (sh.red[w] > best) best = sh.red[w];
    __syncthreads();
    row.M = from_bits((uint32_t)(best >> 32));
    const int first = (int)(0xffffffffu - (uint32_t)best);
    if (best == 0 || row.M == -__builtin_huge_valf()) {
        if (t == 0) {
            a.tok[r] = -1;
            if (a.logp) a.logp[r] = -__builtin_huge_valf();
        }
        return;
    }
    const float T = a.temp ? a.temp[r] : 1.0f;
    if (!(T > 0.0f)) {
        if (t == 0) {
            a.tok[r] = first;
            if (a.logp) a.logp[r] = 0.0f;
        }
        return;
    }
    row.invT = 1.0 / (double)T;
    row.scale = (double)(1ull << a.S);
    row.A = (a.S + 1) * 0.69314718055994530942;
    row.bins = (float)(NB / row.A);
    const int k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    const float mp = a.min_p ? a.min_p[r] : 0.0f;
    row.min_p = mp > 1.0f ? 1.0 : mp > 0.0f ? (double)mp : 0.0;
    const bool by_k = k > 0 && k < a.V, by_p = p < 1.0f;

    uint64_t cut = 0;        // tokens with a composite below it are out
    if (by_k || by_p) {
        clear_bins(sh);
        uint64_t mine = 0;
        row.each([&](int, float x) {
            const double d = row.depth(x);
            const uint64_t w = row.weight(d);
            if (w) {
                const int b = row.bin(d);
                atomicAdd(&sh.count[b], 1u);
                atomicAdd(&sh.wsum[b], (unsigned long long)w);
                mine += w;
            }
        });
        uint64_t total;
        scan64(sh, mine, &total);
        __syncthreads();
        int b;
        uint64_t bn, bw;
        if (by_k) {
            const Want want = {(uint64_t)k, 0.0, false};
            if (find_bin(sh, want, 0, 0, &b, &bn, &bw)) {
                const uint64_t n_in = sh.count[b];
                __syncthreads();
                cut = resolve(sh, row, want, b, bn, bw, n_in, &total);
                if (by_p) {      // resolve may have used the bins
                    clear_bins(sh);
                    row.each([&](int i, float x) {
                        const double d = row.depth(x);
                        const uint64_t w = row.weight(d);
                        if (w && comp_of(x, i) >= cut) {
                            const int bb = row.bin(d);
                            atomicAdd(&sh.count[bb], 1u);
                            atomicAdd(&sh.wsum[bb], (unsigned long long)w);
                        }
                    });
                    __syncthreads();
                }
            }
        }
        if (by_p) {
            const Want want = {0, p > 0.0f ? (double)p * (double)total : 0.5, true};
            if (find_bin(sh, want, 0, 0, &b, &bn, &bw)) {
                const uint64_t n_in = sh.count[b];
                __syncthreads();
                uint64_t sum;
                const uint64_t c2 = resolve(sh, row, want, b, bn, bw, n_in, &sum);
                if (c2 > cut) cut = c2;
            }
        }
    }
    auto kept = [&](int i, float x) -> uint64_t {
        const double d = row.depth(x);
        const uint64_t w = row.weight(d);
        return w && comp_of(x, i) >= cut && (row.min_p <= 0.0 || exp_neg(d, 0) >= row.min_p) ? w : 0;
    };
    // in index order: every wave sums a run of the row, then the run that
    // holds the draw is walked by all
    const int run = (a.V + NT / 64 - 1) / (NT / 64);
    uint64_t ws = 0;
    for (int i = wave * run + lane; i < min(wave * run + run, a.V); i += 64) ws += kept(i, L::one(row.p, i));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = shfl_up64(ws, d);
        if (lane >= d) ws += o;
    }
    if (lane == 63) sh.red[wave] = ws;
    __syncthreads();
    uint64_t total = 0;
    for (int w = 0; w < NT / 64; w++) total += sh.red[w];
    const float uf = a.u[r];
    uint64_t aim = uf > 0.0f ? (uint64_t)((double)(uf < 1.0f ? uf : 1.0f) * (double)total) : 0;
    if (aim >= total) aim = total - 1;
    int w0 = 0;
    uint64_t base = 0;
    while (w0 < NT / 64 - 1 && base + sh.red[w0] <= aim) base += sh.red[w0++];
    const int s0 = w0 * run, s1 = min(s0 + run, a.V);
    const int per = (run + NT - 1) / NT, i0 = min(s0 + t * per, s1), i1 = min(i0 + per, s1);
    uint64_t own = 0, all;
    for (int i = i0; i < i1; i++) own += kept(i, L::one(row.p, i));
    const uint64_t end = scan64(sh, own, &all) + base;
    if (own && end > aim && end - own <= aim) {
        uint64_t at = end - own;
        for (int i = i0; i < i1; i++) {
            const float x = L::one(row.p, i);
            at += kept(i, x);
            if (at > aim) {
                a.tok[r] = i;
                if (a.logp) a.logp[r] = (float)(-row.depth(x) - log((double)total / row.scale));
                break;
            }
        }
    }
}

}  // namespace

extern "C" {

size_t dpuf_hip_sample_workspace(int32_t n, int32_t V) {
    (void)n;
    (void)V;
    return 0;
}

void dpuf_hip_sample(void* s, int32_t type, int32_t n, int32_t V, int64_t stride, const void* x, const float* temp,
                     const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* tok,
                     float* logp, void* ws) {
    (void)ws;
    SmArgs a;
    a.x = x;
    a.stride = stride;
    a.n = n;
    a.V = V;
    int lg = 0;
    while ((1 << lg) < V) lg++;
    a.S = 62 - lg;
    const int es = type == DPUF_AMD_F32 ? 4 : 2;
    a.vec = ((uintptr_t)x & 15) == 0 && (stride * es) % 16 == 0;
    a.temp = temp;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.u = u;
    a.tok = tok;
    a.logp = logp;
    if (type == DPUF_AMD_F32) hipLaunchKernelGGL(k_sample<F32L>, dim3(n), dim3(NT), 0, ST(s), a);
    else if (type == DPUF_AMD_BF16) hipLaunchKernelGGL(k_sample<H16L<Bf16>>, dim3(n), dim3(NT), 0, ST(s), a);
    else hipLaunchKernelGGL(k_sample<H16L<Fp16>>, dim3(n), dim3(NT), 0, ST(s), a);
    LAUNCHED("k_sample");
}

}  // extern "C"
