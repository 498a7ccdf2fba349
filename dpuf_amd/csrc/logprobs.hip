// logprobs.hip -- log probabilities of given tokens, entropy and the largest
// alternatives of rows of logits.
//
// With s_i = x_i log2 e - r (one fma, so that r's own rounding cancels) and any r
// near a row's largest x_i log2 e,
//     l = sum 2^s_i,  u = sum 2^s_i s_i,
//     ln p_t = (s_t - log2 l) ln 2,  -sum p ln p = (log2 l - u / l) ln 2.
// Partial sums (r, l, u) move to another r' by d = r' - r: l' = 2^-d l, u' =
// 2^-d (u - d l).  Rows whose largest logit is 2^20 or more away from 0, where r
// would be off by much of a unit, and +infinity, are summed up again, by
// differences of logits.
//
// The k largest logits, in the order "larger first, then lower index": cut the
// row into groups of neighbouring tokens and order the groups by their largest
// logit, then by place.  The first k groups hold the k largest logits: a token
// of another group has k groups before its own, each with a logit that is larger
// or as large and further to the front.  So one pass over the row leaves the
// groups' largest, and what is read again is k groups; or, without ordering them
// first, the few more that reach a bound which at least k groups' largest reach
// (of 151 936 random logits and 20 alternatives 24 groups; one row 9.5 to 10 us, 11
// by the order of the groups), unless those, or their tokens, are many.
//
//   k_lp_part   a workgroup per chunk of a row: (r, l, u) and the groups' largest;
//   k_lp_row    a workgroup per row: joins the chunks, picks groups, the k tokens
//               among theirs, and writes;
//   k_lp_whole  both, a workgroup per row, where there are many rows.
//
// Bound by the bytes of the logits, in 16 bits nearly as much by the exponential
// and ten other instructions of each: 512 rows of 151 936 fp32 logits 54 us, 5.7
// TB/s, 2 048 in bf16 with 20 alternatives 125 us, 5.0 TB/s (the first thirty
// calls after a pause 142).  Few rows are bound by latency: one with 20
// alternatives 3.8 us (38 workgroups) and 5.6, of which 1.0 are the first loads,
// 0.8 the sums, 0.8 the groups' tokens and the rest the bound, the lists and the
// order.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hip_internal.h"
#include "paged.h"

namespace {

constexpr int NT = 256;              // threads of a workgroup
constexpr int NW = NT / 64;
constexpr int GL = 16;               // lanes of a group: a row of the wave
constexpr int FEW = 10, MOST = 32;   // groups a thread picks from
constexpr int DIRECT = NT * MOST;    // groups that are picked from as they are
constexpr int WHOLE = DIRECT * GL * 4;  // tokens of a row that is not cut, of any type, at most
constexpr int OVER = 64;             // groups of a bundle, where there are more
constexpr int LISTED = 1024;         // candidates that are ranked
constexpr int WHICH = 128;           // groups whose tokens may be listed unranked
constexpr int MAX_TOP = DPUF_AMD_LOGPROBS_MAX_TOP;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;
constexpr float SLACK = 8.0f;        // r stays while no s is larger
constexpr float FAR = 0x1p20f;
const float NEG_INF = -__builtin_huge_valf();

struct LpArgs {
    const void* x;
    int64_t stride;
    int V, chunk, chunks, groups;
    int n_targets, n_top;
    const int* targets;
    float *logp, *entropy, *top_logp;
    int* top;
    float4* part;                    // [row][chunk]: r, l, u, the largest logit
    uint32_t* most;                  // [row][group]: order_bits of the group's largest logit
};

// Logits as they lie in memory, 16 bytes a lane, at any place.
struct __attribute__((packed, aligned(2))) Lines2 { uint32_t w[4]; };
struct __attribute__((packed, aligned(4))) Lines4 { uint32_t w[4]; };
struct F32L {
    static constexpr int VE = 4, U = 4;      // logits of a load; loads of a lane at a time
    typedef float e;
    static constexpr uint32_t NONE = 0xff800000u;       // -infinity
    static DEV float one(const void* p, int64_t i) { return ((const float*)p)[i]; }
    static DEV u32x4 raw(const void* p, int64_t i) {
        const Lines4 v = *(const Lines4*)((const float*)p + i);
        return u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
    }
    static DEV void get(u32x4 v, float* o) {
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = __uint_as_float(v[e]);
    }
};
template <typename T> struct H16L {
    static constexpr int VE = 8, U = 2;
    typedef typename T::e e;
    static constexpr uint32_t NONE = 0x80008000u | T::EXP | T::EXP << 16;
    static DEV float one(const void* p, int64_t i) { return (float)((const typename T::e*)p)[i]; }
    static DEV u32x4 raw(const void* p, int64_t i) {
        const Lines2 v = *(const Lines2*)((const uint16_t*)p + i);
        return u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
    }
    static DEV void get(u32x4 w, float* o) {
        const typename T::v8 v = vec_of<typename T::v8>(w);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (float)v[e];
    }
};
// The VE logits from i on, those from hi on -infinity.
template <typename L> DEV u32x4 load(const void* p, int i, int hi) {
    if (i + L::VE <= hi) return L::raw(p, i);
    u32x4 v = {L::NONE, L::NONE, L::NONE, L::NONE};
    constexpr int PER = L::VE / 4;       // logits of a word
#pragma unroll
    for (int e = 0; e < L::VE; e++)
        if (i + e < hi) {
            uint32_t x = PER == 1 ? ((const uint32_t*)p)[i + e] : ((const uint16_t*)p)[i + e];
            v[e / PER] = PER == 1 ? x : (v[e / PER] & ~(0xffffu << (e % PER * 16))) | x << (e % PER * 16);
        }
    return v;
}

// Larger logit, larger integer; -infinity and NaN are 0, both zeros one value.
DEV uint32_t order_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return x > NEG_INF ? k : 0;
}
DEV float from_bits(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
DEV uint64_t comp_of(uint32_t bits, uint32_t i) { return bits ? (uint64_t)bits << 32 | (0xffffffffu - i) : 0; }
DEV uint32_t index_of(uint64_t c) { return 0xffffffffu - (uint32_t)c; }
DEV uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <int CTRL> DEV uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
template <int CTRL> DEV float dppf(float v) { return __uint_as_float(dpp<CTRL>(__float_as_uint(v))); }
// Over the wave, in every lane (of sums, the same bits only from run to run).
DEV float wave_max(float v) {
    v = fmaxf(v, dppf<0x128>(v));
    v = fmaxf(v, dppf<0x124>(v));
    v = fmaxf(v, dppf<0x122>(v));
    v = fmaxf(v, dppf<0x121>(v));
    return max_xor32(max_xor16(v));
}
DEV float wave_add(float v) {
    v += dppf<0x128>(v);
    v += dppf<0x124>(v);
    v += dppf<0x122>(v);
    v += dppf<0x121>(v);
    return add_xor32(add_xor16(v));
}

struct Sum {
    float r, l, u;       // of nothing: l 0
    // to r' >= r.  Past 1 000 nothing is left, and no product of it is NaN.
    DEV void move(float to) {
        const float d = l == 0.0f ? 0.0f : fminf(to - r, 1000.0f), f = __builtin_amdgcn_exp2f(-d);
        u = f * fmaf(-d, l, u);
        l *= f;
        r = to;
    }
    DEV void add(Sum o) {
        const float to = l == 0.0f ? o.r : o.l == 0.0f ? r : fmaxf(r, o.r);
        move(to);
        o.move(to);
        l += o.l;
        u += o.u;
    }
};
DEV Sum wave_sum(Sum s) {
    s.move(wave_max(s.l == 0.0f ? NEG_INF : s.r));
    return Sum{s.r, wave_add(s.l), wave_add(s.u)};
}

struct RowLds {
    Sum ss[NW];
    float sm[NW];
    unsigned n, n_tokens;
    uint32_t __attribute__((aligned(16))) most[NT];
    uint32_t which[WHICH];
    uint32_t bound;
    uint64_t __attribute__((aligned(16))) list[LISTED];
    uint64_t best[NW];
    uint64_t groups[MAX_TOP], tokens[MAX_TOP];
};

// The workgroup's sum and largest logit, in every thread.
DEV void join(RowLds& sh, Sum& s, float& top) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    s = wave_sum(s);
    top = wave_max(top);
    if (lane == 0) {
        sh.ss[wave] = s;
        sh.sm[wave] = top;
    }
    __syncthreads();
    s = sh.ss[0];
    top = sh.sm[0];
#pragma unroll
    for (int w = 1; w < NW; w++) {
        s.add(sh.ss[w]);
        top = fmaxf(top, sh.sm[w]);
    }
}

// (r, l, u) and the largest of tokens [lo, hi), a thread's share; put(g, bits)
// the groups' largest, by the first lane of each.
template <typename L, bool TOP, typename F> DEV void scan(const void* p, int lo, int hi, Sum& s, float& top, F put) {
    constexpr int VE = L::VE, U = L::U, STEP = 64 * VE;       // tokens a wave loads at once
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    s = Sum{-2.0f * FAR, 0.0f, 0.0f};    // logits far below that are nothing (a mask), or the row is summed up again
    top = NEG_INF;
    // the next U loads of a lane are on their way while these are worked on
    u32x4 now[U], next[U];
    auto fetch = [&](int w0) {
#pragma unroll
        for (int u = 0; u < U; u++) next[u] = load<L>(p, w0 + u * NW * STEP + lane * VE, hi);
    };
    fetch(lo + wave * STEP);
    for (int w0 = lo + wave * STEP; w0 < hi; w0 += NW * STEP * U) {
#pragma unroll
        for (int u = 0; u < U; u++) now[u] = next[u];
        if (w0 + NW * STEP * U < hi) fetch(w0 + NW * STEP * U);
        float x[U][VE];
#pragma unroll
        for (int u = 0; u < U; u++) L::get(now[u], x[u]);
        float most = NEG_INF;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float mx = NEG_INF;
#pragma unroll
            for (int e = 0; e < VE; e++)     // (of a signalling NaN the maximum would be NaN)
                mx = fmaxf(mx, __builtin_canonicalizef(x[u][e]));
            most = fmaxf(most, mx);
            if (TOP) {
                uint32_t k = order_bits(mx);
                k = max(k, dpp<0x128>(k));
                k = max(k, dpp<0x124>(k));
                k = max(k, dpp<0x122>(k));
                k = max(k, dpp<0x121>(k));
                const int i = w0 + u * NW * STEP + lane * VE;
                if (lane % GL == 0 && i < hi) put(i / (GL * VE), k);
            }
        }
        // r follows the largest logit only when it is behind by more than SLACK
        top = fmaxf(top, most);
        const float m2 = most * LOG2E;
        if (m2 > s.r + SLACK) s.move(m2);
        float l = 0.0f, v = 0.0f;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < VE; e++) {
                const float t = fmaxf(fmaf(x[u][e], LOG2E, -s.r), -1000.0f);     // NaN and -infinity: -1000, and so 0
                const float q = __builtin_amdgcn_exp2f(t);
                l += q;
                v = fmaf(q, t, v);
            }
        s.l += l;
        s.u += v;
    }
}

// A number that at least K of the threads' items reach, and not many more: the
// K-th largest of the largest of 64 quads of threads, or, where MANY may be asked
// for, of the threads (64 alternatives of one row of 151 936 16.6 us instead of
// 20.8, 20 11.1 instead of 10.7).  f(key) for each item; 0 is none, and 1 the
// least bound.
template <bool LEAN, bool MANY, typename F> DEV uint32_t bound_of(RowLds& sh, int K, F each) {
    const int t = threadIdx.x, lane = t & 63;
    uint32_t b = 0;
    each([&](uint32_t k, int) { b = max(b, k); });
    if (!MANY) {
        b = max(b, dpp<0xB1>(b));      // lanes 1 0 3 2
        b = max(b, dpp<0x4E>(b));      // lanes 2 3 0 1
        if ((t & 3) == 0) sh.most[t >> 2] = b;
    } else {
        sh.most[t] = b;
    }
    if (t == 0) {
        sh.n = sh.n_tokens = 0;
        sh.bound = ~0u;
    }
    __syncthreads();
    const uint32_t mine = MANY ? b : sh.most[lane];
    int above = 0;
    constexpr int AT_ONCE = LEAN ? 16 : 64;
#pragma unroll 1
    for (int i0 = 0; i0 < (MANY ? NT : 64); i0 += AT_ONCE)
#pragma unroll
        for (int i = i0; i < i0 + AT_ONCE; i += 4) {
            const u32x4 q = *(const u32x4*)&sh.most[i];
#pragma unroll
            for (int e = 0; e < 4; e++) above += q[e] > mine;
        }
    uint32_t bound = above < K ? mine : ~0u;       // the least of the K largest
    bound = min(bound, dpp<0x128>(bound));
    bound = min(bound, dpp<0x124>(bound));
    bound = min(bound, dpp<0x122>(bound));
    bound = min(bound, dpp<0x121>(bound));
    auto row = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)bound, l); };
    bound = min(min(row(0), row(16)), min(row(32), row(48)));
    if (MANY) {
        if (lane == 0) atomicMin(&sh.bound, bound);
        __syncthreads();
        bound = sh.bound;
    }
    return max(bound, 1u);
}

// put(place, i) of those of a thread's items that are in, at the next places of a
// list of *n, a wave's side by side, each round's by lane.
template <typename I, typename F, typename P> DEV void append(unsigned* n, I items, F in, P put) {
    int hits = 0;
    items([&](int i) { hits += __popcll(__ballot(in(i))); });
    if (!hits) return;
    int e = (threadIdx.x & 63) == 0 ? (int)atomicAdd(n, (unsigned)hits) : 0;
    e = __builtin_amdgcn_readfirstlane(e);
    items([&](int i) {
        const bool on = in(i);
        const uint64_t hit = __ballot(on);
        const int at = e + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(hit >> 32),
                                                          __builtin_amdgcn_mbcnt_lo((uint32_t)hit, 0));
        if (on) put(at, i);
        e += __popcll(hit);
    });
}

// The K largest of the list's n, largest first, into out.
DEV void rank(const RowLds& sh, int n, int K, uint64_t* out) {
    for (int i = threadIdx.x; i < n; i += NT) {
        const uint64_t k = sh.list[i];
        int r = 0, e = 0;
        for (; e + 8 <= n; e += 8)
#pragma unroll
            for (int d = 0; d < 8; d += 2) {
                const ulonglong2 q = *(const ulonglong2*)&sh.list[e + d];
                r += (q.x > k) + (q.y > k);
            }
        for (; e < n; e++) r += sh.list[e] > k;
        if (r < K) out[r] = k;
    }
}

// The K largest of the threads' items, first by bits, then by the lower index,
// largest first, into out (as comp_of).  A thread has n items (R of them, in
// registers, or with R 0 n, wherever they are): bits(i), 0 for none, of index
// id(i).  Returns how many there are, K at most.  What reaches a bound is listed
// and ranked.  LEAN: in few registers.  MANY: K may be more than 32.
template <int R, bool LEAN, bool MANY, typename F, typename G>
DEV int pick(RowLds& sh, int n, int K, F bits, G id, uint64_t* out) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // f(item) of a thread's items
    auto items = [&](auto f) {
        if constexpr (R > 0) {
#pragma unroll
            for (int i = 0; i < R; i++) f(i);
        } else {
            for (int i = 0; i < n; i++) f(i);
        }
    };
    auto list = [&](uint32_t bound, auto key) {
        append(&sh.n, items, [&](int i) { return key(i) >= bound; },
               [&](int at, int i) {
                   if (at < LISTED) sh.list[at] = comp_of(bits(i), id(i));
               });
        __syncthreads();
        return (int)sh.n;
    };
    const uint32_t bound = bound_of<LEAN, MANY>(sh, K, [&](auto f) { items([&](int i) { f(bits(i), i); }); });
    int listed = list(bound, bits);
    const int found = min(listed, K);
    if (MANY && listed > LISTED) {
        // long runs of equal ones: of those on the bound the lowest indices
        auto key = [&](int i) {
            const uint32_t k = bits(i);
            return k > bound ? ~0u : k == bound ? ~(uint32_t)id(i) : 0u;
        };
        __syncthreads();
        const uint32_t least = bound_of<LEAN, MANY>(sh, K, [&](auto f) { items([&](int i) { f(key(i), i); }); });
        listed = list(least, key);
    }
    if (listed <= LISTED) {
        rank(sh, listed, K, out);
    } else {
        // too many (long runs of equal ones, or they lie with few of the threads): one at a time
        uint64_t last = ~0ull;
        for (int r = 0; r < K; r++) {
            uint64_t m = 0;
            items([&](int i) {
                const uint64_t c = comp_of(bits(i), id(i));
                m = c < last ? max64(m, c) : m;
            });
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) m = max64(m, __shfl_xor((unsigned long long)m, d));
            if (lane == 0) sh.best[wave] = m;
            __syncthreads();
            last = max64(max64(sh.best[0], sh.best[1]), max64(sh.best[2], sh.best[3]));
            if (t == 0) out[r] = last;
            __syncthreads();
        }
    }
    __syncthreads();
    return found;
}

// The groups' largest: in memory, a thread's first ones on their way before the
// row's sum is known, or in LDS.
struct Stored {
    static constexpr bool LEAN = false;
    const uint32_t* p;
    uint32_t early[FEW];
    DEV Stored(const uint32_t* at, int n) : p(at) {
#pragma unroll
        for (int i = 0; i < FEW; i++) early[i] = at[min(i * NT + (int)threadIdx.x, n - 1)];
    }
    DEV uint32_t at(int g) const { return p[g]; }
};
struct Kept {
    static constexpr bool LEAN = true;
    const uint32_t* p;
    DEV uint32_t at(int g) const { return p[g]; }
};
// f(R, items of a thread, bits, id) of the groups, as in pick.
template <int N> struct Int { static constexpr int value = N; };
template <int R, typename F> DEV int of_stored(int n, const Stored& most, F f) {
    uint32_t v[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int g = i * NT + threadIdx.x;
        v[i] = R <= FEW ? most.early[i % FEW] : most.p[min(g, n - 1)];
        if (g >= n) v[i] = 0;
    }
    return f(Int<R>(), R, [&](int i) { return v[i]; }, [&](int i) { return i * NT + threadIdx.x; });
}
template <typename F> DEV int of_groups(int n, const Stored& most, F f) {
    return n <= NT * FEW / 2 ? of_stored<FEW / 2>(n, most, f)
           : n <= NT * FEW   ? of_stored<FEW>(n, most, f)
                             : of_stored<MOST>(n, most, f);
}
template <typename F> DEV int of_groups(int n, const Kept& most, F f) {
    return f(
        Int<0>(), (n + NT - 1) / NT,
        [&](int i) {
            const int g = i * NT + threadIdx.x;
            return g < n ? most.p[g] : 0;
        },
        [&](int i) { return i * NT + threadIdx.x; });
}

// A lane's load of a group's tokens, the e-th of all groups' loads: their first
// one, and their bits in v; group(i) is the i-th of n.
template <typename L, typename F>
DEV int load_group(const LpArgs& a, const void* p, int e, int n, F group, uint32_t* v) {
    const int tok = e < n * GL ? group(e / GL) * GL * L::VE + e % GL * L::VE : a.V;
    float x[L::VE];
    L::get(load<L>(p, tok, a.V), x);
#pragma unroll
    for (int j = 0; j < L::VE; j++) v[j] = order_bits(x[j]);
    return tok;
}

// The K largest logits into sh.tokens, at once: what at least K groups' largest
// reach, at least K logits do, and those lie in these groups.  Returns how many,
// or -1 where that are more than the lists hold.
template <typename L, bool LEAN, bool MANY, typename M>
DEV int pick_at_once(const LpArgs& a, RowLds& sh, int K, const M& most, const void* p) {
    constexpr int VE = L::VE, R = MANY ? 4 : 2;
    uint32_t bound;
    const int n = of_groups(a.groups, most, [&](auto r, int n, auto bits, auto id) {
        auto items = [&](auto f) {
            if constexpr (r.value > 0) {
#pragma unroll
                for (int i = 0; i < r.value; i++) f(i);
            } else {
                for (int i = 0; i < n; i++) f(i);
            }
        };
        bound = bound_of<LEAN, MANY>(sh, K, [&](auto f) { items([&](int i) { f(bits(i), i); }); });
        append(&sh.n, items, [&](int i) { return bits(i) >= bound; },
               [&](int at, int i) {
                   if (at < WHICH) sh.which[at] = id(i);
               });
        __syncthreads();
        return (int)sh.n;
    });
    if (n > WHICH) return -1;
    for (int e0 = 0; e0 < n * GL; e0 += R * NT) {
        uint32_t v[R][VE];
        int tok[R];
#pragma unroll
        for (int i = 0; i < R; i++)
            tok[i] = load_group<L>(a, p, e0 + i * NT + threadIdx.x, n, [&](int g) { return (int)sh.which[g]; }, v[i]);
        auto items = [&](auto f) {
#pragma unroll
            for (int i = 0; i < R * VE; i++) f(i);
        };
        append(&sh.n_tokens, items, [&](int i) { return v[i / VE][i % VE] >= bound; },
               [&](int at, int i) {
                   if (at < LISTED) sh.list[at] = comp_of(v[i / VE][i % VE], tok[i / VE] + i % VE);
               });
    }
    __syncthreads();
    const int listed = sh.n_tokens;
    if (listed > LISTED) return -1;
    rank(sh, listed, K, sh.tokens);
    __syncthreads();
    return min(listed, K);
}

// The n groups' tokens, a lane's load of a group at a time, R of them a thread.
template <typename L, int R, bool LEAN> DEV int pick_tokens(const LpArgs& a, RowLds& sh, int n, const void* p) {
    constexpr int VE = L::VE;
    uint32_t v[R][VE];
    int tok[R];
#pragma unroll
    for (int i = 0; i < R; i++)
        tok[i] = load_group<L>(a, p, i * NT + threadIdx.x, n, [&](int g) { return (int)index_of(sh.groups[g]); }, v[i]);
    return pick<R * VE, LEAN, (R > 2)>(
        sh, R * VE, a.n_top, [&](int i) { return v[i / VE][i % VE]; }, [&](int i) { return tok[i / VE] + i % VE; },
        sh.tokens);
}

// Loads of a thread for the tokens of K groups: 1, 2 or 4.
__host__ __device__ inline int loads_of(int K) {
    static_assert(MAX_TOP * GL / NT == 4, "loads of all groups' tokens");
    return K <= MAX_TOP / 4 ? 1 : K <= MAX_TOP / 2 ? 2 : 4;
}

// Everything about a row, once its sum and its groups' largest are known.
// Its thread's first target was read before: tok0.  LOADS: loads_of(K), or 0
// without alternatives.
template <typename L, int LOADS, typename M>
DEV void finish(const LpArgs& a, RowLds& sh, int row, const void* p, Sum s, float top, int tok0, const M& most) {
    constexpr bool MANY = LOADS == 4;
    const int t = threadIdx.x;
    auto logit = [&](int tok) { return (unsigned)tok < (unsigned)a.V ? L::one(p, tok) : NEG_INF; };
    const float x0 = logit(tok0);
    const bool far = fabsf(top) >= FAR && top > NEG_INF;
    // difference to the largest, of far rows
    auto below = [&](float x) { return x == top ? 0.0f : fmaxf((x - top) * LOG2E, -1000.0f); };
    if (far) {
        s = Sum{0.0f, 0.0f, 0.0f};
        for (int i0 = 0; i0 < a.V; i0 += 32 * NT) {
            float l = 0.0f, u = 0.0f;
            for (int i = i0 + t; i < min(a.V, i0 + 32 * NT); i += NT) {
                const float d = below(L::one(p, i)), q = __builtin_amdgcn_exp2f(d);
                l += q;
                u = fmaf(q, d, u);
            }
            s.l += l;
            s.u += u;
        }
        float same = 0.0f;
        __syncthreads();
        join(sh, s, same);
    }
    const float log_l = log2f(s.l);
    // (of a token with nearly all the weight d - log_l is what is left of their
    // roundings, of either sign; p is 1 at most)
    auto logp = [&](float x) {
        if (!(x > NEG_INF)) return NEG_INF;
        if (far) return fminf((x == top ? 0.0f : x - top) - log_l * LN2, 0.0f);
        const float d = fmaf(x, LOG2E, -s.r);
        return fminf(d > -1e30f ? (d - log_l) * LN2 : x - top, 0.0f);
    };
    if (t == 0 && a.entropy) a.entropy[row] = top > NEG_INF ? fmaxf((log_l - s.u / s.l) * LN2, 0.0f) : 0.0f;
    if constexpr (LOADS > 0) {
        const int K = a.n_top;
        int n = -1;
        if (M::LEAN || a.groups <= DIRECT) {
            n = pick_at_once<L, M::LEAN, MANY>(a, sh, K, most, p);
            if (n < 0) {
                // the K largest groups, and then among their tokens
                __syncthreads();
                n = of_groups(a.groups, most, [&](auto r, int n, auto bits, auto id) {
                    return pick<r.value, M::LEAN, MANY>(sh, n, K, bits, id, sh.groups);
                });
                n = pick_tokens<L, LOADS, M::LEAN>(a, sh, n, p);
            }
        } else {
            // bundles of OVER groups first, by the same argument; 4 096 of them at most
            const int bundles = (a.groups + OVER - 1) / OVER;
            uint32_t b[16];
#pragma unroll 1
            for (int i = 0; i < 16; i++) {
                const int at = i * NT + t;
                uint32_t k = 0;
                for (int g = at * OVER; g < min(a.groups, (at + 1) * OVER); g++) k = max(k, most.at(g));
                b[i] = at < bundles ? k : 0;
            }
            n = pick<16, false, MANY>(
                sh, 16, K, [&](int i) { return b[i]; }, [&](int i) { return i * NT + t; }, sh.tokens);
            constexpr int RG = MAX_TOP * OVER / NT;
            uint32_t v[RG];
            auto of = [&](int i) {
                const int e = i * NT + t;
                return e < n * OVER ? (int)index_of(sh.tokens[e / OVER]) * OVER + e % OVER : a.groups;
            };
#pragma unroll
            for (int i = 0; i < RG; i++) v[i] = of(i) < a.groups ? most.at(of(i)) : 0;
            n = pick<RG, false, MANY>(sh, RG, K, [&](int i) { return v[i]; }, of, sh.groups);
            n = pick_tokens<L, LOADS, M::LEAN>(a, sh, n, p);
        }
        for (int i = t; i < K; i += NT) {
            const int64_t at = (int64_t)row * K + i;
            a.top[at] = i < n ? (int)index_of(sh.tokens[i]) : -1;
            a.top_logp[at] = i < n ? logp(from_bits((uint32_t)(sh.tokens[i] >> 32))) : NEG_INF;
        }
    }
    for (int i = t; i < a.n_targets; i += NT) {
        const int64_t at = (int64_t)row * a.n_targets + i;
        a.logp[at] = logp(i == t ? x0 : logit(a.targets[at]));
    }
}

template <typename L, bool TOP> __global__ __launch_bounds__(NT) void k_lp_part(LpArgs a) {
    __shared__ RowLds sh;
    const int row = blockIdx.x / a.chunks, lo = (blockIdx.x - row * a.chunks) * a.chunk;
    Sum s;
    float top;
    scan<L, TOP>((const typename L::e*)a.x + row * a.stride, lo, min(a.V, lo + a.chunk), s, top,
                 [&](int g, uint32_t k) { a.most[(size_t)row * a.groups + g] = k; });
    join(sh, s, top);
    if (threadIdx.x == 0) a.part[blockIdx.x] = make_float4(s.r, s.l, s.u, top);
}

// A thread's first target of a row, or -1.
DEV int first_target(const LpArgs& a, int row) {
    const int t = threadIdx.x;
    return t < a.n_targets ? a.targets[(int64_t)row * a.n_targets + t] : -1;
}

template <typename L, int LOADS> __global__ __launch_bounds__(NT) void k_lp_row(LpArgs a) {
    constexpr bool TOP = LOADS > 0;
    __shared__ RowLds sh;
    const int row = blockIdx.x, tok = first_target(a, row);
    const Stored most(TOP ? a.most + (size_t)row * a.groups : (const uint32_t*)a.part, TOP ? a.groups : 1);
    Sum s = {NEG_INF, 0.0f, 0.0f};
    float top = NEG_INF;
    for (int c = threadIdx.x; c < a.chunks; c += NT) {
        const float4 v = a.part[(size_t)row * a.chunks + c];
        s.add(Sum{v.x, v.y, v.z});
        top = fmaxf(top, v.w);
    }
    join(sh, s, top);
    finish<L, LOADS>(a, sh, row, (const typename L::e*)a.x + row * a.stride, s, top, tok, most);
}

// Eight workgroups a CU as long as their registers suffice: 2 048 bf16 rows of
// 151 936 with 20 alternatives 125 us, five a CU 147.  More than 32 alternatives
// take more of them, and none may go to memory.
template <typename L, int LOADS>
__global__ __launch_bounds__(NT, LOADS < 4 ? 8 : L::VE < 8 ? 7 : 4) void k_lp_whole(LpArgs a) {
    constexpr bool TOP = LOADS > 0;
    __shared__ RowLds sh;
    extern __shared__ uint32_t most[];
    const int row = blockIdx.x, tok = first_target(a, row);
    const void* p = (const typename L::e*)a.x + row * a.stride;
    Sum s;
    float top;
    scan<L, TOP>(p, 0, a.V, s, top, [&](int g, uint32_t k) { most[g] = k; });
    join(sh, s, top);
    finish<L, LOADS>(a, sh, row, p, s, top, tok, Kept{most});
}

struct LpPlan {
    int whole, chunk, chunks, groups;
    size_t most, bytes;
};

// One workgroup a row where rows are short (12 000 fp32 logits: one row 8.6 us
// against 9.7 in two launches, 64 rows 9.1 and 10.2; 20 000: 10.3 and 9.6) or
// give every CU one or more: 256 rows of 64 000 20.5 and 22.4 (128: 20.0 and
// 17.1), 384 of 151 936 49 and 60 (bf16 41 and 36; 512: 43 and 45), 256 of them
// 42 and 40.  Up to 2^19 tokens: a thread adds up 16 at a time, and then 128 such
// sums, before sums meet in pairs.
//
// Otherwise chunks of whole loads of a workgroup, as many as give the card about
// 2 048 workgroups, of at most 32 768 tokens.  64 rows of 151 936: 17.6 us, in
// chunks of any multiple of 1 024 tokens, the last load part empty, 20.4.
LpPlan plan(int n, int V, int n_top, int VE) {
    LpPlan p;
    p.groups = n_top ? (V + GL * VE - 1) / (GL * VE) : 0;
    p.whole = V <= 16384 || (V <= WHOLE && n >= (V <= 65536 ? 256 : 384));
    int c = (2048 + n - 1) / n;
    if (c < (V + 32767) / 32768) c = (V + 32767) / 32768;
    p.chunk = ((V + c - 1) / c + 4095) / 4096 * 4096;
    p.chunks = (V + p.chunk - 1) / p.chunk;
    p.most = (size_t)n * p.chunks * sizeof(float4);
    p.bytes = p.whole ? 0 : p.most + (size_t)n * p.groups * 4;
    return p;
}

template <typename L, int LOADS> void launch(const LpArgs& a, const LpPlan& pl, int n, hipStream_t st) {
    if (pl.whole) {
        hipLaunchKernelGGL((k_lp_whole<L, LOADS>), dim3(n), dim3(NT), pl.groups * 4, st, a);
    } else {
        hipLaunchKernelGGL((k_lp_part<L, (LOADS > 0)>), dim3((unsigned)n * a.chunks), dim3(NT), 0, st, a);
        hipLaunchKernelGGL((k_lp_row<L, LOADS>), dim3(n), dim3(NT), 0, st, a);
    }
    LAUNCHED("k_lp");
}

}  // namespace

extern "C" {

// The larger of the types' needs: the size is asked for without one.
size_t dpuf_hip_logprobs_workspace(int32_t n, int32_t V, int32_t n_top) {
    const size_t a = plan(n, V, n_top, F32L::VE).bytes, b = plan(n, V, n_top, H16L<Bf16>::VE).bytes;
    return a > b ? a : b;
}

void dpuf_hip_logprobs(void* s, int32_t type, int32_t n, int32_t V, int64_t stride, const void* x, int32_t n_targets,
                       const int32_t* targets, int32_t n_top, float* logp, float* entropy, int32_t* top,
                       float* top_logp, void* ws) {
    const LpPlan pl = plan(n, V, n_top, type == DPUF_AMD_F32 ? F32L::VE : H16L<Bf16>::VE);
    LpArgs a;
    a.x = x;
    a.stride = stride;
    a.V = V;
    a.chunk = pl.chunk;
    a.chunks = pl.chunks;
    a.groups = pl.groups;
    a.n_targets = n_targets;
    a.n_top = n_top;
    a.targets = targets;
    a.logp = logp;
    a.entropy = entropy;
    a.top_logp = top_logp;
    a.top = top;
    a.part = (float4*)ws;
    a.most = (uint32_t*)((char*)ws + pl.most);
    auto go = [&](auto type_) {
        typedef decltype(type_) L;
        const int loads = n_top ? loads_of(n_top) : 0;
        const auto f = loads == 0 ? launch<L, 0> : loads == 1 ? launch<L, 1> : loads == 2 ? launch<L, 2> : launch<L, 4>;
        f(a, pl, n, ST(s));
    };
    if (type == DPUF_AMD_F32) go(F32L());
    else if (type == DPUF_AMD_BF16) go(H16L<Bf16>());
    else go(H16L<Fp16>());
}

}  // extern "C"
