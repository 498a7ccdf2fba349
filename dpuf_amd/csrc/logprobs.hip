// logprobs.hip -- log probabilities of given tokens, entropy and the largest
// alternatives of rows of logits.
//
// With any m near a row's largest logit,
//     l = sum exp(x_i - m),  u = sum exp(x_i - m) (x_i - m),
//     ln p_t = x_t - m - ln l,  -sum p ln p = ln l - u / l.
// Partial sums (m, l, u) move to another m' by d = m' - m: l' = exp(-d) l, u' =
// exp(-d) (u - d l).
//
// The k largest logits, in the order "larger first, then lower index": cut the
// row into groups of neighbouring tokens and order the groups by their largest
// logit, then by place.  The first k groups hold the k largest logits: a token
// of another group has k groups before its own, each with a logit that is larger
// or as large and further to the front.  So one pass over the row leaves the
// groups' largest, and what is read again is k groups.
//
//   k_lp_part  a workgroup per chunk of a row: (m, l, u) and the groups' largest;
//   k_lp_row   a workgroup per row: joins the chunks, picks the k groups, the k
//              tokens among theirs, and writes.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hip_internal.h"
#include "paged.h"

namespace {

constexpr int NT = 256;              // threads of a workgroup
constexpr int NW = NT / 64;
constexpr int GL = 16;               // lanes of a group: a row of the wave
constexpr int DIRECT = 8192;         // groups that are picked from as they are
constexpr int OVER = 64;             // groups of a bundle, where there are more
constexpr int LISTED = 1024;         // candidates that are ranked
constexpr int MAX_TOP = DPUF_AMD_LOGPROBS_MAX_TOP;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float SLACK = 6.0f;        // m stays while no logit is larger by more
const float NEG_INF = -__builtin_huge_valf(), POS_INF = __builtin_huge_valf();

struct LpArgs {
    const void* x;
    int64_t stride;
    int V, chunk, chunks, groups;
    int n_targets, n_top;
    const int* targets;
    float *logp, *entropy, *top_logp;
    int* top;
    float4* part;                    // [row][chunk]: m, l, u, the largest logit
    uint32_t* most;                  // [row][group]: order_bits of the group's largest logit
};

struct F32L {
    static constexpr int VE = 4;
    typedef float e;
    static DEV float one(const void* p, int64_t i) { return ((const float*)p)[i]; }
    // 4 logits at any place
    static DEV void many(const void* p, int64_t i, float* o) {
        struct __attribute__((packed, aligned(4))) V4 { float f[4]; };
        const V4 v = *(const V4*)((const float*)p + i);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = v.f[e];
    }
};
template <typename T> struct H16L {
    static constexpr int VE = 8;
    typedef typename T::e e;
    static DEV float one(const void* p, int64_t i) { return (float)((const typename T::e*)p)[i]; }
    static DEV void many(const void* p, int64_t i, float* o) {
        struct __attribute__((packed, aligned(2))) V8 { uint32_t w[4]; };
        const V8 w = *(const V8*)((const uint16_t*)p + i);
        const typename T::v8 v = vec_of<typename T::v8>(u32x4{w.w[0], w.w[1], w.w[2], w.w[3]});
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (float)v[e];
    }
};

// Larger logit, larger integer; -infinity and NaN are 0, both zeros one value.
DEV uint32_t order_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return x > NEG_INF ? k : 0;
}
DEV float from_bits(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
DEV uint64_t comp_of(uint32_t bits, uint32_t i) { return (uint64_t)bits << 32 | (0xffffffffu - i); }
DEV uint32_t index_of(uint64_t c) { return 0xffffffffu - (uint32_t)c; }

struct Sum {
    float m, l, u;       // of nothing: l 0
    // to m' >= m.  Past 1 000 nothing is left, and no product of it is NaN.
    DEV void move(float to) {
        const float d = l == 0.0f ? 0.0f : fminf(to - m, 1000.0f), f = __builtin_amdgcn_exp2f(-d * LOG2E);
        u = f * fmaf(-d, l, u);
        l *= f;
        m = to;
    }
    DEV void add(Sum o) {
        const float to = l == 0.0f ? o.m : o.l == 0.0f ? m : fmaxf(m, o.m);
        move(to);
        o.move(to);
        l += o.l;
        u += o.u;
    }
};
// The same sum in every lane of the wave, in one order.
DEV Sum wave_sum(Sum s) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const Sum o = {__shfl_xor(s.m, d), __shfl_xor(s.l, d), __shfl_xor(s.u, d)};
        // both lanes of a pair add in the same order
        const bool low = (threadIdx.x & d) == 0;
        Sum a = low ? s : o;
        a.add(low ? o : s);
        s = a;
    }
    return s;
}

template <typename L, bool TOP> __global__ __launch_bounds__(NT) void k_lp_part(LpArgs a) {
    constexpr int VE = L::VE, U = 4, STEP = 64 * VE;       // tokens a wave loads at once
    __shared__ Sum ss[NW];
    __shared__ float sm[NW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x / a.chunks, c = blockIdx.x - row * a.chunks;
    const void* p = (const typename L::e*)a.x + row * a.stride;
    const int lo = c * a.chunk, hi = min(a.V, lo + a.chunk);
    Sum s = {NEG_INF, 0.0f, 0.0f};
    float top = NEG_INF;
    for (int w0 = lo + wave * STEP; w0 < hi; w0 += NW * STEP * U) {
        float x[U][VE];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = w0 + u * NW * STEP + lane * VE;
            if (i + VE <= hi) {
                L::many(p, i, x[u]);
            } else {
#pragma unroll
                for (int e = 0; e < VE; e++) x[u][e] = i + e < hi ? L::one(p, i + e) : NEG_INF;
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = w0 + u * NW * STEP;
            if (at >= hi) break;
            float mx = NEG_INF;
#pragma unroll
            for (int e = 0; e < VE; e++) mx = fmaxf(mx, __builtin_canonicalizef(x[u][e]));   // (a maximum keeps a signalling NaN)
            top = fmaxf(top, mx);
            if (TOP) {
                uint32_t k = order_bits(mx);
#define LP_ROR(n) k = max(k, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)k, 0x120 + n, 0xF, 0xF, false))
                LP_ROR(8);
                LP_ROR(4);
                LP_ROR(2);
                LP_ROR(1);
#undef LP_ROR
                const int g = at / (GL * VE) + lane / GL;
                if (lane % GL == 0 && g < a.groups) a.most[(size_t)row * a.groups + g] = k;
            }
            // m follows the largest logit only when it is behind by more than SLACK
            if (mx > s.m + SLACK) s.move(mx);
#pragma unroll
            for (int e = 0; e < VE; e++) {
                const float d = fmaxf(x[u][e] - s.m, -1000.0f);     // NaN and -infinity: -1000, and so 0
                const float q = __builtin_amdgcn_exp2f(d * LOG2E);
                s.l += q;
                s.u = fmaf(q, d, s.u);
            }
        }
    }
    s = wave_sum(s);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (lane == 0) {
        ss[wave] = s;
        sm[wave] = top;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < NW; w++) {
            s.add(ss[w]);
            top = fmaxf(top, sm[w]);
        }
        a.part[blockIdx.x] = make_float4(s.m, s.l, s.u, top);
    }
}

struct RowLds {
    Sum ss[NW];
    float sm[NW];
    int count[NW];
    unsigned n;
    uint64_t quad[64], best[NW], list[LISTED];
    uint64_t groups[MAX_TOP], tokens[MAX_TOP];
    uint32_t bundle[(1 << 24) / (GL * 4) / OVER];
};

DEV uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// The K largest of key(0) .. key(n - 1), largest first, into out; keys other
// than 0 are distinct, and 0 is nothing.  Returns how many there are, K at most.
// A bound first: the K-th largest of the largest ones of 64 quads of threads,
// which at least K keys reach; those that do are listed and ranked.
template <typename F> DEV int pick(RowLds& sh, int n, int K, F key, uint64_t* out) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint64_t b = 0;
    for (int i = t; i < n; i += NT) b = max64(b, key(i));
    b = max64(b, __shfl_xor((unsigned long long)b, 1));
    b = max64(b, __shfl_xor((unsigned long long)b, 2));
    if ((t & 3) == 0) sh.quad[t >> 2] = b;
    if (t == 0) sh.n = 0;
    __syncthreads();
    const uint64_t mine = sh.quad[lane];
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < 64; i++) above += sh.quad[i] > mine;
    const uint64_t at = __ballot(above == K - 1 && mine != 0);
    const uint64_t bound = at ? __shfl((unsigned long long)mine, __ffsll((unsigned long long)at) - 1) : 1;
    for (int i = t; i < n; i += NT) {
        const uint64_t k = key(i);
        if (k >= bound) {
            const unsigned e = atomicAdd(&sh.n, 1u);
            if (e < LISTED) sh.list[e] = k;
        }
    }
    __syncthreads();
    const int found = min((int)sh.n, K), listed = sh.n;
    if (listed <= LISTED) {
        for (int i = t; i < listed; i += NT) {
            const uint64_t k = sh.list[i];
            int r = 0;
            for (int e = 0; e < listed; e++) r += sh.list[e] > k;
            if (r < K) out[r] = k;
        }
    } else {
        // too many reach the bound (they lie with few of the threads): one at a time
        uint64_t last = ~0ull;
        for (int r = 0; r < K; r++) {
            uint64_t m = 0;
            for (int i = t; i < n; i += NT) {
                const uint64_t k = key(i);
                if (k < last) m = max64(m, k);
            }
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

template <typename L, bool TOP> __global__ __launch_bounds__(NT) void k_lp_row(LpArgs a) {
    constexpr int GS = GL * L::VE;       // tokens of a group
    __shared__ RowLds sh;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, row = blockIdx.x;
    const void* p = (const typename L::e*)a.x + row * a.stride;
    Sum s = {NEG_INF, 0.0f, 0.0f};
    float top = NEG_INF;
    for (int c = t; c < a.chunks; c += NT) {
        const float4 v = a.part[(size_t)row * a.chunks + c];
        s.add(Sum{v.x, v.y, v.z});
        top = fmaxf(top, v.w);
    }
    s = wave_sum(s);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
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
    if (top == POS_INF) {                // its like alone, all as likely
        int n = 0;
        for (int i = t; i < a.V; i += NT) n += L::one(p, i) == POS_INF;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
        if (lane == 0) sh.count[wave] = n;
        __syncthreads();
        s = Sum{0.0f, (float)(sh.count[0] + sh.count[1] + sh.count[2] + sh.count[3]), 0.0f};
    }
    const float log_l = logf(s.l);
    auto logp = [&](float x) {
        if (top == POS_INF) return x == POS_INF ? -log_l : NEG_INF;
        return x > NEG_INF ? x - s.m - log_l : NEG_INF;
    };
    if (t == 0 && a.entropy) a.entropy[row] = top > NEG_INF ? fmaxf(log_l - s.u / s.l, 0.0f) : 0.0f;
    for (int i = t; i < a.n_targets; i += NT) {
        const int64_t at = (int64_t)row * a.n_targets + i;
        const int tok = a.targets[at];
        a.logp[at] = (unsigned)tok < (unsigned)a.V ? logp(L::one(p, tok)) : NEG_INF;
    }
    if constexpr (TOP) {
        const uint32_t* most = a.most + (size_t)row * a.groups;
        auto group = [&](int g) -> uint64_t {
            const uint32_t k = g < a.groups ? most[g] : 0;
            return k ? comp_of(k, g) : 0;
        };
        int n;
        if (a.groups <= DIRECT) {
            n = pick(sh, a.groups, a.n_top, group, sh.groups);
        } else {
            // bundles of OVER groups first, by the same argument
            const int bundles = (a.groups + OVER - 1) / OVER;
            for (int b = wave; b < bundles; b += NW) {
                const int g = b * OVER + lane;
                uint32_t k = g < a.groups ? most[g] : 0;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) k = max(k, __shfl_xor(k, d));
                if (lane == 0) sh.bundle[b] = k;
            }
            __syncthreads();
            n = pick(sh, bundles, a.n_top, [&](int b) -> uint64_t { return sh.bundle[b] ? comp_of(sh.bundle[b], b) : 0; },
                     sh.tokens);
            n = pick(sh, n * OVER, a.n_top,
                     [&](int i) { return group((int)index_of(sh.tokens[i / OVER]) * OVER + i % OVER); }, sh.groups);
        }
        n = pick(sh, n * GS, a.n_top,
                 [&](int i) -> uint64_t {
                     const int tok = (int)index_of(sh.groups[i / GS]) * GS + i % GS;
                     const uint32_t k = tok < a.V ? order_bits(L::one(p, tok)) : 0;
                     return k ? comp_of(k, tok) : 0;
                 },
                 sh.tokens);
        for (int i = t; i < a.n_top; i += NT) {
            const int64_t at = (int64_t)row * a.n_top + i;
            a.top[at] = i < n ? (int)index_of(sh.tokens[i]) : -1;
            a.top_logp[at] = i < n ? logp(from_bits((uint32_t)(sh.tokens[i] >> 32))) : NEG_INF;
        }
    }
}

struct LpPlan {
    int chunk, chunks, groups;
    size_t most, bytes;
};

// Chunks of whole loads of a workgroup, as many as give the card about 2 048
// workgroups; at most 32 768 tokens, so that a thread adds up no more than 128
// before sums meet in pairs.
LpPlan plan(int n, int V, int n_top, int VE) {
    LpPlan p;
    const int unit = NT * VE;
    int c = (2048 + n - 1) / n;
    if (c < (V + 32767) / 32768) c = (V + 32767) / 32768;
    p.chunk = ((V + c - 1) / c + unit - 1) / unit * unit;
    p.chunks = (V + p.chunk - 1) / p.chunk;
    p.groups = n_top ? (V + GL * VE - 1) / (GL * VE) : 0;
    p.most = (size_t)n * p.chunks * sizeof(float4);
    p.bytes = p.most + (size_t)n * p.groups * 4;
    return p;
}

template <typename L> void launch(const LpArgs& a, int n, hipStream_t st) {
    const dim3 g((unsigned)n * a.chunks);
    if (a.n_top) {
        hipLaunchKernelGGL((k_lp_part<L, true>), g, dim3(NT), 0, st, a);
        hipLaunchKernelGGL((k_lp_row<L, true>), dim3(n), dim3(NT), 0, st, a);
    } else {
        hipLaunchKernelGGL((k_lp_part<L, false>), g, dim3(NT), 0, st, a);
        hipLaunchKernelGGL((k_lp_row<L, false>), dim3(n), dim3(NT), 0, st, a);
    }
    LAUNCHED("k_lp_part/row");
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
    if (type == DPUF_AMD_F32) launch<F32L>(a, n, ST(s));
    else if (type == DPUF_AMD_BF16) launch<H16L<Bf16>>(a, n, ST(s));
    else launch<H16L<Fp16>>(a, n, ST(s));
}

}  // extern "C"
