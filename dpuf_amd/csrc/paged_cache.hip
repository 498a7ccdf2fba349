// paged_cache.hip -- the operators that write a paged KV cache: RoPE with the
// append of new rows, the attention weight each cached row accumulates, and
// eviction by it.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hip_internal.h"
#include "paged.h"

namespace {

// ---------------------------------------------------------------------------
// RoPE + append.  A head's columns are spread over HD / 8 lanes, 8 each; a
// group of lanes keeps its columns for every head it takes, so the angles are
// worked out once per row and lane: in turns, in 64 bits (a position of 2^31
// times a frequency keeps 2^-22 of a turn), reduced to half a turn, then in
// fp32.  Pairs half the rotated columns apart meet through LDS within a wave.
// Bound by latency at few rows (8 of 32 and 8 + 8 heads of 128: 5.4 us; one row
// of them all takes three workgroups) and nearly so at 512 (7.3 us, 1.7 TB/s).
// With several position axes a pair's angle takes the position on its axis, by
// compares with the sections' ends or by the remainder of the pair's number: 6.9
// and 8.8 us for those rows.
// ---------------------------------------------------------------------------
struct RaArgs {
    DpufAmdBatch b;
    DpufAmdPages p;
    int shift, nq;
    const double* turns;
    int rot, inter;
    float mscale;
    const int* pos;
    const void *q, *k, *v;
    int64_t qs, ks, vs;
    const float *qn, *kn;
    float eps;
    uint16_t* q_out;
};

// Position axes: pair j's axis, by the sections' ends or in turn.
struct AxArgs {
    int n, in_turn;
    int end[3];         // pairs of the axes up to this one; in turn: past the axis's last pair (of axes 1 to 3)
    uint32_t inv;       // 2^16 / n, rounded up: j / n of j below 256
    int64_t stride;
};
DEV int axis_of(const AxArgs& x, int j) {
    if (!x.in_turn) return (j >= x.end[0]) + (j >= x.end[1]) + (j >= x.end[2]);
    const int a = j - (int)((uint32_t)j * x.inv >> 16) * x.n;
    return a > 0 && j < (a == 1 ? x.end[0] : a == 2 ? x.end[1] : x.end[2]) ? a : 0;
}

template <bool F32, typename T> struct Raw8 {
    u32x4 w[F32 ? 2 : 1];
    DEV void load(const void* base, int64_t at) {
        const u32x4* p = (const u32x4*)((const char*)base + at * (F32 ? 4 : 2));
        w[0] = p[0];
        if (F32) w[F32 ? 1 : 0] = p[1];
    }
    DEV void get(float* x) const {
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __uint_as_float(w[i >> 2][i & 3]);
        } else {
            const typename T::v8 a = vec_of<typename T::v8>(w[0]);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = (float)a[i];
        }
    }
};

template <typename TI, bool F32, typename T, int HD, bool AX> DEV void rope_row(const RaArgs& a, const AxArgs& ax) {
    constexpr int LH = HD / 8;                 // lanes of a head
    constexpr int GROUPS = 256 / LH;
    __shared__ float xs[256 * 8];
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x;
    const int sub = threadIdx.x % LH, grp = threadIdx.x / LH;
    const int c0 = 8 * sub, half = a.rot >> 1;
    const int nkv = a.p.n_kv_heads, heads = a.nq + 2 * nkv;
    // the first heads' columns, whose place is known, before the row's
    // sequence is looked for; later ones a turn ahead
    auto fetch = [&](int h0) {
        Raw8<F32, TI> r = {};
        const int hh = h0 + grp;
        if (hh < a.nq) r.load(a.q, row * a.qs + (int64_t)hh * HD + c0);
        else if (hh < a.nq + nkv) r.load(a.k, row * a.ks + (int64_t)(hh - a.nq) * HD + c0);
        else if (hh < heads) r.load(a.v, row * a.vs + (int64_t)(hh - a.nq - nkv) * HD + c0);
        return r;
    };
    Raw8<F32, TI> next = fetch(GROUPS * blockIdx.y);
    const double pos = (double)a.pos[row];
    double pos1 = 0.0, pos2 = 0.0, pos3 = 0.0;
    if constexpr (AX) {
        pos1 = ax.n > 1 ? (double)a.pos[row + ax.stride] : 0.0;
        pos2 = ax.n > 2 ? (double)a.pos[row + 2 * ax.stride] : 0.0;
        pos3 = ax.n > 3 ? (double)a.pos[row + 3 * ax.stride] : 0.0;
    }
    const int s = pg_seq_of_row(a.b, row, lane);
    if (s < 0) return;
    const PgSeq sq = pg_seq(a.b, a.shift, s);
    if (row < sq.r0 || row >= sq.r0 + sq.n) return;
    const int slot = sq.ctx - sq.n + row - sq.r0;
    int page = -1;
    if (slot >= 0 && slot < sq.ctx) page = pg_page(a.b, a.shift, s, slot);
    const bool put = (unsigned)page < (unsigned)a.p.n_pages;
    const int in_page = slot & (a.p.page_size - 1);

    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int c = c0 + e;
        cs[e] = 1.0f;
        sn[e] = 0.0f;
        if (c < a.rot) {
            const int j = a.inter ? c >> 1 : (c < half ? c : c - half);
            double at = pos;
            if constexpr (AX) {
                const int axis = axis_of(ax, j);
                at = axis == 0 ? pos : axis == 1 ? pos1 : axis == 2 ? pos2 : pos3;
            }
            const double t = at * a.turns[j];
            const float f = (float)(t - rint(t));
            float si, co;
            sincospif(2.0f * f, &si, &co);
            const bool second = a.inter ? (c & 1) : c >= half;
            cs[e] = co * a.mscale;
            sn[e] = (second ? si : -si) * a.mscale;
        }
    }
    for (int h0 = GROUPS * blockIdx.y; h0 < heads; h0 += GROUPS * gridDim.y) {
        const int hh = h0 + grp;
        const bool on = hh < heads;
        const int kind = hh < a.nq ? 0 : hh < a.nq + nkv ? 1 : 2;    // q, k, v
        const int kh = kind == 0 ? 0 : kind == 1 ? hh - a.nq : hh - a.nq - nkv;
        float x[8];
        next.get(x);
        if (h0 + GROUPS * gridDim.y < heads) next = fetch(h0 + GROUPS * gridDim.y);
        const float* nw = kind == 0 ? a.qn : kind == 1 ? a.kn : nullptr;
        if (a.qn || a.kn) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) ss = fmaf(x[e], x[e], ss);
#pragma unroll
            for (int d = 1; d < LH; d <<= 1) ss += __shfl_xor(ss, d);
            if (nw) {
                const float r = 1.0f / sqrtf(ss / (float)HD + a.eps);
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = x[e] * r * nw[c0 + e];
            }
        }
        float y[8];
        if (a.inter) {
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = x[e ^ 1];
        } else {
            float* mine = xs + grp * HD;
            lds_order();
#pragma unroll
            for (int e = 0; e < 8; e += 4) *(float4*)(mine + c0 + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
            lds_order();
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int c = c0 + e;
                y[e] = mine[c < half ? c + half : c < a.rot ? c - half : c];
            }
        }
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            float o0 = x[e], o1 = x[e + 1];
            if (kind != 2) {
                if (c0 + e < a.rot) o0 = fmaf(x[e], cs[e], y[e] * sn[e]);
                if (c0 + e + 1 < a.rot) o1 = fmaf(x[e + 1], cs[e + 1], y[e + 1] * sn[e + 1]);
            }
            w[e >> 1] = pack2<T>(o0, o1);
        }
        if (!on) continue;
        if (kind == 0) {
            *(u32x4*)(a.q_out + ((int64_t)row * a.nq + hh) * HD + c0) = w;
        } else if (put) {
            uint16_t* dst = (uint16_t*)(kind == 1 ? a.p.k : a.p.v);
            *(u32x4*)(dst + (int64_t)page * a.p.page_stride + kh * a.p.head_stride + in_page * a.p.row_stride + c0) = w;
            if (kind == 1 && a.p.w && sub == 0)
                a.p.w[((size_t)page * nkv + kh) * a.p.page_size + in_page] = 0.0f;
        }
    }
}

template <typename TI, bool F32, typename T, int HD> __global__ __launch_bounds__(256) void k_rope_append(RaArgs a) {
    rope_row<TI, F32, T, HD, false>(a, AxArgs());
}
template <typename TI, bool F32, typename T, int HD>
__global__ __launch_bounds__(256) void k_rope_append_axes(RaArgs a, AxArgs ax) {
    rope_row<TI, F32, T, HD, true>(a, ax);
}

// ---------------------------------------------------------------------------
// Attention weights of cached rows: w' = decay w + sum over packed rows of
// exp(scale q.k - lse).  The keys stay: a wave holds KB x 32 of them as the
// left operand of S^T = K Q^T and walks the sequence's rows, 32 at a time,
// adding the exponentials of its keys in registers; the 32 rows of a step are
// the lanes, added up once at the end in one order.  A workgroup is KG x RG
// waves: KG of them hold different keys, RG share keys and take every RG-th
// step, their sums joined in LDS in one order.  Its queries go through LDS, a
// step ahead, so that each is read from memory once for all its keys (as the
// matrix operand straight from the L1, 32 bytes of a row a load, it was that
// which took the time: 256 rows of 4 heads, 8 kv heads over 4 096 keys 24.3 us
// against 20.4).  Bound then by the matrix instructions and, of about the same
// length, the exponentials and the queries' way through LDS.
// ---------------------------------------------------------------------------
struct PwArgs {
    DpufAmdBatch b;
    DpufAmdPages p;
    int shift, nq, G;
    const uint16_t* q;
    float c2;
    const float* lse;
    float decay;
    const float* w_in;
    int lo, hi;         // packed rows of the sequences that the few-row kernel (up to hi), the other (above lo) takes
};

// Sum over the 16 lanes of a row, in all of them.
DEV float row_sum(float v) {
#define ROW_ROR(n) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + n, 0xF, 0xF, false))
    ROW_ROR(8);
    ROW_ROR(4);
    ROW_ROR(2);
    ROW_ROR(1);
#undef ROW_ROR
    return v;
}

template <typename T, int HD, int KB, int KG, int RG>
__global__ __launch_bounds__(64 * KG * RG) void k_pa_weights(PwArgs a) {
    constexpr int NC = HD / 16, KEYS = 32 * KB * KG;
    constexpr int CH = HD / 8, RP = 64 * KG * RG / CH, ROWS = 32 * RG, NP = ROWS / RP, QP = HD + 8;
    typedef typename T::v8 v8;
    __shared__ float part[RG - 1][KEYS];
    __shared__ __align__(16) uint16_t lq[2][ROWS * QP];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, h = lane >> 5, kg = wave % KG, rg = wave / KG;
    const float NEG_INF = -__builtin_huge_valf();
    // r / G by a product: exact for r below 2^27 and G up to 32
    const uint32_t inv = 0xffffffffu / (uint32_t)a.G + 1;
    auto by_g = [&](int r) { return a.G == 1 ? r : (int)__umulhi((uint32_t)r, inv); };
    // a workgroup's tiles: kv heads fastest, then the tiles of the sequences
    // with more than `lo` packed rows, one sequence after the other
    for (int64_t it = blockIdx.x;; it += gridDim.x) {
        int64_t tile = it / a.p.n_kv_heads;
        const int kvh = (int)(it - tile * a.p.n_kv_heads);
        int s = a.b.n_seqs == 1 ? 0 : -1;
        for (int s0 = 0; s0 < a.b.n_seqs && s < 0; s0 += 64) {
            long long n = 0;
            if (s0 + lane < a.b.n_seqs) {
                const PgSeq q = pg_seq(a.b, a.shift, s0 + lane);
                n = q.n * a.G > a.lo ? (q.ctx + KEYS - 1) / KEYS : 0;
            }
            long long sum = n;
            for (int d = 1; d < 64; d <<= 1) {
                const long long o = __shfl_up(sum, d);
                if (lane >= d) sum += o;
            }
            const uint64_t past = __ballot(sum > tile);
            const int at = past ? __ffsll((unsigned long long)past) - 1 : 63;
            tile -= __shfl(past ? sum - n : sum, at);
            if (past) s = s0 + at;
        }
        s = __builtin_amdgcn_readfirstlane(s);
        if (s < 0) return;
        const PgSeq sq = pg_seq(a.b, a.shift, s);
        const int rows = sq.n * a.G;
        if (tile * KEYS >= sq.ctx) return;
        const int base0 = __builtin_amdgcn_readfirstlane((int)tile) * KEYS, base = base0 + 32 * KB * kg;
        v8 kf[KB][NC];
#pragma unroll
        for (int b = 0; b < KB; b++) {
            const int key = min(base + 32 * b + col, sq.ctx - 1);
            const int page = pg_page(a.b, a.shift, s, key);
            const bool in = (unsigned)page < (unsigned)a.p.n_pages;
            const uint16_t* kp = (const uint16_t*)a.p.k + (size_t)(in ? page : 0) * a.p.page_stride +
                                 (size_t)kvh * a.p.head_stride +
                                 (size_t)(key & (a.p.page_size - 1)) * a.p.row_stride + 8 * h;
#pragma unroll
            for (int c = 0; c < NC; c++) kf[b][c] = vec_of<v8>(*(const u32x4*)(kp + 16 * c));
        }
        float acc[KB][16] = {};
        // rows before the first key of the tile see none of it
        const int first = max(0, base0 - (sq.ctx - sq.n)) * a.G & ~31;
        // a step's queries go to LDS, once for all waves, while the step before
        // it is worked out; the lse to registers
        const int lr = threadIdx.x / CH, lc = 8 * (threadIdx.x % CH);
        u32x4 qn[NP];
        auto load = [&](int r0) {
#pragma unroll
            for (int u = 0; u < NP; u++) {
                const int r = r0 + u * RP + lr, i = by_g(r);
                const size_t row = (size_t)(sq.r0 + i) * a.nq + kvh * a.G + (r - i * a.G);
                qn[u] = r < rows ? *(const u32x4*)(a.q + row * HD + lc) : u32x4{0, 0, 0, 0};
            }
        };
        auto store = [&](int buf) {
#pragma unroll
            for (int u = 0; u < NP; u++) *(u32x4*)(lq[buf] + (u * RP + lr) * QP + lc) = qn[u];
        };
        float ln = 0.0f;
        int qi = 0;
        auto fetch = [&](int r0) {
            const int r = r0 + 32 * rg + col;
            const bool live = r < rows;
            qi = live ? by_g(r) : 0;
            ln = live ? a.lse[(size_t)(sq.r0 + qi) * a.nq + kvh * a.G + (r - qi * a.G)] : NEG_INF;
        };
        v8 qf[NC];
        auto take = [&](int buf) {
#pragma unroll
            for (int c = 0; c < NC; c++)
                qf[c] = vec_of<v8>(*(const u32x4*)(lq[buf] + (32 * rg + col) * QP + 16 * c + 8 * h));
        };
        if (first < rows) {
            load(first);
            fetch(first);
            store(0);
            if (first + ROWS < rows) load(first + ROWS);
            __syncthreads();
            take(0);
        }
        int buf = 0;
        for (int w0 = first; w0 < rows; w0 += ROWS, buf ^= 1) {
            const int r0 = w0 + 32 * rg;
            f32x16 sc[KB];
            const f32x16 zero = {};
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int b = 0; b < KB; b++) sc[b] = T::mma32(kf[b][c], qf[c], c ? sc[b] : zero);
            // a row that saw no key (lse -infinity) or is none gives nothing
            const float l2 = ln == NEG_INF ? -NEG_INF : ln * 1.4426950408889634f;
            const int limit = ln != NEG_INF ? sq.ctx - sq.n + qi : -1;
            // the next step's queries: to LDS, and from there while the
            // exponentials are worked out
            if (w0 + ROWS < rows) {
                store(buf ^ 1);
                fetch(w0 + ROWS);
                if (w0 + 2 * ROWS < rows) load(w0 + 2 * ROWS);
                __syncthreads();
                take(buf ^ 1);
            }
            // keys that the step's first row does not see, and lanes without a
            // row, key by key: whatever an infinity or NaN in K, or a row's
            // lse of NaN, makes of the others' exponentials, they give nothing
            if (base + 32 * KB - 1 > sq.ctx - sq.n + by_g(r0) || r0 + 32 > rows) {
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float e = __builtin_amdgcn_exp2f(fmaf(sc[b][i], a.c2, -l2));
                        acc[b][i] += base + 32 * b + 8 * (i >> 2) + 4 * h + (i & 3) <= limit ? e : 0.0f;
                    }
            } else {
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        acc[b][i] += __builtin_amdgcn_exp2f(fmaf(sc[b][i], a.c2, -l2));
            }
        }
        // over the 32 lanes of each half: entries i and i + 8 of the lower and
        // the upper 16 lanes are exchanged, so each 16 add up 8 entries of all
        // 32; lane i of the lower 16 then keeps entry i, of the upper 8 + i
        float mine[KB];
#pragma unroll
        for (int b = 0; b < KB; b++) {
            mine[b] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[b][i]),
                                                                __float_as_uint(acc[b][i + 8]), false, false);
                const float v = row_sum(__uint_as_float(x[0]) + __uint_as_float(x[1]));
                mine[b] = (lane & 7) == i ? v : mine[b];
            }
        }
        const int e = (lane & 7) + ((lane & 16) >> 1);                    // entry this lane keeps
        const int at0 = 8 * (e >> 2) + 4 * h + (e & 3);                    // its key among 32
        const bool keeps = !(lane & 8);
        if (rg > 0 && keeps) {
#pragma unroll
            for (int b = 0; b < KB; b++) part[rg - 1][32 * (KB * kg + b) + at0] = mine[b];
        }
        __syncthreads();
        if (rg == 0 && keeps) {
#pragma unroll
            for (int g = 0; g < RG - 1; g++)
#pragma unroll
                for (int b = 0; b < KB; b++) mine[b] += part[g][32 * (KB * kg + b) + at0];
        }
        __syncthreads();
        if (rg == 0 && keeps) {
#pragma unroll
            for (int b = 0; b < KB; b++) {
                const int kk = base + 32 * b + at0;
                if (kk >= sq.ctx) continue;
                const int pg = pg_page(a.b, a.shift, s, kk);
                if ((unsigned)pg >= (unsigned)a.p.n_pages) continue;
                const size_t at = ((size_t)pg * a.p.n_kv_heads + kvh) * a.p.page_size + (kk & (a.p.page_size - 1));
                a.p.w[at] = a.w_in ? fmaf(a.decay, a.w_in[at], mine[b]) : mine[b];
            }
        }
    }
}

// The same for few rows: bound by reading K once.  16-key blocks as the left
// operand of 16 x 16 steps, so that a load of the wave takes 64 consecutive
// bytes of 16 rows (of 32 rows 32 bytes, as above, it reached 3.8 TB/s); NB
// blocks a wave, and the next ones in flight.  24 rows of 32 heads, 8 kv heads of
// 128 over 900 to 4 096 keys: 27.6 us, 4.6 TB/s.
template <typename T, int HD>
__global__ __launch_bounds__(256) void k_pa_weights_few(PwArgs a) {
    constexpr int NC = HD / 32, NB = HD == 256 ? 2 : 4, WK = 16 * NB;
    typedef typename T::v8 v8;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g4 = lane >> 4;
    const int kvh = blockIdx.x, s = blockIdx.y;
    const PgSeq sq = pg_seq(a.b, a.shift, s);
    const int rows = sq.n * a.G;
    if (rows > a.hi) return;
    const float NEG_INF = -__builtin_huge_valf();
    const uint16_t* kp = (const uint16_t*)a.p.k + (size_t)kvh * a.p.head_stride + 8 * g4;
    const int* table = a.b.page_table + (size_t)s * a.b.table_stride;
    const int step = 4 * WK * gridDim.z, top = sq.ctx > 0 ? (sq.ctx - 1) >> a.shift : 0;
    u32x4 kn[NB][NC];
    int pn[NB];              // pages: a block of 16 keys lies in one
    auto find = [&](int base) {
#pragma unroll
        for (int b = 0; b < NB; b++) pn[b] = table[min((base + 16 * b) >> a.shift, top)];
    };
    auto load = [&](int base) {
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const bool in = (unsigned)pn[b] < (unsigned)a.p.n_pages;
            const size_t at = (size_t)(in ? pn[b] : 0) * a.p.page_stride +
                              (size_t)((base + 16 * b) & (a.p.page_size - 1)) * a.p.row_stride;
#pragma unroll
            for (int c = 0; c < NC; c++) kn[b][c] = *(const u32x4*)(kp + at + (size_t)col * a.p.row_stride + 32 * c);
        }
    };
    v8 qf[NC];
    float l2 = 0.0f;
    int limit = -1, have = -1;
    auto fetch = [&](int r0) {
        const int r = r0 + col;
        const bool live = r < rows;
        const int qi = live ? r / a.G : 0;
        const size_t row = (size_t)(sq.r0 + qi) * a.nq + kvh * a.G + (live ? r - qi * a.G : 0);
        const float ln = live ? a.lse[row] : NEG_INF;
        // a row that saw no key (lse -infinity) or is none gives nothing
        l2 = ln == NEG_INF ? -NEG_INF : ln * 1.4426950408889634f;
        limit = ln != NEG_INF ? sq.ctx - sq.n + qi : -1;
        have = r0;
#pragma unroll
        for (int c = 0; c < NC; c++)
            qf[c] = vec_of<v8>(live ? *(const u32x4*)(a.q + row * HD + 32 * c + 8 * g4) : u32x4{0, 0, 0, 0});
    };
    int base = WK * (4 * blockIdx.z + wave);
    if (base < sq.ctx) {
        find(base);
        load(base);
        if (base + step < sq.ctx) find(base + step);
    }
    for (; base < sq.ctx; base += step) {
        v8 kf[NB][NC];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int c = 0; c < NC; c++) kf[b][c] = vec_of<v8>(kn[b][c]);
        const int first = max(0, base - (sq.ctx - sq.n)) * a.G & ~15;
        if (first < rows && have != first) fetch(first);
        if (base + step < sq.ctx) {
            load(base + step);
            if (base + 2 * step < sq.ctx) find(base + 2 * step);
        }
        f32x4 acc[NB] = {};
        for (int r0 = first; r0 < rows; r0 += 16) {
            if (have != r0) fetch(r0);
            const f32x4 zero = {};
            f32x4 sc[NB];
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int b = 0; b < NB; b++) sc[b] = T::mma16(kf[b][c], qf[c], c ? sc[b] : zero);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(sc[b][i], a.c2, -l2));
                    acc[b][i] += base + 16 * b + 4 * g4 + i <= limit ? e : 0.0f;
                }
        }
        // over the 16 rows; lane 4 b + i of 16 keeps key i of block b
        float mine = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float v = row_sum(acc[b][i]);
                mine = col == 4 * b + i ? v : mine;
            }
        const int kk = base + 16 * (col >> 2) + 4 * g4 + (col & 3);
        if (col < 4 * NB && kk < sq.ctx) {
            const int pg = table[kk >> a.shift];
            if ((unsigned)pg < (unsigned)a.p.n_pages) {
                const size_t at = ((size_t)pg * a.p.n_kv_heads + kvh) * a.p.page_size + (kk & (a.p.page_size - 1));
                a.p.w[at] = a.w_in ? fmaf(a.decay, a.w_in[at], mine) : mine;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Eviction.  k_ev_pick / k_ev_pick_long: one workgroup per (sequence, kv head)
// finds the keep - sink - recent largest weights of the middle by radix
// selection on order-preserving integers (10 bits a pass from the highest bit
// in which two of them differ), then lists the kept rows in order: latency, of
// the loads (length, page, weight) and of the passes' barriers.  k_ev_move
// copies them, 16 bytes a lane, four rows in flight: bound by bytes (8
// sequences of 6 100 to 9 000 rows to 4 096, 8 kv heads of 128: 59 us, 4.6 TB/s
// read and written; one of 1 290 rows to 1 024: 4.4 us).
// ---------------------------------------------------------------------------
struct EvArgs {
    DpufAmdBatch b;
    DpufAmdPages p, d;
    int shift, dshift;
    int keep;
    const int* dtable;
    int dstride;
    const int* kept;
};
// What the selection reads: below 112 bytes of arguments a launch takes the
// host 2.7 us, above 3.7.
struct PickArgs {
    const int *ctx_len, *table;
    const float* w;
    int *kept, *new_len;
    int table_stride, shift, n_pages, nkv;
    int keep, sink, recent, lds_keys;
    DEV int ctx(int s) const { return min(max(ctx_len[s], 0), table_stride << shift); }
    DEV int page(int s, int i) const { return table[(size_t)s * table_stride + (i >> shift)]; }
    // weight of cached row i of kv head h, on page p of the pool
    DEV float weight(int p, int h, int i) const {
        return w[((((size_t)p * nkv + h) << shift) | (unsigned)(i & ((1 << shift) - 1)))];
    }
};

// Larger weight, larger integer; NaN and absent rows are 0, below every
// number (-infinity gives 0x007fffff), and -0 equals +0.
DEV uint32_t weight_key(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    if (w != w) return 0;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int EV_T = 1024;

// Inclusive sums of (a, b) over the workgroup's threads, in thread order, and
// the totals.
DEV void scan2(int& x, int& y, int& tx, int& ty, int (*sums)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int ox = __shfl_up(x, d), oy = __shfl_up(y, d);
        if (lane >= d) { x += ox; y += oy; }
    }
    if (lane == 63) { sums[wave][0] = x; sums[wave][1] = y; }
    __syncthreads();
    tx = ty = 0;
    int bx = 0, by = 0;
    for (int w = 0; w < EV_T / 64; w++) {
        if (w == wave) { bx = tx; by = ty; }
        tx += sums[w][0];
        ty += sums[w][1];
    }
    x += bx;
    y += by;
    __syncthreads();
}

// Longer rows: keys in LDS, or read again in every pass where it does not hold
// them (30 000 rows of one sequence to 4 096: 43 us with the move).
__global__ __launch_bounds__(EV_T) void k_ev_pick_long(PickArgs a) {
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ int hist[EV_T];
    __shared__ int sums[EV_T / 64][2];
    __shared__ uint32_t bits[EV_T / 64][2];
    __shared__ uint32_t sh_digit;
    __shared__ int sh_need;
    const int kvh = blockIdx.x, s = blockIdx.y, t = threadIdx.x;
    const int c = a.ctx(s), n = min(c, a.keep);
    if (kvh == 0 && t == 0) a.new_len[s] = n;
    int* kept = a.kept + ((size_t)s * a.nkv + kvh) * a.keep;
    if (c <= a.keep) {
        for (int i = t; i < n; i += EV_T) kept[i] = i;
        return;
    }
    const int lo = a.sink, hi = c - a.recent, need = a.keep - a.sink - a.recent;   // of the middle [lo, hi)
    const int mid = hi - lo;
    const bool staged = mid <= a.lds_keys;
    auto fetch = [&](int i) -> uint32_t {
        const int slot = lo + i, page = a.page(s, slot);
        if ((unsigned)page >= (unsigned)a.n_pages) return 0;
        return weight_key(a.weight(page, kvh, slot));
    };
    // the bits in which keys differ, and with a row that fits the keys in LDS
    uint32_t any = 0, all = ~0u;
    constexpr int AT = 8;          // pages, then weights, in flight
    for (int i0 = 0; i0 < mid; i0 += AT * EV_T) {
        int pg[AT];
        float w[AT];
#pragma unroll
        for (int u = 0; u < AT; u++)
            if (i0 + u * EV_T < mid) pg[u] = a.page(s, lo + min(i0 + u * EV_T + t, mid - 1));
#pragma unroll
        for (int u = 0; u < AT; u++)
            if (i0 + u * EV_T < mid) {
                const bool in = (unsigned)pg[u] < (unsigned)a.n_pages;
                w[u] = a.weight(in ? pg[u] : 0, kvh, lo + min(i0 + u * EV_T + t, mid - 1));
                if (!in) pg[u] = -1;
            }
#pragma unroll
        for (int u = 0; u < AT; u++)
            if (i0 + u * EV_T + t < mid) {
                const uint32_t k = pg[u] < 0 ? 0 : weight_key(w[u]);
                any |= k;
                all &= k;
                if (staged) keys[i0 + u * EV_T + t] = k;
            }
    }
    auto key_at = [&](int i) -> uint32_t { return staged ? keys[i] : fetch(i); };
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        any |= __shfl_xor(any, d);
        all &= __shfl_xor(all, d);
    }
    if ((t & 63) == 0) {
        bits[t >> 6][0] = any;
        bits[t >> 6][1] = all;
    }
    __syncthreads();
    for (int w = 0; w < EV_T / 64; w++) {
        any |= bits[w][0];
        all &= bits[w][1];
    }
    int top = any & ~all ? 32 - __clz((int)(any & ~all)) : 0;      // keys agree from this bit up
    uint32_t cut = top < 32 ? all >> top << top : 0;
    int ties = need;               // of the keys equal to cut, the first this many stay
    // the need-th largest key, 10 bits at a time
    while (top > 0 && need > 0) {
        const int low = top > 10 ? top - 10 : 0, mask = (1 << (top - low)) - 1;
        hist[t] = 0;
        __syncthreads();
        for (int i = t; i < mid; i += EV_T) {
            const uint32_t k = key_at(i);
            if (top == 32 || k >> top == cut >> top) atomicAdd(&hist[mask - (int)(k >> low & mask)], 1);
        }
        __syncthreads();
        // the digit, from the top, in which the count reaches what is left
        const int own = hist[t];
        int x = own, y = 0, tx, ty;
        scan2(x, y, tx, ty, sums);
        if (x >= ties && x - own < ties) {
            sh_digit = (uint32_t)(mask - t);
            sh_need = ties - (x - own);
        }
        __syncthreads();
        cut |= sh_digit << low;
        ties = sh_need;
        top = low;
    }
    __syncthreads();
    // every thread takes a run of rows; a run's places follow from the counts
    // of the runs before it
    const int per = (mid + EV_T - 1) / EV_T, b0 = min(t * per, mid), b1 = min(b0 + per, mid);
    int above = 0, equal = 0;
    if (need > 0)
        for (int i = b0; i < b1; i++) {
            const uint32_t k = key_at(i);
            above += k > cut;
            equal += k == cut;
        }
    int xa = above, xe = equal, ta, te;
    scan2(xa, xe, ta, te, sums);
    xa -= above;
    xe -= equal;
    if (need > 0) {
        int at = a.sink + xa + min(xe, ties);
        for (int i = b0; i < b1; i++) {
            const uint32_t k = key_at(i);
            if (k > cut || (k == cut && xe < ties)) kept[at++] = lo + i;
            xe += k == cut;
        }
    }
    for (int i = t; i < a.sink; i += EV_T) kept[i] = i;
    for (int i = t; i < a.recent; i += EV_T) kept[a.keep - a.recent + i] = hi + i;
}

// Rows of at most NT AT keys: they stay in registers, key u NT + t of the middle
// with thread t, and the places of the rows that stay follow from ballots, in
// row order.
template <int NT, int AT> __global__ __launch_bounds__(NT) void k_ev_pick(PickArgs a) {
    constexpr int BINS = 1024, OWN = BINS / NT, NW = NT / 64, CELLS = AT * NW, LC = (CELLS + 63) / 64;
    __shared__ int hist[BINS];
    __shared__ int sums[NW];
    __shared__ uint32_t bits[NW][2];
    __shared__ uint32_t sh_digit;
    __shared__ int sh_need;
    __shared__ int cells[2][64 * LC];      // rows above the cut, equal to it, of 64 consecutive ones
    const int kvh = blockIdx.x, s = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int c = a.ctx(s), n = min(c, a.keep);
    if (kvh == 0 && t == 0) a.new_len[s] = n;
    int* kept = a.kept + ((size_t)s * a.nkv + kvh) * a.keep;
    if (c <= a.keep) {
        for (int i = t; i < n; i += NT) kept[i] = i;
        return;
    }
    const int lo = a.sink, hi = c - a.recent, need = a.keep - a.sink - a.recent, mid = hi - lo;
    int pg[AT];
    uint32_t k[AT];
#pragma unroll
    for (int u = 0; u < AT; u++)
        if (u * NT < mid) pg[u] = a.page(s, lo + min(u * NT + t, mid - 1));
#pragma unroll
    for (int u = 0; u < AT; u++) {
        if (u * NT >= mid) continue;
        const bool in = (unsigned)pg[u] < (unsigned)a.n_pages;
        const float w = a.weight(in ? pg[u] : 0, kvh, lo + min(u * NT + t, mid - 1));
        k[u] = in ? weight_key(w) : 0;
    }
    for (int i = t; i < a.sink; i += NT) kept[i] = i;
    for (int i = t; i < a.recent; i += NT) kept[a.keep - a.recent + i] = hi + i;
    if (need == 0) return;
    // the bits in which keys differ
    uint32_t any = 0, all = ~0u;
#pragma unroll
    for (int u = 0; u < AT; u++)
        if (u * NT + t < mid) {
            any |= k[u];
            all &= k[u];
        }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        any |= __shfl_xor(any, d);
        all &= __shfl_xor(all, d);
    }
    if (lane == 0) {
        bits[wave][0] = any;
        bits[wave][1] = all;
    }
#pragma unroll
    for (int e = 0; e < OWN; e++) hist[OWN * t + e] = 0;
    if (t < 64 * LC - CELLS) cells[0][CELLS + t] = cells[1][CELLS + t] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) {
        any |= bits[w][0];
        all &= bits[w][1];
    }
    int top = any & ~all ? 32 - __clz((int)(any & ~all)) : 0;      // keys agree from this bit up
    uint32_t cut = top < 32 ? all >> top << top : 0;
    int ties = need;               // of the keys equal to cut, the first this many stay
    // the need-th largest key, 10 bits at a time
    while (top > 0) {
        const int low = top > 10 ? top - 10 : 0, mask = (1 << (top - low)) - 1;
#pragma unroll
        for (int u = 0; u < AT; u++)
            if (u * NT + t < mid && (top == 32 || k[u] >> top == cut >> top))
                atomicAdd(&hist[mask - (int)(k[u] >> low & mask)], 1);
        __syncthreads();
        // the digit, from the top, in which the count reaches what is left
        int own[OWN], mine = 0;
#pragma unroll
        for (int e = 0; e < OWN; e++) mine += own[e] = hist[OWN * t + e];
        int x = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(x, d);
            if (lane >= d) x += o;
        }
        if (lane == 63) sums[wave] = x;
#pragma unroll
        for (int e = 0; e < OWN; e++) hist[OWN * t + e] = 0;
        __syncthreads();
        x -= mine;
#pragma unroll
        for (int w = 0; w < NW - 1; w++) x += w < wave ? sums[w] : 0;
#pragma unroll
        for (int e = 0; e < OWN; e++) {
            if (x < ties && x + own[e] >= ties) {
                sh_digit = (uint32_t)(mask - (OWN * t + e));
                sh_need = ties - x;
            }
            x += own[e];
        }
        __syncthreads();
        cut |= sh_digit << low;
        ties = sh_need;
        top = low;
    }
    // places: above the cut, or one of the first `ties` equal to it
    uint64_t above[AT], equal[AT];
#pragma unroll
    for (int u = 0; u < AT; u++) {
        const bool mine = u * NT + t < mid;
        above[u] = __ballot(mine && k[u] > cut);
        equal[u] = __ballot(mine && k[u] == cut);
        if (lane == 0) {
            cells[0][u * NW + wave] = __popcll(above[u]);
            cells[1][u * NW + wave] = __popcll(equal[u]);
        }
    }
    __syncthreads();
    if (wave == 0) {         // the cells' counts become those of the cells before them
        int ca[LC], ce[LC], sa = 0, se = 0;
#pragma unroll
        for (int e = 0; e < LC; e++) {
            ca[e] = cells[0][LC * lane + e];
            ce[e] = cells[1][LC * lane + e];
            sa += ca[e];
            se += ce[e];
        }
        int xa = sa, xe = se;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int oa = __shfl_up(xa, d), oe = __shfl_up(xe, d);
            if (lane >= d) xa += oa, xe += oe;
        }
        xa -= sa;
        xe -= se;
#pragma unroll
        for (int e = 0; e < LC; e++) {
            cells[0][LC * lane + e] = xa;
            cells[1][LC * lane + e] = xe;
            xa += ca[e];
            xe += ce[e];
        }
    }
    __syncthreads();
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int u = 0; u < AT; u++) {
        if (u * NT >= mid) continue;
        const int ba = cells[0][u * NW + wave] + __popcll(above[u] & below);
        const int be = cells[1][u * NW + wave] + __popcll(equal[u] & below);
        if (u * NT + t < mid && (k[u] > cut || (k[u] == cut && be < ties)))
            kept[a.sink + ba + min(be, ties)] = lo + u * NT + t;
    }
}

template <int HD>
__global__ __launch_bounds__(256) void k_ev_move(EvArgs a) {
    constexpr int CH = HD / 8, RP = 256 / CH, NR = 4;
    const int kvh = blockIdx.x, s = blockIdx.y;
    const int c = pg_ctx(a.b, a.shift, s), n = min(c, a.keep);
    const int* kept = a.kept + ((size_t)s * a.p.n_kv_heads + kvh) * a.keep;
    const int sub = threadIdx.x % CH, rw = threadIdx.x / CH;
    for (int i0 = blockIdx.z * RP * NR; i0 < n; i0 += gridDim.z * RP * NR) {
        int from[NR], sp[NR], dp[NR];
#pragma unroll
        for (int u = 0; u < NR; u++) {
            const int i = i0 + u * RP + rw;
            from[u] = i < n ? kept[i] : 0;
            dp[u] = i < n ? a.dtable[(size_t)s * a.dstride + (i >> a.dshift)] : -1;
        }
#pragma unroll
        for (int u = 0; u < NR; u++) sp[u] = pg_page(a.b, a.shift, s, min(max(from[u], 0), c - 1));
        u32x4 kv[NR], vv[NR];
        float w[NR];
#pragma unroll
        for (int u = 0; u < NR; u++) {
            kv[u] = vv[u] = u32x4{0, 0, 0, 0};
            w[u] = 0.0f;
            if ((unsigned)sp[u] < (unsigned)a.p.n_pages) {
                const int in_page = from[u] & (a.p.page_size - 1);
                const size_t at = (size_t)sp[u] * a.p.page_stride + (size_t)kvh * a.p.head_stride +
                                  (size_t)in_page * a.p.row_stride + 8 * sub;
                kv[u] = *(const u32x4*)((const uint16_t*)a.p.k + at);
                vv[u] = *(const u32x4*)((const uint16_t*)a.p.v + at);
                if (sub == 0) w[u] = a.p.w[((size_t)sp[u] * a.p.n_kv_heads + kvh) * a.p.page_size + in_page];
            }
        }
#pragma unroll
        for (int u = 0; u < NR; u++) {
            const int i = i0 + u * RP + rw;
            if (i >= n || (unsigned)dp[u] >= (unsigned)a.d.n_pages) continue;
            const int in_page = i & (a.d.page_size - 1);
            const size_t at = (size_t)dp[u] * a.d.page_stride + (size_t)kvh * a.d.head_stride +
                              (size_t)in_page * a.d.row_stride + 8 * sub;
            *(u32x4*)((uint16_t*)a.d.k + at) = kv[u];
            *(u32x4*)((uint16_t*)a.d.v + at) = vv[u];
            if (sub == 0) a.d.w[((size_t)dp[u] * a.p.n_kv_heads + kvh) * a.d.page_size + in_page] = w[u];
        }
    }
}

template <typename T, int HD, int KB, int KG, int RG>
void weights_many(const PwArgs& a, int64_t ctx, int64_t rows_of_tiles, hipStream_t st) {
    const int64_t tiles = (ctx + 32 * KB * KG - 1) / (32 * KB * KG) * rows_of_tiles, cus = dpuf_hip_cu_count();
    hipLaunchKernelGGL((k_pa_weights<T, HD, KB, KG, RG>), dim3((unsigned)(tiles < cus ? tiles : cus)),
                       dim3(64 * KG * RG), 0, st, a);
}

// Which kernel takes which sequences: those of up to LIM packed rows the
// few-row one (eight chunks of 80 rows over 1 000 to 3 000 keys 22 us against
// 39, of 256 rows 41 against 47, but a single one of 256 over 4 096 14 against
// 11), the others the other, a launch each where there may be both (one chunk
// of 256 rows of 4 heads and 31 single rows over 500 to 6 000 keys 81 us, 381
// by the few-row kernel alone).  One sequence, or a batch whose tiles would
// leave CUs idle, is one launch (a chunk of 131 rows and two single ones over
// 900 keys 14.6 us against 20.8).
//
// A workgroup has as few keys as gives every CU at most one tile, since its
// steps are latency rather than work while the card is not full: 256 rows of 8
// heads, 2 kv heads of 64 columns over 4 096 keys 10.5 us with 32 keys (256
// tiles), 14.5 with 64, 22 with 128; 256 rows of 4 heads, 8 kv heads of 128
// over 2 000 19.7, 12.6, 18.5 (500, 250, 125 tiles); over 4 096 39, 24.5, 20.4.
constexpr int LIM = 128;
template <typename T, int HD> void weights_hd(PwArgs a, int64_t ctx, hipStream_t st) {
    const int64_t G = a.G, nkv = a.p.n_kv_heads, n = a.b.n_seqs, packed = a.b.n_rows * G, cus = dpuf_hip_cu_count();
    constexpr int MOST = HD == 256 ? 64 : 128;           // keys that registers and LDS hold
    const bool none = a.b.n_rows <= n || packed <= LIM;
    const bool all = !none && (n == 1 || (ctx + MOST - 1) / MOST * nkv * n <= cus);
    a.lo = all ? -1 : LIM;
    a.hi = none ? INT32_MAX : LIM;
    if (!none) {
        // sequences of chunks: at most, and if they have 256 packed rows each
        const int64_t most = all || packed / (LIM + 1) > n ? n : packed / (LIM + 1);
        const int64_t about = ((a.b.n_rows - n) * G + 255) / 256, by = nkv * (all || about > n ? n : about);
        if constexpr (HD == 256) {
            weights_many<T, HD, 1, 2, 4>(a, ctx, nkv * most, st);
        } else {
            if ((ctx + 31) / 32 * by <= cus) weights_many<T, HD, 1, 1, 8>(a, ctx, nkv * most, st);
            else if ((ctx + 63) / 64 * by <= cus) weights_many<T, HD, 1, 2, 4>(a, ctx, nkv * most, st);
            else weights_many<T, HD, 2, 2, 4>(a, ctx, nkv * most, st);
        }
    }
    if (all) return;
    // a decode step's workgroups, about four a CU, walk their keys with the
    // next ones in flight
    const int64_t by = nkv * n, keys = HD == 256 ? 128 : 256, tiles = (ctx + keys - 1) / keys;
    const int64_t few = (1024 + by - 1) / by, z = few < tiles ? few : tiles;
    const dim3 g((unsigned)nkv, (unsigned)n, (unsigned)z);
    hipLaunchKernelGGL((k_pa_weights_few<T, HD>), g, dim3(256), 0, st, a);
}
template <typename TI, bool F32, typename T, int HD>
void rope_go(const RaArgs& a, const AxArgs* ax, dim3 g, hipStream_t st) {
    if (ax) hipLaunchKernelGGL((k_rope_append_axes<TI, F32, T, HD>), g, dim3(256), 0, st, a, *ax);
    else hipLaunchKernelGGL((k_rope_append<TI, F32, T, HD>), g, dim3(256), 0, st, a);
}
template <typename TI, bool F32, typename T> void rope_hd(const RaArgs& a, const AxArgs* ax, dim3 g, hipStream_t st) {
    switch (a.p.head_dim) {
        case 64: rope_go<TI, F32, T, 64>(a, ax, g, st); break;
        case 128: rope_go<TI, F32, T, 128>(a, ax, g, st); break;
        default: rope_go<TI, F32, T, 256>(a, ax, g, st); break;
    }
}
template <typename T> void rope_in(const RaArgs& a, const AxArgs* ax, int in_type, dim3 g, hipStream_t st) {
    if (in_type == DPUF_AMD_F32) rope_hd<Bf16, true, T>(a, ax, g, st);
    else if (in_type == DPUF_AMD_BF16) rope_hd<Bf16, false, T>(a, ax, g, st);
    else rope_hd<Fp16, false, T>(a, ax, g, st);
}

}  // namespace

extern "C" {

void dpuf_hip_rope_append(void* s, const DpufAmdBatch* b, const DpufAmdPages* p, const DpufAmdRope* r,
                          const DpufAmdRopeAxes* x, const int32_t* pos, int64_t pos_stride, int32_t in_type, int32_t nq,
                          const void* q, const void* k, const void* v, int64_t qs, int64_t ks, int64_t vs,
                          const float* qn, const float* kn, float eps, void* q_out) {
    RaArgs a;
    a.b = *b;
    a.p = *p;
    a.shift = __builtin_ctz(p->page_size);
    a.nq = nq;
    a.turns = r->turns;
    a.rot = r->rot_dim;
    a.inter = r->interleaved != 0;
    a.mscale = r->scale;
    a.pos = pos;
    a.q = q;
    a.k = k;
    a.v = v;
    a.qs = qs;
    a.ks = ks;
    a.vs = vs;
    a.qn = qn;
    a.kn = kn;
    a.eps = eps;
    a.q_out = (uint16_t*)q_out;
    // a row's heads by one workgroup, or spread over several while the rows
    // alone do not give every CU two (256 rows of 32 heads and 8 + 8 of 128, three
    // turns a row: 8.0 us by two workgroups a row against 8.9 by one, 64 6.6 by
    // three and 8.3, 512 9.8 and 10.3, but bf16 ones without norms 8.3 and 8.0)
    const int groups = 256 / (p->head_dim / 8), turns = (nq + 2 * p->n_kv_heads + groups - 1) / groups;
    int y = 2 * dpuf_hip_cu_count() / b->n_rows;
    if (y < 1) y = 1;
    if (y > turns) y = turns;
    const dim3 g(b->n_rows, y);
    AxArgs ax = {};
    if (x) {
        ax.n = x->n_axes;
        ax.in_turn = x->in_turn != 0;
        for (int i = 0, end = 0; i < 3; i++) {
            end += i < ax.n ? x->sections[i] : 0;
            ax.end[i] = !ax.in_turn ? end : i + 1 < ax.n ? ax.n * x->sections[i + 1] : 0;
        }
        ax.inv = 65536 / ax.n + 1;
        ax.stride = pos_stride;
    }
    if (p->type == DPUF_AMD_BF16) rope_in<Bf16>(a, x ? &ax : nullptr, in_type, g, ST(s));
    else rope_in<Fp16>(a, x ? &ax : nullptr, in_type, g, ST(s));
    LAUNCHED("k_rope_append");
}

void dpuf_hip_paged_attn_weights(void* s, const DpufAmdBatch* b, const DpufAmdPages* p, int32_t nq, const void* q,
                                 float scale, const float* lse, float decay, const float* w_in) {
    PwArgs a;
    a.b = *b;
    a.p = *p;
    a.shift = __builtin_ctz(p->page_size);
    a.nq = nq;
    a.G = nq / p->n_kv_heads;
    a.q = (const uint16_t*)q;
    a.c2 = scale * 1.4426950408889634f;
    a.lse = lse;
    a.decay = decay;
    a.w_in = w_in;
    const int64_t cap = (int64_t)b->table_stride * p->page_size;
    const int64_t ctx = b->max_ctx < 1 ? 1 : b->max_ctx < cap ? b->max_ctx : cap;
    const bool bf = p->type == DPUF_AMD_BF16;
    switch (p->head_dim) {
        case 64: bf ? weights_hd<Bf16, 64>(a, ctx, ST(s)) : weights_hd<Fp16, 64>(a, ctx, ST(s)); break;
        case 128: bf ? weights_hd<Bf16, 128>(a, ctx, ST(s)) : weights_hd<Fp16, 128>(a, ctx, ST(s)); break;
        default: bf ? weights_hd<Bf16, 256>(a, ctx, ST(s)) : weights_hd<Fp16, 256>(a, ctx, ST(s));
    }
    LAUNCHED("k_pa_weights");
}

void dpuf_hip_paged_evict(void* s, const DpufAmdBatch* b, const DpufAmdPages* p, int32_t keep, int32_t sink,
                          int32_t recent, const DpufAmdPages* d, const int32_t* dtable, int32_t dstride, int32_t* kept,
                          int32_t* new_len) {
    EvArgs a;
    a.b = *b;
    a.p = *p;
    a.d = *d;
    a.shift = __builtin_ctz(p->page_size);
    a.dshift = __builtin_ctz(d->page_size);
    a.keep = keep;
    a.dtable = dtable;
    a.dstride = dstride;
    a.kept = kept;
    PickArgs k;
    k.ctx_len = b->ctx_len;
    k.table = b->page_table;
    k.w = p->w;
    k.kept = kept;
    k.new_len = new_len;
    k.table_stride = b->table_stride;
    k.shift = a.shift;
    k.n_pages = p->n_pages;
    k.nkv = p->n_kv_heads;
    k.keep = keep;
    k.sink = sink;
    k.recent = recent;
    const int64_t cap = (int64_t)b->table_stride * p->page_size;
    const dim3 gp(p->n_kv_heads, b->n_seqs);
    k.lds_keys = (int)(cap < 36864 ? cap : 36864);      // 144 KB of the 160
    // what the tables bound the rows by; the whole call, one sequence of 8 kv
    // heads: 1 290 rows 14.4 us by the long rows' kernel, 12.7 by <1024, 4>,
    // 11.6 by <512, 4>; 4 000 rows 17.2 and 14.6; 8 000 rows 23.3, and 20 by
    // <1024, 8>; 9 000 rows 23.5, and 22 by <1024, 12>; 16 000 rows 32.4, and
    // 28.6 by <1024, 16>
    if (cap <= 2048) hipLaunchKernelGGL((k_ev_pick<512, 4>), gp, dim3(512), 0, ST(s), k);
    else if (cap <= 4096) hipLaunchKernelGGL((k_ev_pick<1024, 4>), gp, dim3(1024), 0, ST(s), k);
    else if (cap <= 8192) hipLaunchKernelGGL((k_ev_pick<1024, 8>), gp, dim3(1024), 0, ST(s), k);
    else if (cap <= 12288) hipLaunchKernelGGL((k_ev_pick<1024, 12>), gp, dim3(1024), 0, ST(s), k);
    else if (cap <= 16384) hipLaunchKernelGGL((k_ev_pick<1024, 16>), gp, dim3(1024), 0, ST(s), k);
    else hipLaunchKernelGGL(k_ev_pick_long, gp, dim3(EV_T), (size_t)k.lds_keys * 4, ST(s), k);
    const int rows = 4 * 256 / (p->head_dim / 8);
    int z = (keep + rows - 1) / rows;
    if (z > 1024) z = 1024;
    const dim3 g(p->n_kv_heads, b->n_seqs, z);
    switch (p->head_dim) {
        case 64: hipLaunchKernelGGL(k_ev_move<64>, g, dim3(256), 0, ST(s), a); break;
        case 128: hipLaunchKernelGGL(k_ev_move<128>, g, dim3(256), 0, ST(s), a); break;
        default: hipLaunchKernelGGL(k_ev_move<256>, g, dim3(256), 0, ST(s), a);
    }
    LAUNCHED("k_ev_pick/k_ev_move");
}

}  // extern "C"
