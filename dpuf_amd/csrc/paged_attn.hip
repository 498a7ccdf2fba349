// paged_attn.hip -- attention of new tokens over a paged KV cache.
//
// For a new row i of a sequence (query head j, kv head h = j / G, G query
// heads per kv head), over the cached rows t it sees:
//     s_t = scale q.k_t,  m = max s_t,  l = sum exp(s_t - m),
//     o = sum exp(s_t - m) v_t / l,  lse = m + ln l,
// in one pass over the keys with a running m and l (o and l are multiplied by
// exp(m_old - m_new) when m grows).  The G heads of a kv head share its keys,
// so a kernel's row is a "packed" row r = i G + g: every key read serves
// them all.
//
// Both kernels compute the transposed product S^T = K Q^T: a lane of the
// matrix instruction's result then holds one row and some keys, so maxima and
// sums are mostly within the lane, and its exponentials are, without any
// movement, the right-hand operand of O^T = V^T P^T.  The order of the keys
// within a matrix step is free as long as both operands agree, and V^T's
// operand takes the order in which S^T left them: 4 keys of each half or
// quarter of the wave, which is what one transposing LDS read gives.
//
// The running maximum need not be the largest score so far, only near it: m is
// moved (and l and o multiplied, a product per sum) when a score passes it by
// more than 2^SLACK, so that most tiles move nothing; p is at most 2^SLACK
// then.
//
// Exponentials are of base 2 with the scale folded in (one fma each), every sum
// is fp32.  The 16-bit matrix instructions take p rounded to the pages' type (a
// relative half step, 2^-8 in bf16 and 2^-11 in fp16, of each term).  In bf16
// few rows, which wait for memory, add what that takes off by a second product
// (48 rows over 310 to 6 000 keys 125.4 us without, 125.8 with; the outputs are
// off from 64 bits by 2.2e-3 and 1.7e-3, nearly all of the latter their own
// rounding).  Many rows do not: 512 over 16 384 keys would take 213 us instead
// of 169, for 1.7e-3 instead of 2.3e-3.
//
// fp16 has few exponents: below 2^-14 of the largest, terms would lose their
// bits, and below 2^-25 vanish, however many there are.  So there m is LIFT = 9
// below the maximum: p is at most 2^(9 + SLACK) = 2^15, and whole down to 2^-23
// of the largest.  The maximum is then rounded up to an integer, which keeps
// m + LIFT and the factors that l and o are moved by exact.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "hip_internal.h"
#include "paged.h"

namespace {

const float NEG_INF = -__builtin_huge_valf();
constexpr float SLACK = 6.0f;

enum { PA_BOTH = 0, PA_FEW, PA_MANY, PA_WIDE };

struct PaArgs {
    DpufAmdBatch b;
    DpufAmdPages p;
    int shift;          // log2 of page_size
    int nq, G;
    const uint16_t* q;
    float c2;           // scale * log2 e
    int few;            // packed rows up to which a sequence takes the few-row kernel
    int only;           // PA_BOTH, or the kernel that takes every sequence
    int nz_few, nz_many; // key ranges a sequence is split into at most
    int chunk_few, chunk_many;
    int out_f32;
    void* out;
    float* lse;
    // partial sums of rows whose keys are split: O unnormalised, (m, l);
    // [range][row][head], or, for few rows where others have many,
    // [range][sequence][kv head][packed row]
    float *few_o, *many_o;
    float2 *few_ml, *many_ml;
};

// Keys per range of a sequence of ctx keys: `chunk`, or more where nz ranges
// of it would not reach the end.
DEV int range_keys(int ctx, int chunk, int nz) {
    const int need = (ctx + nz - 1) / nz;
    return need <= chunk ? chunk : (need + 127) & ~127;
}

// Partial of a few-row sequence's packed row r (row: its place in the output).
DEV size_t few_at(const PaArgs& a, int z, int s, int kvh, int r, size_t row) {
    if (a.only == PA_FEW) return (size_t)z * a.b.n_rows * a.nq + row;
    return (((size_t)z * a.b.n_seqs + s) * a.p.n_kv_heads + kvh) * a.few + r;
}

// Writes one packed row's four consecutive columns at d, or its partial.
template <typename T>
DEV void put4(const PaArgs& a, size_t at, const float* o, float inv) {
    if (a.out_f32) {
        *(float4*)((float*)a.out + at) = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    } else {
        uint2 w;
        w.x = pack2<T>(o[0] * inv, o[1] * inv);
        w.y = pack2<T>(o[2] * inv, o[3] * inv);
        *(uint2*)((uint16_t*)a.out + at) = w;
    }
}

// What m is set to for a maximum, and the log sum of (m, l).
template <typename T> DEV float lowered(float top) { return T::LIFT == 0.0f ? top : ceilf(top) - T::LIFT; }
template <typename T> DEV float lse_of(float m2, float l) {
    constexpr float DOWN = T::LIFT == 0.0f ? 1.0f : 0x1p-9f;
    static_assert(T::LIFT == 0.0f || T::LIFT == 9.0f, "2^-LIFT");
    return l == 0.0f ? NEG_INF : (m2 + T::LIFT + __log2f(l * DOWN)) * 0.69314718055994531f;
}

// Infinities and NaN in V.  A row that does not see a key has p = 0 there, and
// 0 * inf would reach its sums all the same.  So in a tile that some row does
// not see whole they are taken out of V on its way to LDS, and, if there were
// any, added at the end to the rows that see them.
template <typename T> DEV uint32_t odd_mask(uint32_t e) {     // the halves of e that are infinite or NaN
    return ((e & T::EXP) == T::EXP ? 0xffffu : 0u) | (((e >> 16) & T::EXP) == T::EXP ? 0xffff0000u : 0u);
}
template <typename T> DEV uint32_t take_odd(u32x4& v) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t m = odd_mask<T>(v[i]);
        any |= m;
        v[i] &= ~m;
    }
    return any;
}
// The infinities and NaN of the four elements at v, 0 for the others.
template <typename T> DEV f32x4 odd4(const uint16_t* v) {
    const uint2 w = *(const uint2*)v;
    return __builtin_convertvector(
        __builtin_bit_cast(typename T::v4, make_uint2(w.x & odd_mask<T>(w.x), w.y & odd_mask<T>(w.y))), f32x4);
}

// Eight probabilities as an operand of the product with V, and, with T::REST,
// what that leaves of them as another.  The first is cut off rather than
// rounded, and the rest at least 2^-30 of p, so that neither is negative, nor 0
// where p is not: an infinity in V stays what it is.
template <typename T> DEV void split8(float* p, typename T::v8& hi, typename T::v8& rest) {
    u32x4 h, r;
    if constexpr (T::REST) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            h[i] = __builtin_amdgcn_perm(__float_as_uint(p[2 * i + 1]), __float_as_uint(p[2 * i]), 0x07060302);
#pragma unroll
            for (int e = 2 * i; e < 2 * i + 2; e++)
                p[e] = fmaxf(p[e] - __uint_as_float(__float_as_uint(p[e]) & 0xffff0000u), p[e] * 0x1p-30f);
            r[i] = pack2<T>(p[2 * i], p[2 * i + 1]);
        }
        rest = vec_of<typename T::v8>(r);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = pack2<T>(p[2 * i], p[2 * i + 1]);
    }
    hi = vec_of<typename T::v8>(h);
}

// ---------------------------------------------------------------------------
// Few rows (decode): bound by reading K and V once.  One workgroup per
// (kv head, sequence and tile of 16 packed rows, key range); its four waves
// take every fourth tile of 32 keys with sums of their own and meet in LDS at
// the end, so there is no barrier in the loop and each wave keeps a whole
// next tile (K and V, 16 KB at 128 columns) in flight in registers.  48 rows of
// 32 heads, 8 kv heads of 128 over 310 to 6 000 keys: 122 us, 5.1 TB/s; one row
// of 16 heads over 75 keys 7.7.
// ---------------------------------------------------------------------------
template <int HD> struct FewLds {
    static constexpr int PITCH = HD + 16;   // elements of a V row: 4 rows of a transposing read in 4 bank groups
    uint16_t v[4][32 * PITCH];
    float2 ml[4][16];
    int odd[4];
};

template <typename T, int HD> DEV void few_rows(const PaArgs& a, FewLds<HD>& sh, int kvh, int y, int z) {
    constexpr int NC = HD / 32;          // 32-column steps of a key
    constexpr int ND = HD / 16;          // 16-column tiles of the output
    constexpr int PITCH = FewLds<HD>::PITCH;
    typedef typename T::v8 v8;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g4 = lane >> 4;
    const int tiles = (a.few + 15) >> 4;
    const int s = y / tiles;
    const int* table = a.b.page_table + (size_t)s * a.b.table_stride;
    // the first range's first pages, beside the lengths
    int early[2];
#pragma unroll
    for (int u = 0; u < 2; u++) early[u] = table[min((32 * wave + 16 * u) >> a.shift, a.b.table_stride - 1)];
    const PgSeq sq = pg_seq(a.b, a.shift, s);
    const int rows = sq.n * a.G;
    if (rows > a.few && a.only == PA_BOTH) return;
    const int per = range_keys(sq.ctx, a.chunk_few, a.nz_few);
    const int ranges = sq.ctx > per ? (sq.ctx + per - 1) / per : 1;
    if (z >= ranges) return;

    // one tile of rows, unless a sequence has more than the others' few
    for (int tile = y - s * tiles; 16 * tile < rows; tile += tiles) {
        const int r = 16 * tile + col;
        const bool live = r < rows;
        const int qi = live ? r / a.G : 0, head = kvh * a.G + (live ? r - qi * a.G : 0);
        const size_t row = (size_t)(sq.r0 + qi) * a.nq + head;
        const int limit = live ? sq.ctx - sq.n + qi : -1;             // last key this row sees
        const int last = min(rows, 16 * tile + 16) - 1;
        const int first_limit = sq.ctx - sq.n + 16 * tile / a.G;      // of the tile's first row
        const int k0 = z * per, kend = min(min(sq.ctx - sq.n + last / a.G + 1, sq.ctx), k0 + per);

        v8 qf[NC];
#pragma unroll
        for (int c = 0; c < NC; c++)
            qf[c] = vec_of<v8>(live ? *(const u32x4*)(a.q + row * HD + 32 * c + 8 * g4) : u32x4{0, 0, 0, 0});

        f32x4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = NEG_INF, l = 0.0f;

        const uint16_t* kp = (const uint16_t*)a.p.k + (size_t)kvh * a.p.head_stride + 8 * g4;
        const uint16_t* vp = (const uint16_t*)a.p.v + (size_t)kvh * a.p.head_stride + 8 * g4;
        const int top = sq.ctx > 0 ? (sq.ctx - 1) >> a.shift : 0;
        uint16_t* lv = sh.v[wave];

        u32x4 kf[2][NC], vf[2][NC];
        int pg[2], pn[2];      // pages of the tile in kf / vf, and of the one after it
        // A 16-key half of a tile lies in one page (pages hold a multiple of 16
        // rows); halves past the last key repeat it, pages outside the pool read
        // page 0: both are masked below.
        auto pages = [&](int base, int* out) {
#pragma unroll
            for (int u = 0; u < 2; u++) out[u] = table[min((base + 16 * u) >> a.shift, top)];
        };
        auto load = [&](int base, const int* pid) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int key = base + 16 * u + col;
                const bool in = (unsigned)pid[u] < (unsigned)a.p.n_pages;
                const size_t off = (size_t)(in ? pid[u] : 0) * a.p.page_stride +
                                   (size_t)(key & (a.p.page_size - 1)) * a.p.row_stride;
#pragma unroll
                for (int c = 0; c < NC; c++) kf[u][c] = *(const u32x4*)(kp + off + 32 * c);
#pragma unroll
                for (int c = 0; c < NC; c++) vf[u][c] = *(const u32x4*)(vp + off + 32 * c);
            }
        };

        auto whole_at = [&](int base, const int* pid) {
            return base + 32 <= min(kend, first_limit + 1) && (unsigned)pid[0] < (unsigned)a.p.n_pages &&
                   (unsigned)pid[1] < (unsigned)a.p.n_pages;
        };
        uint32_t odd = 0;
        int base = k0 + 32 * wave;
        if (base < kend) {
            if (z == 0) {
                pg[0] = early[0];
                pg[1] = base + 16 < sq.ctx ? early[1] : early[0];
            } else {
                pages(base, pg);
            }
            load(base, pg);
            pages(base + 128, pn);
        }
        for (; base < kend; base += 128) {
            // V goes to LDS for the transposing reads; the wave's own LDS
            // operations are in order, so nothing but the compiler has to be held
            const bool whole = whole_at(base, pg);
            lds_order();
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int c = 0; c < NC; c++) *(u32x4*)(lv + (16 * u + col) * PITCH + 32 * c + 8 * g4) = vf[u][c];
            if (!whole)
#pragma unroll 1
                for (int e = 0; e < 2 * NC; e++) {
                    u32x4* at = (u32x4*)(lv + (e / NC * 16 + col) * PITCH + 32 * (e % NC) + 8 * g4);
                    u32x4 v = *at;
                    odd |= take_odd<T>(v);
                    *at = v;
                }
            f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int u = 0; u < 2; u++) sc[u] = T::mma16(vec_of<v8>(kf[u][c]), qf[c], sc[u]);
            const int here = base;
            const bool ok[2] = {(unsigned)pg[0] < (unsigned)a.p.n_pages, (unsigned)pg[1] < (unsigned)a.p.n_pages};
            if (base + 128 < kend) {
                pg[0] = pn[0];
                pg[1] = pn[1];
                load(base + 128, pg);
                pages(base + 256, pn);
            }
            // keys 16 u + 4 g4 + i of the tile
            if (!whole) {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (!ok[u] || here + 16 * u + 4 * g4 + i > limit) sc[u][i] = NEG_INF;
            }
            float mt = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                             fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
            mt = max_xor32(max_xor16(mt)) * a.c2;
            // m follows the maximum only when it is behind by more than 2^SLACK
            if (__any(mt > m + (T::LIFT + SLACK))) {
                const float mn = fmaxf(m, lowered<T>(mt)), f = __builtin_amdgcn_exp2f(m - (mn == NEG_INF ? 0.0f : mn));
                l *= f;
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= f;
                m = mn;
            }
            const float ms = m == NEG_INF ? 0.0f : m;
            float pr[8];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    pr[4 * u + i] = __builtin_amdgcn_exp2f(fmaf(sc[u][i], a.c2, -ms));
                    l += pr[4 * u + i];
                }
            v8 pf, rf;
            split8<T>(pr, pf, rf);
            lds_order();
            const uint16_t* tr = lv + (4 * g4 + (col >> 2)) * PITCH + 4 * (col & 3);
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const s16x4 lo = lds_tr4(tr + 16 * d), hi = lds_tr4(tr + 16 * PITCH + 16 * d);
                const uint2 a0 = __builtin_bit_cast(uint2, lo), a1 = __builtin_bit_cast(uint2, hi);
                const v8 vt = vec_of<v8>(u32x4{a0.x, a0.y, a1.x, a1.y});
                o[d] = T::mma16(vt, pf, o[d]);
                if (T::REST) o[d] = T::mma16(vt, rf, o[d]);
            }
        }

        // join the four waves: m, l of the 16 rows, then O by output column
        l = add_xor32(add_xor16(l));
        if (lane < 16) sh.ml[wave][lane] = make_float2(m, l);
        const bool my_odd = __any(odd != 0);
        if (lane == 0) sh.odd[wave] = my_odd;
        __syncthreads();
        const bool some_odd = sh.odd[0] | sh.odd[1] | sh.odd[2] | sh.odd[3];
        float M = NEG_INF, L = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) M = fmaxf(M, sh.ml[w][col].x);
        const float Ms = M == NEG_INF ? 0.0f : M;
#pragma unroll
        for (int w = 0; w < 4; w++) L += sh.ml[w][col].y * __builtin_amdgcn_exp2f(sh.ml[w][col].x - Ms);
        const float f = __builtin_amdgcn_exp2f(m - Ms);
        // [wave][16 rows][HD + 4] floats over the V tiles, a half of the columns
        // at a time (16 * (HD / 2 + 4) floats fit a wave's 32 * (HD + 16) halves)
        constexpr int OP = HD / 2 + 4;
        float* lo = (float*)sh.v[0];
        constexpr int WS = 32 * PITCH / 2;   // floats of a wave's region
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
#pragma unroll
            for (int d = 0; d < ND / 2; d++) {
                const f32x4 v = o[hf * (ND / 2) + d] * f;
                *(f32x4*)(lo + wave * WS + col * OP + 16 * d + 4 * g4) = v;
            }
            __syncthreads();
            for (int e = threadIdx.x; e < 16 * (HD / 8); e += 256) {
                const int rr = e / (HD / 8), d4 = 4 * (e - rr * (HD / 8));
                const int pr = 16 * tile + rr;
                if (pr < rows) {
                    f32x4 v = *(const f32x4*)(lo + rr * OP + d4);
#pragma unroll
                    for (int w = 1; w < 4; w++) v += *(const f32x4*)(lo + w * WS + rr * OP + d4);
                    const int i = pr / a.G;
                    if (some_odd)
                        for (int t0 = k0; t0 < kend; t0 += 32) {
                            int pid[2];
                            pages(t0, pid);
                            if (whole_at(t0, pid)) continue;
                            for (int t = t0; t < t0 + 32 && t <= sq.ctx - sq.n + i; t++) {
                                const int p = pid[(t >> 4) & 1];
                                if ((unsigned)p < (unsigned)a.p.n_pages)
                                    v += odd4<T>((const uint16_t*)a.p.v + (size_t)kvh * a.p.head_stride +
                                                 (size_t)p * a.p.page_stride +
                                                 (size_t)(t & (a.p.page_size - 1)) * a.p.row_stride +
                                                 hf * (HD / 2) + d4);
                            }
                        }
                    const size_t orow = (size_t)(sq.r0 + i) * a.nq + kvh * a.G + (pr - i * a.G);
                    const int d = hf * (HD / 2) + d4;
                    if (ranges > 1) {
                        *(f32x4*)(a.few_o + few_at(a, z, s, kvh, pr, orow) * HD + d) = v;
                    } else {
                        float Lr = 0.0f, Mr = NEG_INF;
#pragma unroll
                        for (int w = 0; w < 4; w++) Mr = fmaxf(Mr, sh.ml[w][rr].x);
                        const float Mz = Mr == NEG_INF ? 0.0f : Mr;
#pragma unroll
                        for (int w = 0; w < 4; w++) Lr += sh.ml[w][rr].y * __builtin_amdgcn_exp2f(sh.ml[w][rr].x - Mz);
                        const float ov[4] = {v[0], v[1], v[2], v[3]};
                        put4<T>(a, orow * HD + d, ov, Lr > 0.0f ? 1.0f / Lr : Lr == 0.0f ? 0.0f : Lr);
                    }
                }
            }
            __syncthreads();
        }
        if (threadIdx.x < 16 && live) {
            if (ranges > 1) a.few_ml[few_at(a, z, s, kvh, r, row)] = make_float2(M, L);
            else if (a.lse) a.lse[row] = lse_of<T>(M, L);
        }
    }
}

// ---------------------------------------------------------------------------
// Many rows (chunks of a prompt): bound by the matrix instructions and the
// exponentials.  One workgroup per (kv head, 32 WAVES packed rows, key range);
// its waves take 32 rows each and share tiles of KT keys of K and V in LDS, two
// of them: while one is computed, the other takes the tile after it from
// registers, whose loads were issued a tile earlier.  Two workgroups of four
// waves a CU, whose vector and matrix work overlap, or one of eight, which
// loads and stores half the tiles for the same rows.  512 rows of 32 heads, 8
// kv heads of 128 over 16 384 keys: 150 to 170 us, 800 to 900 TFLOP/s; the
// reads of K and V from LDS (32 rows a wave use each) take as long as the
// matrix instructions.
// ---------------------------------------------------------------------------
template <int HD> struct ManyLds {
    static constexpr int KT = HD == 256 ? 32 : 64;
    static constexpr int KP = HD + 8;    // K row: 16 rows' 16 bytes in distinct banks
    static constexpr int VP = HD + 32;   // V row: 4 rows' 64 bytes in distinct banks
    uint16_t k[2][KT * KP];
    uint16_t v[2][KT * VP];
    int odd;
};

template <typename T, int HD, int WAVES>
DEV void many_rows(const PaArgs& a, ManyLds<HD>& sh, int kvh, int tile, int z) {
    constexpr int KT = ManyLds<HD>::KT, KP = ManyLds<HD>::KP, VP = ManyLds<HD>::VP;
    constexpr int NC = HD / 16;          // 16-column steps of a key
    constexpr int ND = HD / 32;          // 32-column tiles of the output
    constexpr int CH = HD / 8;           // 16-byte pieces of a row
    constexpr int TR = 32 * WAVES;       // packed rows of a workgroup
    constexpr int RP = 64 * WAVES / CH;  // rows a pass of the workgroup loads
    constexpr int NP = KT / RP;
    constexpr int NB = KT / 32;          // 32-key blocks of a tile
    typedef typename T::v8 v8;
    uint16_t (*lk)[KT * KP] = sh.k;
    uint16_t (*lv)[KT * VP] = sh.v;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, h = lane >> 5;
    // sequence of the tile, and its tile there, among the sequences with many rows
    int s = -1;
    for (int s0 = 0; s0 < a.b.n_seqs && s < 0; s0 += 64) {
        int n = 0;
        if (s0 + lane < a.b.n_seqs) {
            const PgSeq t = pg_seq(a.b, a.shift, s0 + lane);
            const int rows = t.n * a.G;
            n = rows > a.few || a.only != PA_BOTH ? (rows + TR - 1) / TR : 0;
        }
        int sum = n;
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        const uint64_t past = __ballot(sum > tile);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            tile -= __shfl(sum - n, at);
            s = s0 + at;
        } else {
            tile -= __shfl(sum, 63);
        }
    }
    s = __builtin_amdgcn_readfirstlane(s);
    tile = __builtin_amdgcn_readfirstlane(tile);
    if (s < 0) return;
    const PgSeq sq = pg_seq(a.b, a.shift, s);
    const int rows = sq.n * a.G;
    const int per = range_keys(sq.ctx, a.chunk_many, a.nz_many);
    const int ranges = sq.ctx > per ? (sq.ctx + per - 1) / per : 1;
    if (z >= ranges) return;

    const int r = TR * tile + 32 * wave + col;
    const bool live = r < rows;
    const int qi = live ? r / a.G : 0, head = kvh * a.G + (live ? r - qi * a.G : 0);
    const size_t row = (size_t)(sq.r0 + qi) * a.nq + head;
    const int limit = live ? sq.ctx - sq.n + qi : -1;
    // keys past a wave's last row's limit are skipped by the wave, past the
    // workgroup's by all
    const int wl = min(rows, TR * tile + 32 * wave + 32) - 1, gl = min(rows, TR * tile + TR) - 1;
    const int first_limit = sq.ctx - sq.n + (TR * tile + 32 * wave) / a.G;
    const int k0 = z * per;
    const int wend = TR * tile + 32 * wave < rows ? min(sq.ctx - sq.n + wl / a.G + 1, k0 + per) : 0;
    const int kend = min(min(sq.ctx - sq.n + gl / a.G + 1, sq.ctx), k0 + per);

    v8 qf[NC];
#pragma unroll
    for (int c = 0; c < NC; c++)
        qf[c] = vec_of<v8>(live ? *(const u32x4*)(a.q + row * HD + 16 * c + 8 * h) : u32x4{0, 0, 0, 0});
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    float m = NEG_INF, l = 0.0f;

    // A tile's pages, one for each 16 keys (pages hold a multiple of 16 rows),
    // are the same for all lanes: a thread's address is its own offset within
    // 16 rows plus a scalar base.
    constexpr int NG = KT / 16;
    const int lr = threadIdx.x / CH, lc = 8 * (threadIdx.x % CH);   // row and column of this thread's pieces
    const int wr = __builtin_amdgcn_readfirstlane(lr) >> 4;          // the wave's 16 of a pass of 32 or 64
    const uint32_t lo = (uint32_t)((lr & 15) * (int)a.p.row_stride + lc);
    const uint16_t* kp = (const uint16_t*)a.p.k + (size_t)kvh * a.p.head_stride;
    const uint16_t* vp = (const uint16_t*)a.p.v + (size_t)kvh * a.p.head_stride;
    const int* table = a.b.page_table + (size_t)s * a.b.table_stride;
    const int top = sq.ctx > 0 ? (sq.ctx - 1) >> a.shift : 0;
    u32x4 kf[NP], vf[NP];
    int pn[NG];              // pages of the tile to be loaded next
    uint32_t odd = 0;
    const int seen = min(kend, sq.ctx - sq.n + TR * tile / a.G + 1);     // keys before it: by all rows
    uint32_t bad1 = 0, bad2 = 0;   // of the tile in kf / vf (one bit per 16 keys: outside the pool), and of the next
    auto pages = [&](int base) {
#pragma unroll
        for (int g = 0; g < NG; g++) pn[g] = table[min((base + 16 * g) >> a.shift, top)];
    };
    auto load = [&](int base) {
        bad2 = 0;
#pragma unroll
        for (int g = 0; g < NG; g++) bad2 |= ((unsigned)pn[g] >= (unsigned)a.p.n_pages) << g;
#pragma unroll
        for (int u = 0; u < NP; u++) {
            const int g = u * RP / 16 + (RP > 16 ? wr : 0);
            int pg = pn[u * RP / 16 % NG];
#pragma unroll
            for (int e = 1; e < RP / 16; e++) pg = wr == e ? pn[(u * RP / 16 + e) % NG] : pg;
            if ((bad2 >> g) & 1) pg = 0;
            const size_t at = (size_t)pg * a.p.page_stride +
                              (size_t)((base + 16 * g) & (a.p.page_size - 1)) * a.p.row_stride +
                              (RP == 8 ? (size_t)(u & 1) * 8 * a.p.row_stride : 0);
            kf[u] = *(const u32x4*)(kp + at + lo);
            vf[u] = *(const u32x4*)(vp + at + lo);
        }
        if (bad2 || base + KT > seen)
#pragma unroll
            for (int u = 0; u < NP; u++) odd |= take_odd<T>(vf[u]);
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int u = 0; u < NP; u++) {
            *(u32x4*)(lk[buf] + (u * RP + lr) * KP + lc) = kf[u];
            *(u32x4*)(lv[buf] + (u * RP + lr) * VP + lc) = vf[u];
        }
    };

    if (threadIdx.x == 0) sh.odd = 0;
    if (k0 < kend) {
        pages(k0);
        load(k0);
        pages(k0 + KT);
        store(0);
        bad1 = bad2;
        if (k0 + KT < kend) {
            load(k0 + KT);
            pages(k0 + 2 * KT);
        }
    }
    int buf = 0;
    for (int base = k0; base < kend; base += KT, buf ^= 1) {
        __syncthreads();
        if (base + KT < kend) store(buf ^ 1);
        const uint32_t bad = bad1;
        bad1 = bad2;
        if (base + 2 * KT < kend) {
            load(base + 2 * KT);
            pages(base + 3 * KT);
        }
        if (base >= wend) continue;
        const f32x16 zero = {};
        f32x16 sc[NB];
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const v8 kv = vec_of<v8>(*(const u32x4*)(lk[buf] + (32 * b + col) * KP + 16 * c + 8 * h));
                sc[b] = T::mma32(kv, qf[c], c ? sc[b] : zero);
            }
        // sc[b][i]: key 32 b + 8 (i / 4) + 4 h + i % 4
        if (base + KT > min(wend, first_limit + 1) || bad) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int key = 32 * b + 8 * (i >> 2) + 4 * h + (i & 3);
                    if (base + key > limit || ((bad >> (key >> 4)) & 1)) sc[b][i] = NEG_INF;
                }
        }
        float mt = NEG_INF;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) mt = fmaxf(mt, sc[b][i]);
        mt = max_xor32(mt) * a.c2;
        // m follows the maximum only when it is behind by more than 2^SLACK
        if (__any(mt > m + (T::LIFT + SLACK))) {
            const float mn = fmaxf(m, lowered<T>(mt)), f = __builtin_amdgcn_exp2f(m - (mn == NEG_INF ? 0.0f : mn));
            l *= f;
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= f;
            m = mn;
        }
        const float ms = m == NEG_INF ? 0.0f : m;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float pr[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    pr[i] = __builtin_amdgcn_exp2f(fmaf(sc[b][8 * k + i], a.c2, -ms));
                    l += pr[i];
                }
                const u32x4 pw = {pack2<T>(pr[0], pr[1]), pack2<T>(pr[2], pr[3]), pack2<T>(pr[4], pr[5]),
                                  pack2<T>(pr[6], pr[7])};
                const v8 pf = vec_of<v8>(pw);
                // keys 4 h .. + 3 and 8 + 4 h .. + 3 of the 16, columns 16 * (lane / 16 % 2) + lane % 16
                const uint16_t* tr = lv[buf] + (32 * b + 16 * k + 4 * h + ((lane & 15) >> 2)) * VP +
                                     16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    const uint2 a0 = __builtin_bit_cast(uint2, lds_tr4(tr + 32 * d));
                    const uint2 a1 = __builtin_bit_cast(uint2, lds_tr4(tr + 8 * VP + 32 * d));
                    o[d] = T::mma32(vec_of<v8>(u32x4{a0.x, a0.y, a1.x, a1.y}), pf, o[d]);
                }
            }
    }
    __syncthreads();
    if (__any(odd != 0) && lane == 0) sh.odd = 1;
    __syncthreads();
    if (sh.odd)
        for (int base = k0; base < kend; base += 16) {
            const int pg = table[min(base >> a.shift, top)], t0 = base & ~(KT - 1);
            if ((unsigned)pg >= (unsigned)a.p.n_pages) continue;
            bool whole = t0 + KT <= seen;
            for (int g = 0; g < NG; g++)
                whole = whole && (unsigned)table[min((t0 + 16 * g) >> a.shift, top)] < (unsigned)a.p.n_pages;
            if (whole) continue;
#pragma unroll 1
            for (int key = base; key < base + 16; key++) {
                const uint16_t* v = vp + (size_t)pg * a.p.page_stride +
                                    (size_t)(key & (a.p.page_size - 1)) * a.p.row_stride + 4 * h;
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const f32x4 x = odd4<T>(v + 32 * d + 2 * i);
#pragma unroll
                        for (int e = 0; e < 4; e++) o[d][i + e] += key <= limit ? x[e] : 0.0f;
                    }
            }
        }
    l = add_xor32(l);
    if (!live) return;
    // o[d][i]: column 32 d + 8 (i / 4) + 4 h + i % 4
    if (ranges > 1) {
        float* po = a.many_o + ((size_t)z * a.b.n_rows * a.nq + row) * HD;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(f32x4*)(po + 32 * d + 2 * i + 4 * h) = f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
        if (h == 0) a.many_ml[(size_t)z * a.b.n_rows * a.nq + row] = make_float2(m, l);
    } else {
        const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float ov[4] = {o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
                put4<T>(a, row * HD + 32 * d + 2 * i + 4 * h, ov, inv);
            }
        if (h == 0 && a.lse) a.lse[row] = lse_of<T>(m, l);
    }
}

// Blocks of the three kernels: kv heads fastest, so that the workgroups that
// read the same keys run on the same XCDs (8 kv heads: one XCD each) and share
// their L2.
template <typename T, int HD> __global__ __launch_bounds__(256, HD == 256 ? 1 : 3) void k_pa_few(PaArgs a) {
    __shared__ __align__(16) FewLds<HD> sh;
    few_rows<T, HD>(a, sh, blockIdx.x, blockIdx.y, blockIdx.z);
}
template <typename T, int HD> __global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void k_pa_many(PaArgs a) {
    __shared__ __align__(16) ManyLds<HD> sh;
    many_rows<T, HD, 4>(a, sh, blockIdx.x, blockIdx.y, blockIdx.z);
}
template <typename T, int HD> __global__ __launch_bounds__(512, 2) void k_pa_wide(PaArgs a) {
    __shared__ __align__(16) ManyLds<HD> sh;
    many_rows<T, HD, 8>(a, sh, blockIdx.x, blockIdx.y, blockIdx.z);
}
// Chunks and decoding sequences in one call: the chunks' workgroups, which are
// bound by arithmetic, first, and beside them those that are bound by memory.
template <typename T, int HD>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void k_pa_mixed(PaArgs a, int y_many, int y_few) {
    __shared__ __align__(16) char raw[sizeof(ManyLds<HD>) > sizeof(FewLds<HD>) ? sizeof(ManyLds<HD>)
                                                                               : sizeof(FewLds<HD>)];
    const int nkv = a.p.n_kv_heads, many = nkv * y_many * a.nz_many;
    int b = blockIdx.x;
    if (b < many) {
        const int kvh = b % nkv;
        b /= nkv;
        many_rows<T, HD, 4>(a, *(ManyLds<HD>*)raw, kvh, b % y_many, b / y_many);
    } else {
        b -= many;
        const int kvh = b % nkv;
        b /= nkv;
        few_rows<T, HD>(a, *(FewLds<HD>*)raw, kvh, b % y_few, b / y_few);
    }
}

// Joins the key ranges of rows that were split: HD / 4 lanes a (row, head) and
// ZG groups of them, each with every ZG-th range, four of a group's in flight,
// their sums joined in LDS: 512 rows of 32 heads in four ranges 7.6 us, 4.7 TB/s.
template <typename T, int HD, int ZG>
__global__ __launch_bounds__(256) void k_pa_join(PaArgs a) {
    constexpr int LPR = HD / 4, PER = 256 / LPR / ZG;
    __shared__ float2 sml[ZG][PER];
    __shared__ f32x4 so[ZG > 1 ? ZG : 1][PER * LPR];
    const int lane = threadIdx.x & 63, row = blockIdx.x, unit = threadIdx.x / LPR, zg = unit / PER;
    const int head = blockIdx.y * PER + unit % PER, d = 4 * (threadIdx.x % LPR);
    const int s = pg_seq_of_row(a.b, row, lane);
    if (s < 0) return;
    const PgSeq sq = pg_seq(a.b, a.shift, s);
    const bool few = a.only == PA_FEW || (a.only == PA_BOTH && sq.n * a.G <= a.few);
    const int per = range_keys(sq.ctx, few ? a.chunk_few : a.chunk_many, few ? a.nz_few : a.nz_many);
    const int ranges = sq.ctx > per ? (sq.ctx + per - 1) / per : 1;
    if (ranges == 1 || row >= sq.r0 + sq.n) return;
    const bool live = head < a.nq;
    const int hd = live ? head : a.nq - 1, kvh = hd / a.G;
    const size_t at = (size_t)row * a.nq + hd, total = (size_t)a.b.n_rows * a.nq;
    const size_t first = few ? few_at(a, 0, s, kvh, (row - sq.r0) * a.G + hd - kvh * a.G, at) : at;
    const size_t step = few && a.only == PA_BOTH ? (size_t)a.b.n_seqs * a.p.n_kv_heads * a.few : total;
    const float2* mls = (few ? a.few_ml : a.many_ml) + first;
    const float* os = (few ? a.few_o : a.many_o) + first * HD + d;
    float M = NEG_INF, L = 0.0f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](float m, float l, f32x4 p) {
        const float mn = fmaxf(M, m), ms = mn == NEG_INF ? 0.0f : mn;
        const float f0 = __builtin_amdgcn_exp2f(M - ms), f1 = __builtin_amdgcn_exp2f(m - ms);
        L = L * f0 + l * f1;
        o = o * f0 + p * f1;
        M = mn;
    };
    for (int z0 = zg; z0 < ranges; z0 += 4 * ZG) {
        float2 ml[4];
        f32x4 po[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const size_t z = min(z0 + e * ZG, ranges - 1) * step;
            ml[e] = mls[z];
            po[e] = *(const f32x4*)(os + z * HD);
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (z0 + e * ZG < ranges) add(ml[e].x, ml[e].y, po[e]);
    }
    if constexpr (ZG > 1) {
        const int own = threadIdx.x % (PER * LPR);
        if (d == 0) sml[zg][unit % PER] = make_float2(M, L);
        so[zg][own] = o;
        __syncthreads();
        if (zg > 0) return;
#pragma unroll
        for (int z = 1; z < ZG; z++) add(sml[z][unit % PER].x, sml[z][unit % PER].y, so[z][own]);
    }
    if (!live) return;
    const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
    const float ov[4] = {o[0], o[1], o[2], o[3]};
    put4<T>(a, at * HD + d, ov, inv);
    if (d == 0 && a.lse) a.lse[at] = lse_of<T>(M, L);
}

struct PaPlan {
    int only, few, nz_few, nz_many, chunk_few, chunk_many, y_few, y_many;
    size_t few_rows, many_rows;   // partial sums in the workspace
};

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Keys per range: about `times` sqrt(ctx), in whole 128.
int range_of(int64_t ctx, double times) { return ((int)(times * sqrt((double)ctx)) + 127) & ~127; }

// Which kernel takes which sequences.  Row counts are on the device; what the
// host knows is their sum and the number of sequences.  No more rows than
// sequences: a decode step (a sequence that has several rows all the same has
// its tiles done in turn), the few-row kernel alone.  One sequence with more
// than a tile of rows: the many-row kernel alone, in workgroups of 256 rows
// where there are at least 384 and 2 048 keys (512 rows of 4 heads over 16 384
// keys 150 us against 169, 100 rows over 4 096 29 against 32; over 600 keys
// 19.9 against 17.2).  Otherwise each sequence by its own count: up to `few`
// packed rows (a tile of 16; two where a single row has more than 16 query
// heads per kv head) or more.
//
// Key ranges of decoding sequences: of 128 keys or more, such that every CU has
// one, but not so long that a batch's shorter sequences leave them idle.  One
// row of 32 heads, 8 kv heads of 128: over 1 500 keys 22.3 us in ranges of
// 1 024, 15.9 in 512, 12.6 in 256, 10.7 in 128; over 4 096 22.6, 15.7, 12.6,
// 10.6; over 16 384 23.9, 19.8, 20.9, 20.8.  16 rows over 500 to 8 000 keys
// 56.2, 53.7, 53.4, 61.6; 48 rows 160.5, 164, 164, 172.
//
// Short contexts are one range, since the join is a launch more: one row over
// 200 keys 8.7 us in one, 9.4 in two, over 150 8.2 and 8.8.  From 257 keys on
// they are split where all ranges of 128 fit on the card at once, four of
// them from up to 64 (sequence, kv head): one row over 300 keys 10.2 in one,
// 9.3 in three, over 512 11.7 and 9.2; 8 rows 10.4 and 9.6, 12.5 and 10.8; but
// 12 rows 11.0 and 12.5, 12.7 and 12.9, 16 rows 11.6 and 12.1, 12.8 and 14.0.
PaPlan plan(const DpufAmdBatch& b, const DpufAmdPages& p, int nq) {
    const int G = nq / p.n_kv_heads;
    PaPlan r;
    r.few = G > 16 ? 32 : 16;
    const int64_t cap = (int64_t)b.table_stride * p.page_size;
    const int64_t ctx = b.max_ctx < 1 ? 1 : b.max_ctx < cap ? b.max_ctx : cap;
    const int64_t packed = (int64_t)b.n_rows * G;
    r.only = b.n_rows <= b.n_seqs || packed <= r.few ? PA_FEW : b.n_seqs > 1 ? PA_BOTH
             : packed >= 384 && ctx >= 2048 && p.head_dim <= 128 ? PA_WIDE : PA_MANY;
    const int tr = r.only == PA_WIDE ? 256 : 128;
    const int64_t most = packed / (r.few + 1);
    r.y_few = r.only >= PA_MANY ? 0 : b.n_seqs * ((r.few + 15) / 16);
    r.y_many = r.only == PA_FEW ? 0 : r.only == PA_BOTH ? (int)(packed / 128 + (most < b.n_seqs ? most : b.n_seqs))
                                                        : ceil_div(packed, tr);
    const int64_t units = (int64_t)b.n_seqs * p.n_kv_heads;
    const int64_t even = (ctx * units / 256 + 127) & ~127, long_few = units >= 256 ? 1024 : 512;
    const bool whole = ctx <= (units <= 64 ? 256 : 512);
    r.chunk_few = whole || even > long_few ? (int)long_few : even < 128 ? 128 : (int)even;
    r.nz_few = ceil_div(ctx, r.chunk_few);
    if (r.nz_few > 64) r.nz_few = 64;
    // (kv heads x sequences) that fill the card by themselves need no ranges,
    // and the partial sums stay below 16 384 x `few` rows
    const int64_t cap_z = 16384 / units;
    if (r.nz_few > cap_z) r.nz_few = cap_z < 1 ? 1 : (int)cap_z;
    // as many ranges of a chunk's keys as fit on the card beside its tiles at
    // once: two workgroups of 128 rows a CU, or one of 256.  Beside decoding
    // sequences fewer, so that those, which wait for memory, run at the same
    // time (a chunk of 256 rows and 31 single rows over 500 to 6 000 keys: 122
    // us with room for 400, 134 for 512, 140 for 768), unless the chunks are
    // nearly all of the work: then more, since the shorter contexts end sooner
    // (three of 128 rows and a single one over 4 096 to 16 384: 201, 157, 119).
    // Two values for what varies with tiles, single rows and contexts: of 54
    // batches of 1 to 4 chunks of 64 to 256 rows beside 1, 7 or 31 single rows,
    // 39 are within 10 % of the best of 256 to 1 024, 7 % in the middle; the
    // farthest is four of 64 and a single one over 4 096 to 16 384, 131 with
    // 400 and 85 with 768
    const bool chunks = (int64_t)(b.n_rows - b.n_seqs) * G > 220 * (int64_t)b.n_seqs;
    const int64_t room = r.only == PA_WIDE ? 256 : r.only == PA_MANY ? 512 : chunks ? 768 : 400;
    const int64_t wgs = (packed + tr - 1) / tr * p.n_kv_heads;
    const int64_t nz = wgs >= room ? 1 : room / (wgs > 0 ? wgs : 1);
    r.chunk_many = (ceil_div(ctx, nz) + 127) & ~127;
    if (r.chunk_many < range_of(ctx, 4.0)) r.chunk_many = range_of(ctx, 4.0);
    r.nz_many = ceil_div(ctx, r.chunk_many);
    const size_t all = (size_t)b.n_rows * nq, some = (size_t)b.n_seqs * p.n_kv_heads * r.few;
    r.few_rows = r.only <= PA_FEW && r.nz_few > 1 ? r.nz_few * (r.only == PA_FEW ? all : some) : 0;
    r.many_rows = r.only != PA_FEW && r.nz_many > 1 ? r.nz_many * all : 0;
    return r;
}

template <typename T, int HD>
void launch(const PaArgs& a, const PaPlan& pl, hipStream_t st) {
    const int nkv = a.p.n_kv_heads;
    if (pl.only == PA_FEW)
        hipLaunchKernelGGL((k_pa_few<T, HD>), dim3(nkv, pl.y_few, pl.nz_few), dim3(256), 0, st, a);
    else if (pl.only == PA_MANY)
        hipLaunchKernelGGL((k_pa_many<T, HD>), dim3(nkv, pl.y_many, pl.nz_many), dim3(256), 0, st, a);
    else if (pl.only == PA_WIDE) {
        if constexpr (HD <= 128)
            hipLaunchKernelGGL((k_pa_wide<T, HD>), dim3(nkv, pl.y_many, pl.nz_many), dim3(512), 0, st, a);
    } else
        hipLaunchKernelGGL((k_pa_mixed<T, HD>), dim3(nkv * (pl.y_many * pl.nz_many + pl.y_few * pl.nz_few)), dim3(256),
                           0, st, a, pl.y_many, pl.y_few);
    if (pl.few_rows + pl.many_rows > 0) {
        constexpr int ZG = HD == 256 ? 4 : 8;
        const int nz = pl.nz_few > pl.nz_many ? pl.nz_few : pl.nz_many;
        // few rows of many ranges wait for their loads (one row over 65 536
        // keys in 64 ranges 52 us, 58 by one group), many are bound by bytes
        // (a mixed batch of 269 rows of 32 heads, 7 ranges: 60.8 and 53)
        if (nz > 4 && (int64_t)a.b.n_rows * a.nq <= 4096)
            hipLaunchKernelGGL((k_pa_join<T, HD, ZG>), dim3(a.b.n_rows, ceil_div(a.nq, 256 / (HD / 4) / ZG)), dim3(256),
                               0, st, a);
        else
            hipLaunchKernelGGL((k_pa_join<T, HD, 1>), dim3(a.b.n_rows, ceil_div(a.nq, 256 / (HD / 4))), dim3(256), 0, st,
                               a);
    }
    LAUNCHED("k_pa");
}

}  // namespace

extern "C" {

size_t dpuf_hip_paged_attn_workspace(const DpufAmdBatch* b, const DpufAmdPages* p, int32_t nq) {
    const PaPlan pl = plan(*b, *p, nq);
    return (pl.few_rows + pl.many_rows) * ((size_t)p->head_dim * 4 + 8);
}

void dpuf_hip_paged_attn(void* s, const DpufAmdBatch* b, const DpufAmdPages* p, int32_t nq, const void* q, float scale,
                         int32_t out_f32, void* out, float* lse, void* ws) {
    const PaPlan pl = plan(*b, *p, nq);
    PaArgs a;
    a.b = *b;
    a.p = *p;
    a.shift = __builtin_ctz(p->page_size);
    a.nq = nq;
    a.G = nq / p->n_kv_heads;
    a.q = (const uint16_t*)q;
    a.c2 = scale * 1.4426950408889634f;
    a.few = pl.few;
    a.only = pl.only;
    a.nz_few = pl.nz_few;
    a.nz_many = pl.nz_many;
    a.chunk_few = pl.chunk_few;
    a.chunk_many = pl.chunk_many;
    a.out_f32 = out_f32;
    a.out = out;
    a.lse = lse;
    a.few_o = (float*)ws;
    a.many_o = a.few_o + pl.few_rows * p->head_dim;
    a.few_ml = (float2*)(a.many_o + pl.many_rows * p->head_dim);
    a.many_ml = a.few_ml + pl.few_rows;
    const bool bf = p->type == DPUF_AMD_BF16;
    switch (p->head_dim) {
        case 64: bf ? launch<Bf16, 64>(a, pl, ST(s)) : launch<Fp16, 64>(a, pl, ST(s)); break;
        case 128: bf ? launch<Bf16, 128>(a, pl, ST(s)) : launch<Fp16, 128>(a, pl, ST(s)); break;
        default: bf ? launch<Bf16, 256>(a, pl, ST(s)) : launch<Fp16, 256>(a, pl, ST(s)); break;
    }
}

}  // extern "C"
