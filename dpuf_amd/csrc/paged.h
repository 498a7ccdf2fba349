// paged.h -- device helpers shared by the paged-cache kernels (paged_attn.hip,
// paged_cache.hip): element types, matrix instructions, and where a
// sequence's rows lie.
#ifndef DPUF_PAGED_H
#define DPUF_PAGED_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dev_common.h"
#include "../../include/dpuf_amd.h"

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef s16x4 __attribute__((address_space(3))) * lds_s16x4;

// The two 16-bit element types: vectors of 8 (one matrix operand) and the
// matrix instructions with fp32 sums.
struct Bf16 {
    static constexpr uint32_t EXP = 0x7f80;     // exponent bits
    static constexpr float LIFT = 0.0f;
    static constexpr bool REST = true;          // probabilities of few rows as two terms: 8 bits are few
    typedef __bf16 e;
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    static DEV f32x4 mma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static DEV f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
struct Fp16 {
    static constexpr uint32_t EXP = 0x7c00;
    // Probabilities are 2^LIFT times as large: fp16's normal numbers end at 2^-14
    static constexpr float LIFT = 9.0f;
    static constexpr bool REST = false;
    typedef _Float16 e;
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    static DEV f32x4 mma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static DEV f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// Two floats rounded (to nearest even) into one 32-bit word of T.
template <typename T> DEV uint32_t pack2(float a, float b) {
    const f32x2 x = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, typename T::v2));
}

template <typename V> DEV V vec_of(u32x4 x) { return __builtin_bit_cast(V, x); }

// 4 x 16-bit of each of 16 lanes, transposed: lane i of a 16-lane row passes
// the address of row i / 4, columns 4 * (i % 4) .. + 3 of a 4 x 16 block and
// gets column i of its 4 rows.
DEV s16x4 lds_tr4(const uint16_t* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p); }

// Between a wave's own LDS writes and its other lanes' reads of them: the
// hardware keeps a wave's LDS operations in order, this keeps the compiler's.
DEV void lds_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// A value of two lanes 32 or 16 apart, in both of them.  The swap exchanges
// half of one register with half of another; both hold v here, and the copy is
// hidden from the compiler, which would otherwise put both in one register.
DEV uint32_t hidden_copy(uint32_t u) {
    asm("" : "+v"(u));
    return u;
}
DEV float2 both_of_32(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, hidden_copy(u), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
DEV float2 both_of_16(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, hidden_copy(u), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
DEV float max_xor32(float v) { const float2 b = both_of_32(v); return fmaxf(b.x, b.y); }
DEV float max_xor16(float v) { const float2 b = both_of_16(v); return fmaxf(b.x, b.y); }
DEV float add_xor32(float v) { const float2 b = both_of_32(v); return b.x + b.y; }
DEV float add_xor16(float v) { const float2 b = both_of_16(v); return b.x + b.y; }

// A sequence's new rows [r0, r0 + n) of the call and its ctx cached rows,
// clamped to the call's rows and to its page table, so that no index derived
// from them leaves either.
struct PgSeq {
    int r0, n, ctx;
};
DEV int pg_ctx(const DpufAmdBatch& b, int shift, int s) {
    return min(max(b.ctx_len[s], 0), b.table_stride << shift);
}
DEV PgSeq pg_seq(const DpufAmdBatch& b, int shift, int s) {
    PgSeq q;
    q.r0 = min(max(b.row_start[s], 0), b.n_rows);
    q.n = min(max(b.row_start[s + 1], q.r0), b.n_rows) - q.r0;
    q.ctx = pg_ctx(b, shift, s);
    return q;
}

// Sequence of a call's row, or -1 behind the last one's (every lane of a wave
// gets it): the number of row starts up to the row, 64 at a time.
DEV int pg_seq_of_row(const DpufAmdBatch& b, int row, int lane) {
    int below = 0;
    for (int s0 = 0; s0 <= b.n_seqs; s0 += 64) {
        const int s = s0 + lane;
        below += __popcll(__ballot(s <= b.n_seqs && b.row_start[s <= b.n_seqs ? s : 0] <= row));
    }
    return below >= 1 && below <= b.n_seqs ? below - 1 : -1;
}

// Page of cached row i of sequence s (i below the sequence's clamped ctx).
DEV int pg_page(const DpufAmdBatch& b, int shift, int s, int i) {
    return b.page_table[(size_t)s * b.table_stride + (i >> shift)];
}

#endif
