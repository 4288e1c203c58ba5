// Device pieces shared by the sequence-attention kernels (seq_attention_fwd.hip, seq_attention_bwd.hip).
//
// Every product runs on v_mfma_f32_32x32x16_bf16.  NP = bf16 planes per value: 1 for bf16 tensors, 3 for fp32 ones (x = h + m + l,
// split3.h; six plane products of order <= 2^-16 each, what is dropped is below 2^-24 of the operands' product).  DP = the head
// width padded to 32, 64 or 128 (columns beyond D are zeros in LDS).
//
// A 32 x 32 result tile: lane l holds column l & 31 and the rows 8 (i >> 2) + 4 (l >> 5) + (i & 3), i = 0 .. 15.  The kernels put the
// rows of softmax statistics on COLUMNS (one lane pair per row, no broadcast) and reuse a result tile as the right operand of the
// next product without moving it between lanes: the 16 contraction indices of a step are then {4 hi + 0..3, 8 + 4 hi + 0..3} per half
// wave hi, and the left operand is read from LDS in the same order (lds_tr, ds_read_b64_tr_b16: 4 rows of one column per lane).
//
// LDS tile: [rows][DP] bf16 per plane, 16-byte pieces XOR-swizzled by row so that both readers are free of bank conflicts: the row
// reader (16 consecutive rows, one piece each) and the transposing one (4 consecutive rows x 64 bytes per half wave).
//
// Times beside a choice are of both sides measured in turn when it was made; later steps moved both (the softmax sums' second parts cost the
// training steps 2 to 3 %).
#pragma once
#include "common.h"
#include "seq_geometry.h"
#include "split3.h"
#include "vec8.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) char* sa_lds;
typedef __attribute__((address_space(3))) bf16x4* sa_lds_tr;
typedef __attribute__((address_space(3))) bf16x8* sa_lds_v;

#define SA_LOG2E 1.4426950408889634f

struct SaK {
    int64_t Tq, Tk;
    int B, Hq, Hk, G, D, causal;
    float c;                               // scale * log2(e)
    float scale;
    int n_dist, n_buckets, reach, row;     // reach: largest |distance| with an entry of its own; row: sa_row_entries
    int vq, vk, vv, vo, vdo;               // elements per load of q, k, v, out, dout rows: 8, 4 or 1
    bool fast;                             // all of them 8, row strides below 2^23 elements (64 rows within 32-bit byte offsets)
    const void *q, *k, *v; int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    void* out; float* lse; float* out32;   // lse: [2][Hq][Tq] (sa_keep_sum)
    const int32_t *cu_q, *cu_k, *q_len, *k_len;
    const uint8_t* key_mask;
    const float* bias; const int32_t* buckets;
    const void* dout; int64_t do_row, do_head;
    void *dq, *dk, *dv; float* dbias; int accumulate;
    uint32_t* err_flag;
    // launch geometry
    int tiles, per_unit, units, together;  // column tiles per sequence, workgroups per (sequence, key head), B * Hk, sa_unit
    int rest;                              // units behind the last: they write the rows of no sequence
    unsigned blocks;                       // SaGrid's
    int pack;                              // query heads side by side in the columns (1 or G)
    int splits;                            // workgroups per key range
    float* part;                           // forward, splits > 1: [splits][Hq][Tq] (max, sum), then [splits][Hq][Tq][D]
    float* delta;                          // backward: [Hq][Tq]
    float* bias_part; int bias_slots;      // backward: [Hq][n_buckets][bias_slots]
};

// one sequence: first rows, rows present (the cu arrays' span), rows in use (q_len / k_len)
struct SaSeq {
    int64_t q0, k0;
    int q_span, k_span, lq, lk, shift;     // shift = lk - lq: query i stands at key position i + shift
};
__device__ __forceinline__ int64_t sa_clamp(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : (x > hi ? hi : x); }
__device__ __forceinline__ SaSeq sa_seq(const SaK& a, int b) {
    SaSeq s;
    const int64_t q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
    s.q0 = sa_clamp(q0, 0, a.Tq);
    s.k0 = sa_clamp(k0, 0, a.Tk);
    s.q_span = static_cast<int>(sa_clamp(q1, s.q0, a.Tq) - s.q0);
    s.k_span = static_cast<int>(sa_clamp(k1, s.k0, a.Tk) - s.k0);
    int lq = s.q_span, lk = s.k_span;
    bool bad = q0 < 0 || q1 < q0 || q1 > a.Tq || k0 < 0 || k1 < k0 || k1 > a.Tk;
    if (a.q_len) { const int n = a.q_len[b]; bad |= n < 0 || n > lq; lq = max(0, min(n, lq)); }
    if (a.k_len) { const int n = a.k_len[b]; bad |= n < 0 || n > lk; lk = max(0, min(n, lk)); }
    s.lq = lq; s.lk = lk; s.shift = lk - lq;
    if (bad && a.err_flag && threadIdx.x == 0) atomicOr(a.err_flag, SWR_FLAG_INDEX_OOR);
    return s;
}

template <int NP> struct SaT { typedef uint16_t type; };
template <> struct SaT<3> { typedef float type; };
template <int NP> using SaRaw = Raw8<typename SaT<NP>::type>;
// -> the planes of 8 values
__device__ __forceinline__ void sa_planes(const Raw8<uint16_t>& r, bf16x8 (&o)[1]) { o[0] = __builtin_bit_cast(bf16x8, r.v); }
__device__ __forceinline__ void sa_split8(const float* f, bf16x8 (&o)[3]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) SPLIT3_PAIR(f[j], f[j + 1], o[0], o[1], o[2], j);
}
__device__ __forceinline__ void sa_planes(const Raw8<float>& r, bf16x8 (&o)[3]) {
    float f[8];
    floats8(r, f);
    sa_split8(f, o);
}
// 8 fp32 values (probabilities, score gradients) as a right operand: rounded to bf16 once for bf16 tensors (2^-9 relative, the size
// of the rounding of the outputs themselves), split exactly for fp32 ones
__device__ __forceinline__ void sa_planes_f(const float* f, bf16x8 (&o)[3]) { sa_split8(f, o); }
__device__ __forceinline__ void sa_planes_f(const float* f, bf16x8 (&o)[1]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) CVT_PAIR(f[j], f[j + 1], o[0], j);
}

// ... and to 2^-17 in two planes: the probabilities of a training forward on bf16 tensors
__device__ __forceinline__ void sa_planes_f(const float* f, bf16x8 (&o)[2]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        CVT_PAIR(f[j], f[j + 1], o[0], j);
        const float r0 = f[j] - static_cast<float>(o[0][j]), r1 = f[j + 1] - static_cast<float>(o[0][j + 1]);
        CVT_PAIR(r0, r1, o[1], j);
    }
}

__device__ __forceinline__ f32x16 sa_mma(const bf16x8 (&a)[1], const bf16x8 (&b)[2], f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 sa_mma(const bf16x8 (&a)[1], const bf16x8 (&b)[1], f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 sa_mma(const bf16x8 (&a)[3], const bf16x8 (&b)[3], f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2], b[0], c, 0, 0, 0);     // smallest terms first
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 sa_zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// ---- LDS tile
template <int DP>
__device__ __forceinline__ int sa_swz(int row) {
    if (DP == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    if (DP == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    return (row >> 2) & 3;
}
template <int DP>
__device__ __forceinline__ int sa_off(int row, int chunk) { return row * (DP * 2) + ((chunk ^ sa_swz<DP>(row)) << 4); }

// x, with what is computed from it kept where it is used: addresses and comparisons hoisted out of the tile loops would fill the
// vector and scalar registers
__device__ __forceinline__ int sa_here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}
// the same for a uniform value (a flag: without it the loop it is constant in is compiled once for either value, with more registers)
__device__ __forceinline__ void sa_scalar_here(int& x) { asm volatile("" : "+s"(x)); }
// The kernel's arguments read again where they are used: what only the start and the end of a tile need does not sit in scalar
// registers through its inner loop.
typedef const __attribute__((address_space(4))) SaK* SaArgs;
__device__ __forceinline__ SaArgs sa_again() {
    SaArgs p = (SaArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}
// R rows of a [*, DP] operand moved by NT threads: global -> registers (load), registers -> LDS planes (store).
// FAST: 16-byte rows and D % 8 == 0 -- every lane loads from a valid address (the last row, the first columns) without a branch and
// what it should not have read becomes zeros on the way to LDS.  Otherwise 4 or 1 elements at a time under their conditions.
template <int NP, int DP, int R, int NT, bool FAST>
struct SaStage {
    static constexpr int CPR = DP / 8, N = R * CPR / NT, STEP = NT / CPR;
    static_assert(R * CPR % NT == 0 && NT % CPR == 0, "whole chunks per thread");
    static constexpr int PLANE = R * DP * 2, BYTES = NP * PLANE;
    typedef typename SaT<NP>::type T;
    SaRaw<NP> r[N];
    uint32_t keep;                         // bit i: r[i] counts (rows in use, not masked)
    // rows first .. first + R - 1 of a sequence whose row 0 is `row0`; rows >= limit (limit > first) or masked read as zeros
    __device__ __forceinline__ void load(const void* base, int64_t row0, int first, int limit, int64_t stride, int64_t head_off, int D, int vw,
                                         const uint8_t* mask) {
        const int tid = sa_here(threadIdx.x);
        const int chunk = tid % CPR, row = tid / CPR;
        const T* p = static_cast<const T*>(base) + (row0 + first) * stride + head_off;
        keep = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int rr = row + i * STEP;
            bool ok = first + rr < limit;
            const int rc = min(rr, limit - 1 - first);
            if (FAST) {
                r[i] = load8(p + static_cast<uint32_t>(rc) * static_cast<uint32_t>(stride) + (chunk * 8 < D ? chunk * 8 : 0), 8, 8);
                ok = ok && chunk * 8 < D;
            }
            if (mask) ok = ok && mask[row0 + first + rc] != 0;
            if (!FAST) r[i] = load8(p + rc * stride + chunk * 8, ok ? D - chunk * 8 : 0, vw);
            keep |= static_cast<uint32_t>(ok) << i;
        }
    }
    __device__ __forceinline__ void store(sa_lds dst) const {
        const int tid = sa_here(threadIdx.x);
        const int chunk = tid % CPR, row = tid / CPR;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            SaRaw<NP> x = r[i];
            if (FAST && !((keep >> i) & 1)) x = zero8(x);
            bf16x8 p[NP];
            sa_planes(x, p);
            const int off = sa_off<DP>(row + i * STEP, chunk);
#pragma unroll
            for (int pl = 0; pl < NP; ++pl) *reinterpret_cast<sa_lds_v>(dst + pl * PLANE + off) = p[pl];
        }
    }
};

// The same by LDS-DMA (bf16, FAST): 16-byte copies from HBM into the tile, no registers and no VALU in between.  The swizzle is in the
// source address (LDS places are lane-linear); rows and columns that do not count copy a zero piece.  Inline asm because the compiler
// would wait for every copy in flight in front of each LDS read; the kernels wait themselves (sa_dma_wait) before the barrier that
// hands a tile over.
static __device__ __attribute__((aligned(16))) uint32_t sa_zero_piece[4];
__device__ __forceinline__ void sa_dma16(uint32_t lds_addr, const void* src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_addr), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void sa_dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void sa_dma16(uint32_t lds_addr, uint32_t offset, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_addr), "v"(offset), "s"(base) : "memory", "m0");
}
template <int DP, int R, int NT>
struct SaDma {
    static constexpr int CPR = DP / 8, N = R * CPR / NT, STEP = NT / CPR;
    static_assert(R * CPR % NT == 0 && NT % CPR == 0, "whole chunks per thread");
    static __device__ __forceinline__ void copy(sa_lds dst, const void* base, int64_t row0, int first, int limit, int64_t stride, int64_t head_off, int D,
                                                const uint8_t* mask) {
        const int tid = sa_here(threadIdx.x);
        const int slot = tid % CPR, row = tid / CPR;
        const uint16_t* p = static_cast<const uint16_t*>(base) + (row0 + first) * stride + head_off;
        const uint32_t at = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(dst)) + (threadIdx.x & ~63u) * 16);
        if (D == DP && first + R <= limit && !mask) {              // every piece counts: one offset per lane, the rest is scalar
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int same = STEP % 16 == 0 ? row : row + i * STEP;        // (rows 16 apart have the same swizzle)
                sa_dma16(at + i * NT * 16, 2 * (static_cast<uint32_t>(row) * static_cast<uint32_t>(stride) + (slot ^ sa_swz<DP>(same)) * 8), p + i * STEP * stride);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int rr = row + i * STEP, col = (slot ^ sa_swz<DP>(rr)) * 8;
            bool ok = first + rr < limit && col < D;
            if (mask) ok = ok && mask[row0 + first + rr] != 0;
            sa_dma16(at + i * NT * 16, ok ? static_cast<const void*>(p + static_cast<uint32_t>(rr) * static_cast<uint32_t>(stride) + col)
                                          : static_cast<const void*>(sa_zero_piece));
        }
    }
};

// What a lane reads of a tile.  Both readers' byte offsets are a lane constant XOR a compile-time constant (the swizzle only sees the
// low row bits), so one instruction makes an address; `fresh` keeps the compiler from hoisting dozens of them out of the tile loop
// into registers.
template <int NP, int DP, int R>
struct SaLane {
    int row, col;
    __device__ __forceinline__ SaLane(int lane) {
        row = sa_off<DP>(lane & 31, lane >> 5);
        const int chunk = ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1);
        col = sa_off<DP>(4 * (lane >> 5) + ((lane >> 2) & 3), chunk) + (lane & 1) * 8;
    }
    __device__ __forceinline__ void fresh() { asm volatile("" : "+v"(row), "+v"(col)); }
    // left operand of a product over the columns: row (lane & 31) of block rb, columns 16 s + 8 hi .. + 7
    __device__ __forceinline__ void rows(sa_lds tile, int rb, int s, bf16x8 (&o)[NP]) const {
        const sa_lds p = tile + rb * (32 * DP * 2) + (row ^ (s << 5));
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) o[pl] = *reinterpret_cast<sa_lds_v>(p + pl * (R * DP * 2));
    }
    // left operand of a product over the rows: column 32 db + (lane & 31), rows 16 ks + {4 hi + 0..3, 8 + 4 hi + 0..3}
    __device__ __forceinline__ void cols(sa_lds tile, int ks, int db, bf16x8 (&o)[NP]) const {
        const sa_lds p0 = tile + ks * (16 * DP * 2) + (col ^ (db << 6)), p1 = tile + ks * (16 * DP * 2) + 8 * DP * 2 + (col ^ (db << 6) ^ (2 << 4));
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) {
            const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(reinterpret_cast<sa_lds_tr>(p0 + pl * (R * DP * 2)));
            const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(reinterpret_cast<sa_lds_tr>(p1 + pl * (R * DP * 2)));
            o[pl] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};
// N groups of left operands one ahead of their products: load(buffer, i) brings group i from LDS into registers, mul(buffer, i) uses it
// -- a read right in front of its product makes the matrix instruction wait for LDS.  Without FIRST the first group has been loaded
// before.  Measured (without it): training steps of 24 packed sequences up to 2 048, heads of 64, bf16, 0.91 / 1.00 ms, of 4 sequences up
// to 4 096, heads of 128, 1.22 / 1.32 ms; prompts up to 8 192 2.29 / 2.44 ms; 64 fp32 sequences up to 600 both ways 0.148 / 0.155 ms.
// Two or four groups together take the same times, a fence between read and product 1 % more.
template <int N, bool FIRST, class Load, class Mul>
__device__ __forceinline__ void sa_ahead(Load load, Mul mul) {
    if (FIRST) load(0, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i + 1 < N) load((i + 1) & 1, i + 1);
        mul(i & 1, i);
    }
}
// right operand held in registers: row `off` (elements) of a matrix, columns 16 s + 8 hi .. + 7 (zeros beyond D or where !ok)
// (FAST: `off` has to be a valid row where !ok, too)
template <int NP, bool FAST>
__device__ __forceinline__ SaRaw<NP> sa_row8(const void* base, int64_t off, int col, bool ok, int D, int vw) {
    const typename SaT<NP>::type* p = static_cast<const typename SaT<NP>::type*>(base) + off;
    if (!FAST) return load8(p + col, ok ? D - col : 0, vw);
    const SaRaw<NP> x = load8(p + (col < D ? col : 0), 8, 8);
    return ok && col < D ? x : zero8(x);
}
template <int NP, int DP, bool FAST>
__device__ __forceinline__ void sa_row_frags(const void* base, int64_t off, bool ok, int D, int vw, int lane, bf16x8 (&o)[DP / 16][NP]) {
    const int col = sa_here(8 * (lane >> 5));
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) sa_planes(sa_row8<NP, FAST>(base, off, 16 * s + col, ok, D, vw), o[s]);
}

// ... kept as loaded and split at every use where the planes of two operands do not fit the registers (fp32, D > 64: 192 of them)
template <int NP, int DP, bool FAST, bool SPLIT_LATE>
struct SaRows {
    bf16x8 p[DP / 16][NP];
    __device__ __forceinline__ void load(const void* base, int64_t off, bool ok, int D, int vw, int lane) {
        sa_row_frags<NP, DP, FAST>(base, off, ok, D, vw, lane, p);
    }
    __device__ __forceinline__ void get(int s, bf16x8 (&o)[NP]) const {
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) o[pl] = p[s][pl];
    }
};
template <int NP, int DP, bool FAST>
struct SaRows<NP, DP, FAST, true> {
    SaRaw<NP> r[DP / 16];
    __device__ __forceinline__ void load(const void* base, int64_t off, bool ok, int D, int vw, int lane) {
        const int col = sa_here(8 * (lane >> 5));
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) r[s] = sa_row8<NP, FAST>(base, off, 16 * s + col, ok, D, vw);
    }
    __device__ __forceinline__ void get(int s, bf16x8 (&o)[NP]) const {
        float f[8];
        floats8(r[s], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(f[j]));       // (the split stays in the loop: hoisted, its planes spill)
        sa_split8(f, o);
    }
};

// What the forward keeps of a row's softmax, in two parts: p = 2^(x - first) second.  first = m + log2 l and second = 1 where m is small
// enough that the sum keeps log2 l to 2^-18; beside a large m (large scores, a large bias on every key of the row) it would be rounded away
// and p would no longer sum to one (to the number of keys at the type's lowest value): there first = m, which x is near, second = 1 / l.
// A row without a key: +inf, 1.  The backward reads second parts only where a row's first says that there may be one (sa_parts).
__device__ __forceinline__ bool sa_parts(float first) { return fabsf(first) > 64.f && first != INFINITY; }
__device__ __forceinline__ void sa_keep_sum(float* lse, int64_t at, int64_t rows, float m, float l) {
    const bool two = l != 0.f && sa_parts(m);
    lse[at] = l == 0.f ? INFINITY : (two ? m : m + __builtin_amdgcn_logf(l));
    lse[rows + at] = two ? 1.f / l : 1.f;
}

// 4 consecutive result columns d .. d + 3 of a row at `p` (row of D elements)
template <int NP>
__device__ __forceinline__ void sa_store4(void* base, int64_t row_off, int d, int D, const float* x) {
    if (d >= D) return;
    if (NP == 3) {
        float* p = static_cast<float*>(base) + row_off + d;
        if ((D & 3) == 0) {
            *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d + j < D) p[j] = x[j];
        }
    } else {
        uint16_t* p = static_cast<uint16_t*>(base) + row_off + d;
        bf16x4 v;
        CVT_PAIR(x[0], x[1], v, 0);
        CVT_PAIR(x[2], x[3], v, 2);
        const uint2 w = __builtin_bit_cast(uint2, v);
        if ((D & 3) == 0) {
            *reinterpret_cast<uint2*>(p) = w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d + j < D) p[j] = static_cast<uint16_t>((j < 2 ? w.x : w.y) >> (16 * (j & 1)));
        }
    }
}

// ---- workgroup -> (unit = sequence and key head, work item inside it).  Consecutive workgroups go to the 8 XCDs in turn: all
// workgroups of a unit stay on one XCD, whose L2 holds the unit's keys and values.  The XCD's units go in rounds of `together`: item 0
// of each, then item 1, ...  With all of them in one round the heaviest items of long and short sequences start first and no long one
// is left for the end; with one at a time its keys stay in the L2 (4 MB) while its workgroups run.  Measured, unit by unit against all
// in one round: training steps (their backward) of 24 packed sequences up to 2 048, heads of 64, bf16, 1.03 / 0.88 ms, of 4 sequences
// up to 4 096, heads of 128, 1.48 / 1.32 ms; forward of 8 prompts up to 8 192, heads of 128, 2.90 / 3.05 ms, of 64 both ways up to 600,
// fp32, 0.157 / 0.173 ms.  So the backward takes one round, the forward one unit at a time.
__device__ __forceinline__ int sa_unit(int id, int per_unit, int together, int& within) {
    const int slot = id >> 3, round = slot / (per_unit * together), r = slot % (per_unit * together);
    within = r / together;
    return (round * together + r % together) * 8 + (id & 7);
}

// Position bias in LDS: one row per head, entry (distance + SA_PAD), with the table's ends repeated and, causal, -inf below distance
// 0 (which masks): a 32 x 32 block that touches the table reads it at one base per lane and constant offsets, without a clamp or a
// comparison.  Blocks wholly beyond the reach take one value.  Without a bias the row is that of a one-entry table of 0, both ways none.
#define SA_PAD 64
__host__ __device__ __forceinline__ int sa_row_entries(int n_dist, int reach, int causal) {
    return (n_dist || causal) ? ((causal ? reach : 2 * reach) + 2 * SA_PAD + 1 + 3) & ~3 : 0;        // (a multiple of 4: what follows is aligned)
}
// bias in the exponent's base-2 unit; a finite value stays finite (a bias of the type's lowest value masks relative to the row's
// other scores, it does not empty the row)
__device__ __forceinline__ float sa_bias2(float b) {
    const float x = b * SA_LOG2E;
    return (__builtin_isinf(x) && !__builtin_isinf(b)) ? copysignf(3.402823466e38f, x) : x;
}
// Scores are fp32 values, s = S c + bias rounded once: a large bias absorbs digits of the products, all of them at the type's lowest
// value.  Every block of a row has to round alike, or the same keys weigh differently in blocks of one bias (whose raw products would
// enter beside bias - maximum, and overflow) and in blocks that touch the table.  Up to 2^10 the digits lost are below 2^-14 of a score,
// and the one fma of raw products, bias and maximum stays.  (-inf absorbs everything in either form.)
__device__ __forceinline__ bool sa_wide(float add) { return fabsf(add) > 1024.f && add != -INFINITY; }
__device__ __forceinline__ int sa_bucket(const SaK& a, int i) { return max(0, min(a.buckets[i], a.n_buckets - 1)); }
// rows of heads h .. h + heads - 1.  A value is two loads deep (bucket, bias) and a single token's whole work is a few loads deep: every
// thread has the buckets of several entries in flight, then their values (one wave, 193 entries, one after the other: the query pass of
// 1 024 histories up to 50 took 61 us, so 49).
template <int NT>
__device__ __forceinline__ void sa_bias_rows(const SaK& a, int h, int heads, float* rows) {
    constexpr int U = 512 / NT;
    const int low = a.causal ? 0 : -a.reach, n = heads * a.row;
    for (int i0 = threadIdx.x; i0 < n; i0 += U * NT) {
        int d[U], at[U];
        float x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(i0 + u * NT, n - 1), hh = i / a.row;
            d[u] = i - hh * a.row - SA_PAD + low;
            at[u] = (h + hh) * a.n_buckets;
            x[u] = 0.f;
        }
        if (a.n_dist) {
            int bu[U];
#pragma unroll
            for (int u = 0; u < U; ++u) bu[u] = a.buckets[max(low, min(d[u], a.reach)) - low];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = a.bias[at[u] + max(0, min(bu[u], a.n_buckets - 1))];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * NT < n) rows[i0 + u * NT] = a.causal && d[u] < 0 ? -INFINITY : sa_bias2(x[u]);
    }
}
// what a block whose distances span near .. far needs: 0 = one value (at .x of the row), 1 = the row
struct SaSpan { bool apart; int entry; };
__device__ __forceinline__ SaSpan sa_span(const SaK& a, int near_d, int far_d) {
    SaSpan s;
    const bool hi = near_d >= a.reach, lo = !a.causal && far_d <= -a.reach;
    s.apart = a.row == 0 || hi || lo;
    s.entry = hi ? (a.causal ? a.reach : 2 * a.reach) + SA_PAD : SA_PAD;
    return s;
}
// whether the bias beyond the reach (either side) is sa_wide for one of this lane's of the heads h .. h + heads - 1
__device__ __forceinline__ bool sa_wide_ends(const SaK& a, int h, int heads, int lane) {
    bool w = false;
    if (a.n_dist) {
        const int near_b = sa_bucket(a, 0), far_b = sa_bucket(a, a.n_dist - 1);
        for (int i = lane; i < heads; i += 64) {
            const float* b = a.bias + (h + i) * a.n_buckets;
            w |= sa_wide(sa_bias2(b[far_b])) || (!a.causal && sa_wide(sa_bias2(b[near_b])));
        }
    }
    return w;
}
// the first of 28 entries that hold a block's one value (the padded ends; SA_FLAT zeros where there is no row): the backward's form for it in
// a row whose lse is in two parts
#define SA_FLAT 28
__device__ __forceinline__ int sa_flat_entry(const SaK& a, SaSpan s) { return a.row == 0 || (s.entry == SA_PAD && a.reach) ? 0 : s.entry; }
// entry of distance d
__device__ __forceinline__ int sa_entry(const SaK& a, int d) { return d + SA_PAD + (a.causal ? 0 : a.reach); }
// hidden key of result row i (km: the block's flags from row 4 hi on, 4-byte aligned)
__device__ __forceinline__ bool sa_masked(const uint8_t* km, int i) {
    return ((*reinterpret_cast<const uint32_t*>(km + 8 * (i >> 2)) >> (8 * (i & 3))) & 0xff) == 0;
}
// rows outside every sequence (before the first, behind the last) are zeros in every output: the work of the units behind the last
// one.  base is 16-byte aligned; the edges of a span that is not go 2 bytes at a time.
__device__ __forceinline__ void sa_zero_rows(void* base, int elem, int64_t r0, int64_t r1, int64_t row_elems, int nthreads, int part, int parts) {
    char* p = static_cast<char*>(base);
    const int64_t n0 = r0 * row_elems * elem, n1 = r1 * row_elems * elem;
    if (n0 >= n1) return;
    const int64_t a0 = min((n0 + 15) & ~15ll, n1), a1 = max(n1 & ~15ll, a0);
    if (part == 0) {
        for (int64_t i = n0 + 2 * threadIdx.x; i < a0; i += 2 * nthreads) *reinterpret_cast<uint16_t*>(p + i) = 0;
        for (int64_t i = a1 + 2 * threadIdx.x; i < n1; i += 2 * nthreads) *reinterpret_cast<uint16_t*>(p + i) = 0;
    }
    for (int64_t i = a0 + 16 * (static_cast<int64_t>(part) * nthreads + threadIdx.x); i < a1; i += 16ll * nthreads * parts)
        *reinterpret_cast<uint4*>(p + i) = make_uint4(0, 0, 0, 0);
}
