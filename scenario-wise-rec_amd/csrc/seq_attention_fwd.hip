// Attention over packed sequences, forward: whole prompts, training, and a few new tokens over cached keys.
//
//   s_ij = scale q_i . k_j + bias[h, bucket(i + lk - lq - j)],   p_ij = softmax over the allowed j,   o_i = sum_j p_ij v_j
//
// allowed: j < lk, key_mask[j], and j <= i + lk - lq when causal (the last query stands at the last key).  One pass over the keys with
// the running maximum m and sum l of every row (both fp32, base-2 exponents: p = 2^(x - m), x = s log2 e); a row without an allowed
// key keeps l = 0 and is written as zeros.  Saved for the backward: m + log2 l, in two parts where m is large (+inf for an empty row: every
// p becomes 0).
//
// A workgroup holds NW x 32 columns = query rows (token-major, `pack` heads of a key head side by side), S^T = K Q^T and
// O^T = V^T P^T (seq_attention.h); the keys and values of a tile are staged in LDS once for all its columns.  Few queries: the key
// range is cut into `splits` workgroups whose (m, l, O) a second launch joins.
#include <algorithm>

#include "seq_attention.h"

// waves per SIMD the registers are bounded for (512 / waves each): as many as spill nothing.  (One wave a workgroup at DP = 64, fp32, and at
// DP = 128, bf16, would bear one more; these are launches of few columns, whose workgroups do not fill the chip.)
#define SA_WAVES(NP, DP, NW) ((NP) * (DP) >= 384 || ((NP) * (DP) == 192 && (NW) < 4) || ((NP) * (DP) == 128 && (NW) == 1) ? 1 : (((DP) == 32 && (NW) == 1) || (NP) * (DP) == 64 ? 3 : 2))

template <int NP, int DP, int NW, bool FAST>
struct SaFwd {
    static constexpr bool DMA = FAST && NP == 1;               // two buffers filled by LDS-DMA; else one, through registers
    // keys per tile: 64 where two waves a SIMD have the registers for it, 32 where that makes room for a third (bf16, D <= 64: 0.896 /
    // 0.880 ms for the packed training step) or where one wave stages alone (prompts of 128 a head, 64 against 32: 2.49 / 2.57 ms)
    static constexpr int KT = (NW == 1 || (DP == 128 && !(DMA && NW == 4)) || (NP == 1 && DP == 64)) ? 32 : 64, NBUF = DMA ? 2 : 1;
    static constexpr int TILE = NP * KT * DP * 2;
    static int lds(const SaK& a) { return NBUF * (2 * TILE + KT) + a.pack * a.row * 4; }
};

// TRAIN (bf16): the probabilities enter the second product in two planes and the unrounded rows are kept.  The backward's delta = do . o
// has to agree with its fp32 sums of p (do . v): with o from probabilities rounded to 2^-9 the bias gradient, whose terms nearly cancel
// in every row, was off by 2.8e-3 of its norm.
template <int NP, int DP, int NW, bool FAST, bool TRAIN>
__global__ __launch_bounds__(NW * 64, SA_WAVES(NP, DP, NW)) void seq_attention_fwd_kernel(const SaK a) {
    typedef SaFwd<NP, DP, NW, FAST> Cfg;
    constexpr int KT = Cfg::KT, KB = KT / 32, NT = NW * 64, QT = NW * 32, TILE = Cfg::TILE;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    uint8_t* km0 = reinterpret_cast<uint8_t*>(smem) + Cfg::NBUF * 2 * TILE;
    float* bt = reinterpret_cast<float*>(km0 + Cfg::NBUF * KT);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5;
    SaLane<NP, DP, KT> ln(lane);

    int within;
    const int unit = sa_unit(blockIdx.x, a.per_unit, a.together, within);
    if (unit >= a.units) {                     // rows of no sequence
        if (unit >= a.units + a.rest) return;
        const int part = (unit - a.units) * a.per_unit + within, parts = a.rest * a.per_unit;
        const int64_t end0 = sa_clamp(a.cu_q[0], 0, a.Tq), beg1 = sa_clamp(a.cu_q[a.B], end0, a.Tq);
        if (a.splits == 1) {
            const int64_t row = static_cast<int64_t>(a.Hq) * a.D;
            sa_zero_rows(a.out, NP == 3 ? 4 : 2, 0, end0, row, NT, part, parts);
            sa_zero_rows(a.out, NP == 3 ? 4 : 2, beg1, a.Tq, row, NT, part, parts);
        }
        const int64_t n_tail = end0 + a.Tq - beg1, heads = static_cast<int64_t>(a.Hq) * (a.splits > 1 ? a.splits : 1);
        for (int64_t i = static_cast<int64_t>(part) * NT + threadIdx.x; i < n_tail * heads; i += static_cast<int64_t>(parts) * NT) {
            const int64_t h = i / n_tail, r = i % n_tail, at = h * a.Tq + (r < end0 ? r : beg1 + r - end0);
            if (a.splits > 1) { a.part[2 * at] = -INFINITY; a.part[2 * at + 1] = 0.f; }
            else if (a.lse) a.lse[at] = INFINITY;
        }
        return;
    }
    const int b = unit / a.Hk, hk = unit % a.Hk;
    const int split = within % a.splits;
    within /= a.splits;
    const int ng = a.G / a.pack, g = within % ng;
    const SaSeq sq = sa_seq(a, b);
    const int h0 = hk * a.G + g;
    if (a.n_dist && a.err_flag && unit == 0) {
        for (int i = threadIdx.x; i < a.n_dist; i += NT)
            if (a.buckets[i] < 0 || a.buckets[i] >= a.n_buckets) atomicOr(a.err_flag, SWR_FLAG_INDEX_OOR);
    }

    const int ncol = sq.q_span * a.pack;       // (below 2^31: the host packs heads only where all rows' columns are)
    const int64_t tile0 = a.tiles - 1 - within / ng;
    int wide = 0;                              // the bias of blocks beyond the reach (either side) is sa_wide
    for (int64_t tile = tile0; tile * QT < ncol; tile += a.tiles) {
        const int col0 = static_cast<int>(tile * QT) + wave * 32, col = col0 + (lane & 31);
        const int tok = min(col, ncol) / a.pack, hsub = col % a.pack, h = h0 + hsub;
        const bool exists = col < ncol, live = exists && tok < sq.lq;
        const int qpos = tok + sq.shift;
        // the wave's and the workgroup's token range; keys any of them may read
        const int wfirst = min(col0, ncol) / a.pack, wlast = min(sq.lq, min(col0 + 31, ncol - 1) / a.pack + 1) - 1;
        const int bfirst = static_cast<int>(tile * QT) / a.pack;
        const int blast = min(sq.lq, min(static_cast<int>(tile * QT) + QT - 1, ncol - 1) / a.pack + 1) - 1;
        int kend = a.causal ? min(sq.lk, blast + sq.shift + 1) : sq.lk;
        if (bfirst >= sq.lq || kend < 0) kend = 0;
        const int ntile = (kend + KT - 1) / KT;
        const int t0 = static_cast<int>(static_cast<int64_t>(ntile) * split / a.splits);
        const int t1 = static_cast<int>(static_cast<int64_t>(ntile) * (split + 1) / a.splits);

        SaStage<NP, DP, KT, NT, FAST> sk, sv;
        uint8_t mk = 1;
        auto fetch = [&](int t, int buf) {
            if (Cfg::DMA) {
                const sa_lds to = (sa_lds)smem + buf * 2 * TILE;
                SaDma<DP, KT, NT>::copy(to, a.k, sq.k0, t * KT, sq.lk, a.k_row, hk * a.k_head, a.D, a.key_mask);
                SaDma<DP, KT, NT>::copy(to + TILE, a.v, sq.k0, t * KT, sq.lk, a.v_row, hk * a.v_head, a.D, a.key_mask);
            } else {
                sk.load(a.k, sq.k0, t * KT, sq.lk, a.k_row, hk * a.k_head, a.D, a.vk, a.key_mask);
                sv.load(a.v, sq.k0, t * KT, sq.lk, a.v_row, hk * a.v_head, a.D, a.vv, a.key_mask);
            }
            if (a.key_mask && threadIdx.x < KT) {
                const int key = t * KT + threadIdx.x;
                mk = key < sq.lk ? a.key_mask[sq.k0 + key] : 0;
            }
        };
        // the first tile's loads go out before anything waits (a column tile before this one has been read: barrier first)
        if (tile != tile0) __syncthreads();
        if (t0 < t1) fetch(t0, 0);
        bf16x8 Q[DP / 16][NP];
        sa_row_frags<NP, DP, FAST>(a.q, (sq.q0 + (exists ? tok : 0)) * a.q_row + static_cast<int64_t>(h) * a.q_head, live, a.D, a.vq, lane, Q);
        f32x16 O[DP / 32];
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) O[db] = sa_zero16();
        float m = -INFINITY, l = 0.f;

        if (tile == tile0) {
            const bool ends = sa_wide_ends(a, h0, a.pack, lane);       // (in flight beside the rows')
            sa_bias_rows<NT>(a, h0, a.pack, bt);
            wide = __builtin_amdgcn_readfirstlane(__any(ends));
        }
        for (int t = t0; t < t1; ++t) {
            const int buf = Cfg::DMA ? (t - t0) & 1 : 0;
            const sa_lds kt = (sa_lds)smem + buf * 2 * TILE, vt = kt + TILE;
            const uint8_t* km = km0 + buf * KT;
            if (Cfg::DMA) {
                // one barrier: the copies of this tile have landed, the readers of the other buffer are done
                if (a.key_mask && threadIdx.x < KT) km0[buf * KT + threadIdx.x] = mk;
                sa_dma_wait();
                __syncthreads();
            } else {
                if (t > t0) __syncthreads();           // (the tile's readers are done)
                sk.store(kt);
                sv.store(vt);
                if (a.key_mask && threadIdx.x < KT) km0[threadIdx.x] = mk;
                __syncthreads();
            }
            if (t + 1 < t1) fetch(t + 1, buf ^ 1);
            sa_scalar_here(wide);
            const int k0 = t * KT;
            if (wfirst > wlast || (a.causal && k0 > wlast + sq.shift)) continue;

            ln.fresh();
            f32x16 S[KB];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) S[kb] = sa_zero16();
            {
                constexpr int NS = DP / 16;
                bf16x8 A[2][NP];
                sa_ahead<KB * NS, true>([&](int b, int i) { ln.rows(kt, i / NS, i % NS, A[b]); },
                                        [&](int b, int i) { S[i / NS] = sa_mma(A[b], Q[i % NS], S[i / NS]); });
            }
            // (the second product's first operands come in under the exponentials)
            bf16x8 T[2][DP / 32][NP];
            auto cols = [&](int b, int ks) {
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) ln.cols(vt, ks, db, T[b][db]);
            };
            cols(0, 0);
            // A block's exponents are x = S mul + add: a block of one bias keeps the raw products (mul = c, folded into one fma with the
            // row's maximum below), one that touches the table or hides keys is written out (mul = 1, add = 0), and so is one whose bias
            // absorbs digits of the products (sa_wide).
            const float* bh = bt + hsub * a.row;
            float mul[KB], add[KB], mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const int kf = k0 + kb * 32;
                const SaSpan sp = sa_span(a, wfirst + sq.shift - (kf + 31), wlast + sq.shift - kf);
                const bool cut = !a.causal && kf + 32 > sq.lk;                    // (causal: keys behind the last are masked by distance)
                mul[kb] = a.c;
                add[kb] = sp.apart && a.row ? bh[sp.entry] : 0.f;
                if (!sp.apart || cut || a.key_mask || a.c < 0.f || wide) {
                    if (sp.apart) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) S[kb][i] = S[kb][i] * a.c + add[kb];
                    } else if (!a.causal || kf <= wlast + sq.shift) {
                        const float* be = bh + sa_entry(a, qpos - kf - 4 * hi - 27);
#pragma unroll
                        for (int i = 0; i < 16; ++i) S[kb][i] = S[kb][i] * a.c + be[27 - 8 * (i >> 2) - (i & 3)];
                    } else {                   // a block no query of the wave may see
#pragma unroll
                        for (int i = 0; i < 16; ++i) S[kb][i] = -INFINITY;
                    }
                    mul[kb] = 1.f;
                    add[kb] = 0.f;
                    if (cut) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) S[kb][i] = kf + 4 * hi + 8 * (i >> 2) + (i & 3) < sq.lk ? S[kb][i] : -INFINITY;
                    }
                    if (a.key_mask) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) S[kb][i] = sa_masked(km + kb * 32 + 4 * hi, i) ? -INFINITY : S[kb][i];
                    }
                }
                float top = S[kb][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxf(top, S[kb][i]);
                mx = fmaxf(mx, top * mul[kb] + add[kb]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            // The reference exponent m follows the maximum only in steps of 2^8 (p and l stay below 2^8 times the row's length): O is
            // rescaled in the first tile and hardly ever again, not whenever one of 32 rows finds a new maximum.
            if (__any(mx > m + 8.f)) {
                const float up = mx > m + 8.f ? mx : m;
                const float corr = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - up);
                m = up;
                l *= corr;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) O[db][i] *= corr;
            }
            const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const float sh = add[kb] - ms;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    S[kb][i] = __builtin_amdgcn_exp2f(S[kb][i] * mul[kb] + sh);
                    sum += S[kb][i];
                }
                l += sum;
            }
            sa_ahead<KT / 16, false>(cols, [&](int b, int ks) {
                float pf[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) pf[j] = S[ks >> 1][8 * (ks & 1) + j];
                bf16x8 P[TRAIN ? 2 : NP];
                sa_planes_f(pf, P);
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) O[db] = sa_mma(T[b][db], P, O[db]);
            });
        }
        l += __shfl_xor(l, 32);
        if (!live) {                           // a column without a query went through the products as a row of zeros
            m = -INFINITY;
            l = 0.f;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) O[db] = sa_zero16();
        }
        if (exists) {
            const int hi4 = sa_here(4 * hi);
            const int64_t at = static_cast<int64_t>(h) * a.Tq + sq.q0 + tok;
            if (a.splits == 1) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const int64_t row = ((sq.q0 + tok) * a.Hq + h) * a.D;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float x[4] = {O[db][i] * inv, O[db][i + 1] * inv, O[db][i + 2] * inv, O[db][i + 3] * inv};
                        sa_store4<NP>(a.out, row, db * 32 + 2 * i + hi4, a.D, x);
                        if (TRAIN) sa_store4<3>(a.out32, row, db * 32 + 2 * i + hi4, a.D, x);
                    }
                if (a.lse && hi == 0) sa_keep_sum(a.lse, at, static_cast<int64_t>(a.Hq) * a.Tq, m, l);
            } else {
                const int64_t pr = split * static_cast<int64_t>(a.Hq) * a.Tq + at;
                if (hi == 0) { a.part[2 * pr] = m; a.part[2 * pr + 1] = l; }
                float* po = a.part + 2ll * a.splits * a.Hq * a.Tq + pr * DP;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<float4*>(po + db * 32 + 2 * i + hi4) = make_float4(O[db][i], O[db][i + 1], O[db][i + 2], O[db][i + 3]);
            }
        }
    }
}

// joins the key ranges of a row: 32 lanes per (head, row), fixed order over the ranges
template <int NP, int DP>
__global__ __launch_bounds__(256) void seq_attention_join_kernel(const SaK a) {
    const int64_t rows = static_cast<int64_t>(a.Hq) * a.Tq;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (at >= rows) return;
    const int j = threadIdx.x & 31;
    float M = -INFINITY;
    for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.part[2 * (s * rows + at)]);
    const float ms = M == -INFINITY ? 0.f : M;
    float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
        const float l = a.part[2 * (s * rows + at) + 1];
        if (l == 0.f) continue;                                    // (no key of this range: its O was not written for rows of no sequence)
        const float w = __builtin_amdgcn_exp2f(a.part[2 * (s * rows + at)] - ms);
        L += l * w;
        if (4 * j < DP) {
            const float4 p = *reinterpret_cast<const float4*>(a.part + 2 * a.splits * rows + (s * rows + at) * DP + 4 * j);
            o[0] += w * p.x; o[1] += w * p.y; o[2] += w * p.z; o[3] += w * p.w;
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int64_t h = at / a.Tq, t = at % a.Tq;
    const float x[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    sa_store4<NP>(a.out, (t * a.Hq + h) * a.D, 4 * j, a.D, x);
    if (NP == 1 && a.out32) sa_store4<3>(a.out32, (t * a.Hq + h) * a.D, 4 * j, a.D, x);
    if (a.lse && j == 0) sa_keep_sum(a.lse, at, rows, M, L);
}

// ------------------------------------------------------------------------------------------------------------------- host
int sa_check(const swr_seq_attention_args* p, bool backward) {
    SWR_REQUIRE(p, SWR_ERR_ARG);
    SWR_REQUIRE(p->B >= 0 && p->Tq >= 0 && p->Tk >= 0 && p->max_q >= 0 && p->max_k >= 0, SWR_ERR_ARG);
    SWR_REQUIRE(p->Tq < (1ll << 31) - 4096 && p->Tk < (1ll << 31) - 4096, SWR_ERR_UNSUPPORTED);
    SWR_REQUIRE(p->dtype == SWR_F32 || p->dtype == SWR_BF16, SWR_ERR_DTYPE);
    SWR_REQUIRE(p->D >= 1 && p->Hk >= 1 && p->Hq >= p->Hk, SWR_ERR_ARG);
    SWR_REQUIRE(p->D <= SWR_SEQ_MAX_DIM && p->Hq % p->Hk == 0, SWR_ERR_UNSUPPORTED);
    SWR_REQUIRE(p->cu_q && p->cu_k && p->out, SWR_ERR_ARG);
    SWR_REQUIRE(p->Tq == 0 || p->q, SWR_ERR_ARG);
    SWR_REQUIRE(p->Tk == 0 || (p->k && p->v), SWR_ERR_ARG);
    SWR_REQUIRE(p->n_dist >= 0, SWR_ERR_ARG);
    if (p->n_dist) {
        SWR_REQUIRE(p->bias && p->buckets && p->n_buckets >= 1, SWR_ERR_ARG);
        SWR_REQUIRE(p->n_dist <= SWR_SEQ_MAX_DIST && p->n_buckets <= SWR_SEQ_MAX_BUCKETS && (p->causal || p->n_dist % 2 == 1), SWR_ERR_UNSUPPORTED);

    }
    // (the bias rows of a group and the per-distance sums have their place in LDS beside the tiles)
    const int64_t reach = p->n_dist ? (p->causal ? p->n_dist - 1 : p->n_dist / 2) : 0;
    SWR_REQUIRE(static_cast<int64_t>(sa_row_entries(p->n_dist, static_cast<int>(reach), p->causal)) * (p->Hq / p->Hk) <= SWR_SEQ_MAX_TABLE, SWR_ERR_UNSUPPORTED);
    SWR_REQUIRE(static_cast<int64_t>(p->B) * p->Hk < (1ll << 30), SWR_ERR_UNSUPPORTED);
    SWR_REQUIRE(((reinterpret_cast<uintptr_t>(p->out) | reinterpret_cast<uintptr_t>(p->out32)) & 15) == 0, SWR_ERR_ALIGN);
    if (backward) {
        SWR_REQUIRE(p->lse && (p->out32 || p->dtype == SWR_F32) && p->dout && p->dq && p->dk && p->dv, SWR_ERR_ARG);
        SWR_REQUIRE(((reinterpret_cast<uintptr_t>(p->dq) | reinterpret_cast<uintptr_t>(p->dk) | reinterpret_cast<uintptr_t>(p->dv)) & 15) == 0, SWR_ERR_ALIGN);
    }
    return SWR_OK;
}

SaK sa_args(const swr_seq_attention_args* p) {
    SaK a{};
    const int elem = p->dtype == SWR_F32 ? 4 : 2;
    a.Tq = p->Tq; a.Tk = p->Tk; a.B = p->B; a.Hq = p->Hq; a.Hk = p->Hk; a.G = p->Hq / p->Hk; a.D = p->D; a.causal = p->causal != 0;
    a.scale = p->scale; a.c = p->scale * SA_LOG2E;
    a.n_dist = p->n_dist; a.n_buckets = p->n_buckets; a.reach = p->n_dist ? (p->causal ? p->n_dist - 1 : p->n_dist / 2) : 0;
    a.row = sa_row_entries(p->n_dist, a.reach, a.causal);
    a.q = p->q; a.k = p->k; a.v = p->v;
    a.q_row = p->q_row; a.q_head = p->q_head; a.k_row = p->k_row; a.k_head = p->k_head; a.v_row = p->v_row; a.v_head = p->v_head;
    a.vq = swr_vec8(p->q, p->q_row, p->q_head, p->D, elem);
    a.vk = swr_vec8(p->k, p->k_row, p->k_head, p->D, elem);
    a.vv = swr_vec8(p->v, p->v_row, p->v_head, p->D, elem);
    a.vo = swr_vec8(p->out, static_cast<int64_t>(p->Hq) * p->D, p->D, p->D, 4);
    a.vdo = swr_vec8(p->dout, p->do_row, p->do_head, p->D, elem);
    const int64_t far = 1ll << 23;
    a.fast = a.vq == 8 && a.vk == 8 && a.vv == 8 && (!p->dout || a.vdo == 8) && p->q_row < far && p->k_row < far && p->v_row < far && p->do_row < far;
    a.out32 = p->dtype == SWR_F32 ? static_cast<float*>(p->out) : p->out32;
    a.out = p->out; a.lse = p->lse; a.cu_q = p->cu_q; a.cu_k = p->cu_k; a.q_len = p->q_len; a.k_len = p->k_len; a.key_mask = p->key_mask;
    a.bias = p->bias; a.buckets = p->buckets; a.dout = p->dout; a.do_row = p->do_row; a.do_head = p->do_head;
    a.dq = p->dq; a.dk = p->dk; a.dv = p->dv; a.dbias = p->dbias; a.accumulate = p->accumulate; a.err_flag = p->err_flag;
    a.units = p->B * p->Hk; a.pack = 1; a.splits = 1;
    return a;
}

// waves of 32 columns per workgroup: as many as the longest sequence fills, at most four.  fp32 rows of up to 32 columns take one wave for
// up to 256 query columns: no wave of a workgroup waits for the others' tiles, and a short sequence leaves none idle.  Measured, one wave
// against up to four: training steps of 1 024 histories up to 50, 4 heads of 16, 118 / 144 us, 512 up to 200 213 / 277, 512 up to 200,
// 8 heads of 32, 398 / 520; where few sequences leave the chip empty it loses: 64 of 200 to 256 98 / 71, 16 of 100 to 256 72 / 61.
// fp32 rows above 64 columns always take four: the registers that stage a tile (and double by half the waves) do not fit beside the
// operands'.  So do rows that are not 16-byte aligned (one variant for all of them).
int sa_waves(int64_t columns, const SaK& a, bool fp32) {
    if (!a.fast || (fp32 && a.D > 64)) return 4;
    if (fp32 && a.D <= 32 && a.pack == 1 && columns <= 256) return 1;
    return columns <= 32 ? 1 : (columns <= 64 ? 2 : 4);
}

void sa_set_grid(SaK& a, int64_t tiles, int64_t inner, int64_t together, int waves) {
    const SaGrid g = sa_grid(a.units, tiles, inner, together, waves * 64);
    a.tiles = g.tiles; a.per_unit = g.per_unit; a.rest = g.rest; a.together = g.together; a.blocks = g.blocks;
}

// Geometry of the forward.  pack: below 128 queries a workgroup of one head would leave columns empty while every head of the group
// reads the same keys, so the group's heads share the columns.  splits: workgroups are added along the keys until there are 512 (two a
// CU), 4 096 of one-wave workgroups (a SIMD holds more than one, and each has little in flight); a range keeps two tiles of 64 keys, eight
// where there were 512 workgroups already.  Measured: 4 096 against 512 for one-wave workgroups, a token for each of 128 caches of 1 000,
// fp32, 4 heads of 16, 39 / 62 us, but of 8 caches of 4 000 41 / 34, bf16, 32/8 heads of 128, 8 of 4 000 60 / 39, 128 of 4 000 373 / 352;
// eight against two tiles from 512 on, the 128 of 1 000 39 / 46, bf16 32 of 4 000 132 / 128.
static void sa_plan(const swr_seq_attention_args* p, SaK& a, int& nw) {
    a.pack = a.G > 1 && p->max_q < 128 && p->Tq * a.G < (1ll << 31) - 4096 ? a.G : 1;
    const int64_t cols = static_cast<int64_t>(p->max_q) * a.pack;
    nw = sa_waves(cols, a, p->dtype == SWR_F32);
    const int64_t tiles = std::max<int64_t>(1, (cols + nw * 32 - 1) / (nw * 32));
    // (as many as max_q says, or as the rows there are fill: with a max_q below the mean the ranges' workspace would follow the rows)
    const int64_t rows = static_cast<int64_t>(a.Hq) * a.Tq;
    const int64_t wgs = std::max(static_cast<int64_t>(a.units) * tiles * (a.G / a.pack), (rows + nw * 32 - 1) / (nw * 32));
    const int64_t key_tiles = (p->max_k + 63) / 64;
    a.splits = 1;
    const int64_t want = nw == 1 ? 4096 : 512;
    if (wgs > 0 && wgs < want && (rows + 7) / 8 <= sa_most_blocks(256)) a.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({(want + wgs - 1) / wgs, key_tiles / (wgs < 512 ? 2 : 8), 64})));
    sa_set_grid(a, tiles, static_cast<int64_t>(a.G / a.pack) * a.splits, 1, nw);
}

extern "C" size_t swr_seq_attention_fwd_workspace_bytes(const swr_seq_attention_args* p) {
    if (sa_check(p, false) != SWR_OK) return 0;
    SaK a = sa_args(p);
    int nw;
    sa_plan(p, a, nw);
    const int64_t dp = p->D <= 32 ? 32 : (p->D <= 64 ? 64 : 128);
    return a.splits == 1 ? 0 : static_cast<size_t>(a.splits) * a.Hq * a.Tq * (2 + dp) * sizeof(float);
}

template <int NP, int DP, int NW, bool FAST, bool TRAIN>
static int sa_fwd_launch(SaK& a, hipStream_t st) {
    const int lds = SaFwd<NP, DP, NW, FAST>::lds(a);
    const void* fn = reinterpret_cast<const void*>(seq_attention_fwd_kernel<NP, DP, NW, FAST, TRAIN>);
    if (lds > 64 * 1024 && !swr_raise_lds(fn, 160 * 1024)) return SWR_ERR_LAUNCH;
    hipLaunchKernelGGL((seq_attention_fwd_kernel<NP, DP, NW, FAST, TRAIN>), dim3(a.blocks), dim3(NW * 64), lds, st, a);
    if (a.splits > 1) {
        const int64_t rows = static_cast<int64_t>(a.Hq) * a.Tq;
        hipLaunchKernelGGL((seq_attention_join_kernel<NP, DP>), dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0, st, a);
    }
    return swr_launch_status();
}
template <int NP, int DP, bool TRAIN>
static int sa_fwd_nw(SaK& a, int nw, hipStream_t st) {
    if (!a.fast) return sa_fwd_launch<NP, DP, 4, false, TRAIN>(a, st);
    if constexpr (NP * DP >= 384) return sa_fwd_launch<NP, DP, 4, true, TRAIN>(a, st);
    else return nw == 1 ? sa_fwd_launch<NP, DP, 1, true, TRAIN>(a, st)
                        : (nw == 2 ? sa_fwd_launch<NP, DP, 2, true, TRAIN>(a, st) : sa_fwd_launch<NP, DP, 4, true, TRAIN>(a, st));
}
template <int NP, bool TRAIN>
static int sa_fwd_dp(SaK& a, int nw, hipStream_t st) {
    return a.D <= 32 ? sa_fwd_nw<NP, 32, TRAIN>(a, nw, st) : (a.D <= 64 ? sa_fwd_nw<NP, 64, TRAIN>(a, nw, st) : sa_fwd_nw<NP, 128, TRAIN>(a, nw, st));
}

extern "C" int swr_seq_attention_fwd(const swr_seq_attention_args* p, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = sa_check(p, false);
    if (rc != SWR_OK) return rc;
    if (p->Tq == 0) return SWR_OK;
    SaK a = sa_args(p);
    int nw;
    sa_plan(p, a, nw);
    SWR_REQUIRE(a.blocks, SWR_ERR_UNSUPPORTED);
    const size_t need = swr_seq_attention_fwd_workspace_bytes(p);
    if (need) {
        SWR_REQUIRE(workspace && workspace_bytes >= need, SWR_ERR_WORKSPACE);
        SWR_REQUIRE(swr_aligned16(workspace), SWR_ERR_ALIGN);
        a.part = static_cast<float*>(workspace);
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (p->dtype == SWR_F32) return sa_fwd_dp<3, false>(a, nw, st);
    return a.out32 ? sa_fwd_dp<1, true>(a, nw, st) : sa_fwd_dp<1, false>(a, nw, st);
}
