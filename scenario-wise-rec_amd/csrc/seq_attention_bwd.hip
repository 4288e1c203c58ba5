// Attention over packed sequences, backward (seq_attention_fwd.hip has the forward and its definitions).
//
//   p_ij = 2^(x_ij - lse_i) (times a second part where lse is large, sa_keep_sum),  delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij do_i,   dbias[h, t] = sum of ds over bucket t
//
// Two passes that recompute the scores, so that every sum has one owner and a fixed order (no atomics): a workgroup of query columns
// walks the keys and holds dq (it also makes delta and the bias gradient), a workgroup of key columns walks the queries of all heads
// of its group and holds dk and dv.  7 products instead of 5, against the fp32 read-modify-write of dq for every key tile.
//
// Bias gradient: a 32 x 32 block of ds has 63 distances.  Its wave writes it to LDS skewed, one row per distance, lane t adds up row t
// and owns that entry of the wave's per-distance sums.  Blocks wholly beyond the table's reach add their sum to one register.
#include <algorithm>

#include "seq_attention.h"

int sa_check(const swr_seq_attention_args* p, bool backward);
SaK sa_args(const swr_seq_attention_args* p);
int sa_waves(int64_t columns, const SaK& a, bool fp32);
void sa_set_grid(SaK& a, int64_t tiles, int64_t inner, int64_t together, int waves);

// waves per SIMD the registers are bounded for (512 / waves each): as many as spill nothing -- one more spills in every kernel that has
// not got its registers anyway, but in those of one or two waves at DP = 128, bf16, which take one (steps of 512 histories, 8 heads, one
// against two: up to 60 rows 281 / 241 us, up to 30 rows 200 / 204)
#define SA_WAVES_DQ(NP, DP, NW, FAST) ((NP) * (DP) >= 192 || ((DP) == 128 && ((NW) < 4 || !(FAST))) ? 1 : 2)
#define SA_WAVES_DKV(NP, DP, NW, FAST) ((NP) * (DP) >= 192 || ((DP) == 128 && ((NW) < 4 || !(FAST))) ? 1 : ((NP) * (DP) == 32 ? 3 : 2))
#define SA_PITCH 36                            // a wave's skewed 32 x 32 block: one row per distance (63, and one of zeros), 32 keys
#define SA_SKEW (64 * SA_PITCH)

// dq: DMA and buffers as in the forward; 32 keys a step at DP = 128, so that two workgroups fit a CU's LDS beside the skew blocks
template <int NP, int DP, int NW, bool FAST>
struct SaDq {
    static constexpr bool DMA = FAST && NP == 1;
    static constexpr int KT = (NW == 1 || DP == 128) ? 32 : 64, NBUF = DMA ? 2 : 1;
    static constexpr int TILE = NP * KT * DP * 2;
    static int lds(const SaK& a) { return NBUF * (2 * TILE + KT) + (max(a.row, SA_FLAT) + (a.bias_part ? NW * (SA_SKEW + a.n_dist) + a.n_dist + 2 * a.n_buckets : 0)) * 4; }
};
template <int NP, int DP, int NW, bool FAST>
struct SaDkv {
    static constexpr bool DMA = FAST && NP == 1, LATE = NP * DP >= 384;       // LATE: splits at use, nothing staged ahead (registers)
    static constexpr int RT = (NW == 1 || DP == 128) ? 32 : 64, NBUF = DMA ? 2 : 1;
    static constexpr bool VL = NP == 1 && DP == 128;           // the wave's values stay in LDS: with them in registers one wave fits a SIMD
    static constexpr int TILE = NP * RT * DP * 2, VTILE = VL ? NW * 32 * DP * 2 : 0;
    static int lds(const SaK& a) { return NBUF * (2 * TILE + 2 * RT * 4) + VTILE + max(a.G * a.row, SA_FLAT) * 4; }
};

template <int NP, int DP, int NW, bool FAST>
__global__ __launch_bounds__(NW * 64, SA_WAVES_DQ(NP, DP, NW, FAST)) void seq_attention_dq_kernel(const SaK a) {
    typedef SaDq<NP, DP, NW, FAST> Cfg;
    constexpr int KT = Cfg::KT, KB = KT / 32, NT = NW * 64, QT = NW * 32, TILE = Cfg::TILE;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    uint8_t* km0 = reinterpret_cast<uint8_t*>(smem) + Cfg::NBUF * 2 * TILE;
    float* bt = reinterpret_cast<float*>(km0 + Cfg::NBUF * KT);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5;
    SaLane<NP, DP, KT> ln(lane);
    float* skew = bt + a.row + wave * SA_SKEW;         // (a.row is a multiple of 4)
    float* acc0 = bt + a.row + NW * SA_SKEW;
    float* acc = acc0 + wave * a.n_dist;
    int *bucket = reinterpret_cast<int*>(acc0 + NW * a.n_dist), *range = bucket + a.n_dist;

    int within;
    const int unit = sa_unit(blockIdx.x, a.per_unit, a.together, within);
    if (unit >= a.units) {                     // rows of no sequence
        if (unit >= a.units + a.rest) return;
        const int part = (unit - a.units) * a.per_unit + within, parts = a.rest * a.per_unit;
        const int64_t end0 = sa_clamp(a.cu_q[0], 0, a.Tq), beg1 = sa_clamp(a.cu_q[a.B], end0, a.Tq), row = static_cast<int64_t>(a.Hq) * a.D;
        sa_zero_rows(a.dq, NP == 3 ? 4 : 2, 0, end0, row, NT, part, parts);
        sa_zero_rows(a.dq, NP == 3 ? 4 : 2, beg1, a.Tq, row, NT, part, parts);
        return;
    }
    const int b = unit / a.Hk, hk = unit % a.Hk, g = within % a.G, h = hk * a.G + g, tile0 = a.tiles - 1 - within / a.G;
    const SaSeq sq = sa_seq(a, b);
    float beyond_hi = 0.f, beyond_lo = 0.f;    // ds at distances >= reach / <= -reach (this lane's share)

    for (int64_t tile = tile0; tile * QT < sq.q_span; tile += a.tiles) {
        const int first = static_cast<int>(tile * QT), wfirst = first + wave * 32, tok = wfirst + (lane & 31);
        const bool exists = tok < sq.q_span, live = tok < sq.lq;
        const int qpos = tok + sq.shift, wlast = min(wfirst + 31, sq.lq - 1), blast = min(first + QT - 1, sq.lq - 1);
        int kend = a.causal ? min(sq.lk, blast + sq.shift + 1) : sq.lk;
        if (first >= sq.lq || kend < 0) kend = 0;
        const int ntile = (kend + KT - 1) / KT;

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
        // the first tile's loads go out before anything waits (a tile before this one has been read: barrier first)
        if (tile != tile0) __syncthreads();
        if (ntile > 0) fetch(0, 0);
        const SaArgs n = sa_again();
        const int64_t row = sq.q0 + (exists ? tok : 0), at = static_cast<int64_t>(h) * n->Tq + row;
        bf16x8 Q[DP / 16][NP], dO[DP / 16][NP];
        sa_row_frags<NP, DP, FAST>(n->q, row * n->q_row + static_cast<int64_t>(h) * n->q_head, live, a.D, n->vq, lane, Q);
        // fp32: odd rows enter the product do . v with their signs flipped and leave it flipped back.  The matrix pipe's sums are rounded
        // down (3e-8 on average per row of 16 columns of N(0, 1) values): that drifts into the bias gradient, whose other terms cancel in
        // every row, and with alternating signs it cancels between rows (1 024 histories up to 50: off by 1.2e-6 / 1.7e-7 of its norm,
        // 512 up to 200 1.5e-6 / 2.4e-7, the same times).  On bf16 tensors the two terms of the forward's probabilities leave 1.5e-6 either
        // way, and at 128 columns the flips cost 1 %.
        const int odd = static_cast<int>(sq.q0 + wfirst) & 1;              // (of the row of lane 0: a column's row is odd where lane ^ odd is)
        float delta = 0.f;
        const int hi8 = sa_here(8 * hi);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int col = 16 * s + hi8;
            const SaRaw<NP> x = sa_row8<NP, FAST>(n->dout, row * n->do_row + static_cast<int64_t>(h) * n->do_head, col, live, a.D, n->vdo);
            const SaRaw<3> y = sa_row8<3, FAST>(n->out32, (row * n->Hq + h) * a.D, col, live, a.D, n->vo);
            float fx[8], fy[8];
            floats8(x, fx);
            floats8(y, fy);
#pragma unroll
            for (int j = 0; j < 8; ++j) delta += fx[j] * fy[j];
            if constexpr (NP == 3) {
#pragma unroll
                for (int j = 0; j < 8; ++j) fx[j] = (lane ^ odd) & 1 ? -fx[j] : fx[j];
                sa_split8(fx, dO[s]);
            } else {
                sa_planes(x, dO[s]);
            }
        }
        delta += __shfl_xor(delta, 32);
        const float lse = live ? n->lse[at] : INFINITY;
        const bool parts = __any(sa_parts(lse));       // (then the scores are written out as the forward rounded them, also under one bias)
        if (tile == tile0) {
            sa_bias_rows<NT>(a, h, 1, bt);
            if (a.row == 0 && threadIdx.x < SA_FLAT) bt[threadIdx.x] = 0.f;
            if (a.bias_part) {
                for (int i = lane; i < SA_SKEW / 4; i += 64) reinterpret_cast<float4*>(skew)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int i = lane; i < a.n_dist; i += 64) acc[i] = 0.f;
                for (int i = threadIdx.x; i < a.n_dist; i += NT) bucket[i] = sa_bucket(a, i);
            }
        }
        if (exists && hi == 0) a.delta[at] = delta;
        f32x16 dQ[DP / 32];
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) dQ[db] = sa_zero16();

        for (int t = 0; t < ntile; ++t) {
            const int buf = Cfg::DMA ? t & 1 : 0;
            const sa_lds kt = (sa_lds)smem + buf * 2 * TILE, vt = kt + TILE;
            const uint8_t* km = km0 + buf * KT;
            if (Cfg::DMA) {
                if (a.key_mask && threadIdx.x < KT) km0[buf * KT + threadIdx.x] = mk;
                sa_dma_wait();
                __syncthreads();
            } else {
                if (t > 0) __syncthreads();
                sk.store(kt);
                sv.store(vt);
                if (a.key_mask && threadIdx.x < KT) km0[threadIdx.x] = mk;
                __syncthreads();
            }
            if (t + 1 < ntile) fetch(t + 1, buf ^ 1);
#pragma unroll 1
            for (int kb = 0; kb < KB; ++kb) {
                const int k0 = t * KT + kb * 32;
                if (wfirst > wlast || k0 >= sq.lk || (a.causal && k0 > wlast + sq.shift)) continue;      // (whole waves)
                ln.fresh();
                f32x16 S = sa_zero16(), dP = sa_zero16();
                {
                    bf16x8 A[2][2][NP];
                    sa_ahead<DP / 16, true>(
                        [&](int buf, int s) {
                            ln.rows(kt, kb, s, A[buf][0]);
                            ln.rows(vt, kb, s, A[buf][1]);
                        },
                        [&](int buf, int s) {
                            S = sa_mma(A[buf][0], Q[s], S);
                            dP = sa_mma(A[buf][1], dO[s], dP);
                        });
                }
                // (the second product's first operands come in under the exponentials)
                bf16x8 T[2][DP / 32][NP];
                auto cols = [&](int buf, int ks) {
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) ln.cols(kt, kb * 2 + ks, db, T[buf][db]);
                };
                cols(0, 0);
                const int near_d = wfirst + sq.shift - (k0 + 31), far_d = wlast + sq.shift - k0;
                const SaSpan sp = sa_span(a, near_d, far_d);
                const float sign = NP == 3 ? __uint_as_float(0x3f800000u | (static_cast<uint32_t>(sa_here(threadIdx.x) ^ odd) << 31)) : 1.f;
                if (sp.apart && !parts) {
                    const float add = (a.row ? bt[sp.entry] : 0.f) - lse;
#pragma unroll
                    for (int i = 0; i < 16; ++i) S[i] = __builtin_amdgcn_exp2f(S[i] * a.c + add) * (dP[i] * sign - delta);
                } else {
                    const float* be = bt + (sp.apart ? sa_flat_entry(a, sp) : sa_entry(a, qpos - k0 - 4 * hi - 27));
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float p = __builtin_amdgcn_exp2f((S[i] * a.c + be[27 - 8 * (i >> 2) - (i & 3)]) - lse);
                        S[i] = p * (dP[i] * sign - delta);
                    }
                    if (parts) {
                        const SaArgs n = sa_again();
                        const float part = n->lse[static_cast<int64_t>(n->Hq + h) * n->Tq + row];
#pragma unroll
                        for (int i = 0; i < 16; ++i) S[i] *= part;
                    }
                }
                if (!a.causal && k0 + 32 > sq.lk) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) S[i] = k0 + 4 * hi + 8 * (i >> 2) + (i & 3) < sq.lk ? S[i] : 0.f;
                }
                if (a.key_mask) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) S[i] = sa_masked(km + kb * 32 + 4 * hi, i) ? 0.f : S[i];
                }
                float total = 0.f;
                if (a.bias_part && sp.apart) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) total += S[i];
                }
                if (a.bias_part) {
                    if (near_d >= a.reach) {
                        beyond_hi += total;
                    } else if (sp.apart) {
                        beyond_lo += total;
                    } else {
                        float* to = skew + (lane & 31) * SA_PITCH + 31 * SA_PITCH - (SA_PITCH - 1) * (4 * hi + 27);      // (lane, key 4 hi + 27)
#pragma unroll
                        for (int i = 0; i < 16; ++i) to[(SA_PITCH - 1) * (27 - 8 * (i >> 2) - (i & 3))] = S[i];
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        float sum = 0.f;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float4 x = *reinterpret_cast<const float4*>(skew + lane * SA_PITCH + 4 * k);
                            sum += (x.x + x.y) + (x.z + x.w);
                        }
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        // row 31 of the skewed block = the distance of query wfirst to key k0
                        const int dist = wfirst + sq.shift - k0 + lane - 31;
                        if (dist >= a.reach) beyond_hi += sum;
                        else if (dist <= -a.reach || (a.causal && dist < 0)) beyond_lo += sum;         // (causal: zeros)
                        else acc[a.causal ? dist : dist + a.reach] += sum;
                    }
                }
                bf16x8 P[2][NP];
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    float f[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = S[8 * ks + j];
                    sa_planes_f(f, P[ks]);
                }
                sa_ahead<2, false>(cols, [&](int buf, int ks) {
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) dQ[db] = sa_mma(T[buf][db], P[ks], dQ[db]);
                });
            }
        }
        if (exists) {
            const int hi4 = sa_here(4 * hi);
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float x[4] = {dQ[db][i] * a.scale, dQ[db][i + 1] * a.scale, dQ[db][i + 2] * a.scale, dQ[db][i + 3] * a.scale};
                    sa_store4<NP>(a.dq, (row * a.Hq + h) * a.D, db * 32 + 2 * i + hi4, a.D, x);
                }
        }
    }
    if (a.bias_part) {
        if (tile0 * QT >= sq.q_span) {         // nothing of the sequence is this workgroup's
            for (int t = threadIdx.x; t < a.n_buckets; t += NT)
                a.bias_part[(static_cast<int64_t>(h) * a.n_buckets + t) * a.bias_slots + static_cast<int64_t>(b) * a.tiles + tile0] = 0.f;
            return;
        }
        // entries of the waves -> one per distance -> buckets, all in fixed order
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { beyond_hi += __shfl_xor(beyond_hi, o); beyond_lo += __shfl_xor(beyond_lo, o); }
        if (lane == 0) {
            acc[a.n_dist - 1] += beyond_hi;
            if (!a.causal) acc[0] += beyond_lo;
        }
        for (int t = threadIdx.x; t < a.n_buckets; t += NT) { range[2 * t] = a.n_dist; range[2 * t + 1] = 0; }
        __syncthreads();
        for (int i = threadIdx.x; i < a.n_dist; i += NT) {
            float s = acc0[i];
#pragma unroll
            for (int w = 1; w < NW; ++w) s += acc0[w * a.n_dist + i];
            acc0[i] = s;
            atomicMin(&range[2 * bucket[i]], i);                   // first entry of a bucket and the one behind its last
            atomicMax(&range[2 * bucket[i] + 1], i + 1);
        }
        __syncthreads();
        for (int t = threadIdx.x; t < a.n_buckets; t += NT) {
            float s = 0.f;
            for (int i = range[2 * t]; i < range[2 * t + 1]; ++i) s += bucket[i] == t ? acc0[i] : 0.f;
            a.bias_part[(static_cast<int64_t>(h) * a.n_buckets + t) * a.bias_slots + static_cast<int64_t>(b) * a.tiles + tile0] = s;
        }
    }
}

// dbias[h, t] = sum of its partials: one workgroup each, strided per thread, then a fixed tree
__global__ __launch_bounds__(256) void seq_attention_dbias_kernel(const SaK a) {
    __shared__ double sm[4];
    const float* p = a.bias_part + static_cast<int64_t>(blockIdx.x) * a.bias_slots;
    double s = 0.;
    for (int i = threadIdx.x; i < a.bias_slots; i += 256) s += static_cast<double>(p[i]);
    s = swr_block_sum_f64<256>(s, sm);
    if (threadIdx.x == 0) a.dbias[blockIdx.x] = static_cast<float>(a.accumulate ? a.dbias[blockIdx.x] + s : s);
}

template <int NP, int DP, int NW, bool FAST>
__global__ __launch_bounds__(NW * 64, SA_WAVES_DKV(NP, DP, NW, FAST)) void seq_attention_dkv_kernel(const SaK a) {
    typedef SaDkv<NP, DP, NW, FAST> Cfg;
    constexpr int RT = Cfg::RT, RB = RT / 32, NT = NW * 64, KT = NW * 32, TILE = Cfg::TILE;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const sa_lds vt = (sa_lds)smem + Cfg::NBUF * 2 * TILE;
    float* rows0 = reinterpret_cast<float*>(smem + Cfg::NBUF * 2 * TILE + Cfg::VTILE);      // per buffer: lse of the rows, then delta
    float* tables = rows0 + Cfg::NBUF * 2 * RT;                                // the group's bias rows
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5;
    SaLane<NP, DP, RT> ln(lane);

    int within;
    const int unit = sa_unit(blockIdx.x, a.per_unit, a.together, within);
    if (unit >= a.units) {                     // rows of no sequence
        if (unit >= a.units + a.rest) return;
        const int part = (unit - a.units) * a.per_unit + within, parts = a.rest * a.per_unit;
        const int64_t end0 = sa_clamp(a.cu_k[0], 0, a.Tk), beg1 = sa_clamp(a.cu_k[a.B], end0, a.Tk), row = static_cast<int64_t>(a.Hk) * a.D;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            sa_zero_rows(w ? a.dv : a.dk, NP == 3 ? 4 : 2, 0, end0, row, NT, part, parts);
            sa_zero_rows(w ? a.dv : a.dk, NP == 3 ? 4 : 2, beg1, a.Tk, row, NT, part, parts);
        }
        return;
    }
    const int b = unit / a.Hk, hk = unit % a.Hk;
    const SaSeq sq = sa_seq(a, b);
    for (int64_t tile = within; tile * KT < sq.k_span; tile += a.tiles) {
        const int first = static_cast<int>(tile * KT), wfirst = first + wave * 32, key = wfirst + (lane & 31);
        const bool exists = key < sq.k_span;
        const int64_t row = sq.k0 + (exists ? key : 0);
        const bool live = key < sq.lk && (!a.key_mask || a.key_mask[row] != 0);
        const int wlast = min(wfirst + 31, sq.lk - 1);
        f32x16 dK[DP / 32], dV[DP / 32];
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) { dK[db] = sa_zero16(); dV[db] = sa_zero16(); }

        // queries that see this tile: all of them, or (causal) those at or behind its first key
        const int q_first = a.causal ? max(0, first - sq.shift) : 0;
        const int r_begin = q_first / RT, r_end = first < sq.lk ? (sq.lq + RT - 1) / RT : 0, n_r = max(0, r_end - r_begin);
        const int steps = n_r * a.G;
        SaStage<NP, DP, RT, NT, FAST> sQ, sD;
        float ld_l = 0.f, ld_d = 0.f;
        int next_g = 0, next_r = 0;                    // head of the group and row tile of the step to fetch next
        auto fetch = [&](int buf) {
            const int h = hk * a.G + next_g, q0 = (r_begin + next_r) * RT;
            if (++next_r == n_r) { next_r = 0; ++next_g; }
            if (Cfg::DMA) {
                const sa_lds to = (sa_lds)smem + buf * 2 * TILE;
                SaDma<DP, RT, NT>::copy(to, a.q, sq.q0, q0, sq.lq, a.q_row, static_cast<int64_t>(h) * a.q_head, a.D, nullptr);
                SaDma<DP, RT, NT>::copy(to + TILE, a.dout, sq.q0, q0, sq.lq, a.do_row, static_cast<int64_t>(h) * a.do_head, a.D, nullptr);
            } else {
                sQ.load(a.q, sq.q0, q0, sq.lq, a.q_row, static_cast<int64_t>(h) * a.q_head, a.D, a.vq, nullptr);
                sD.load(a.dout, sq.q0, q0, sq.lq, a.do_row, static_cast<int64_t>(h) * a.do_head, a.D, a.vdo, nullptr);
            }
            if (threadIdx.x < RT) {
                const int tok = q0 + threadIdx.x;
                const int64_t at = static_cast<int64_t>(h) * a.Tq + sq.q0 + tok;
                ld_l = tok < sq.lq ? a.lse[at] : INFINITY;
                ld_d = tok < sq.lq ? a.delta[at] : 0.f;
            }
        };
        if (tile != within) __syncthreads();       // (a tile before this one has been read)
        if (steps > 0) {
            if constexpr (Cfg::VL) {
                if constexpr (Cfg::DMA) {
                    SaDma<DP, KT, NT>::copy(vt, a.v, sq.k0, first, sq.lk, a.v_row, hk * a.v_head, a.D, a.key_mask);
                } else {
                    SaStage<NP, DP, KT, NT, FAST> sv;
                    sv.load(a.v, sq.k0, first, sq.lk, a.v_row, hk * a.v_head, a.D, a.vv, a.key_mask);
                    sv.store(vt);
                }
            }
            if (!Cfg::LATE) fetch(0);
        }
        const SaArgs kv = sa_again();
        SaRows<NP, DP, FAST, Cfg::LATE> K, V;
        K.load(kv->k, row * kv->k_row + hk * kv->k_head, live, kv->D, kv->vk, lane);
        if (!Cfg::VL) V.load(kv->v, row * kv->v_row + hk * kv->v_head, live, kv->D, kv->vv, lane);
        if (tile == within) {
            sa_bias_rows<NT>(a, hk * a.G, a.G, tables);
            if (a.row == 0 && threadIdx.x < SA_FLAT) tables[threadIdx.x] = 0.f;
        }
        int g = 0, r = 0;
        for (int step = 0; step < steps; ++step) {
            const int q0 = (r_begin + r) * RT, buf = Cfg::DMA ? step & 1 : 0;
            const sa_lds qt = (sa_lds)smem + buf * 2 * TILE, dt = qt + TILE;
            float *lse_s = rows0 + buf * 2 * RT, *delta_s = lse_s + RT;
            const float* bt = tables + g * a.row;
            const int h = hk * a.G + g;
            if (++r == n_r) { r = 0; ++g; }
            if (Cfg::LATE) fetch(0);
            if (!Cfg::DMA) {
                if (step > 0) __syncthreads();
                sQ.store(qt);
                sD.store(dt);
            }
            if (threadIdx.x < RT) { lse_s[threadIdx.x] = ld_l; delta_s[threadIdx.x] = ld_d; }
            if (Cfg::DMA) sa_dma_wait();
            __syncthreads();
            if (!Cfg::LATE && step + 1 < steps) fetch(buf ^ 1);
            if (wfirst > wlast) continue;
#pragma unroll 1
            for (int rb = 0; rb < RB; ++rb) {
                const int r0 = q0 + rb * 32, rlast = min(r0 + 31, sq.lq - 1);
                if (r0 >= sq.lq || (a.causal && rlast + sq.shift < wfirst)) continue;
                ln.fresh();
                f32x16 S = sa_zero16(), dP = sa_zero16();
                {
                    bf16x8 A[2][2][NP];
                    sa_ahead<DP / 16, true>(
                        [&](int buf, int s) {
                            ln.rows(qt, rb, s, A[buf][0]);
                            ln.rows(dt, rb, s, A[buf][1]);
                        },
                        [&](int buf, int s) {
                            bf16x8 B[NP];
                            K.get(s, B);
                            S = sa_mma(A[buf][0], B, S);
                            if constexpr (Cfg::VL) ln.rows(vt + wave * (32 * DP * 2), 0, s, B);
                            else V.get(s, B);
                            dP = sa_mma(A[buf][1], B, dP);
                        });
                }
                const float first = lse_s[rb * 32 + (sa_here(lane) & 31)];
                // dv and dk take the rows in two halves each: group 2 ks + (0 dv, 1 dk); the first operands come in under the exponentials
                bf16x8 T[2][DP / 32][NP];
                auto cols = [&](int buf, int i) {
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) ln.cols(i & 1 ? qt : dt, rb * 2 + (i >> 1), db, T[buf][db]);
                };
                cols(0, 0);
                // (columns that are no key in use compute something finite or not: columns do not mix, theirs is not stored.  Rows
                // behind the last query have lse = +inf, p = 0)
                const SaSpan sp = sa_span(a, r0 + sq.shift - wlast, rlast + sq.shift - wfirst);
                const float *lr = lse_s + rb * 32 + ((sa_here(threadIdx.x) >> 3) & 4), *dr = lr + RT;
                const bool parts = __any(sa_parts(first));             // (as in the query pass)
                if (sp.apart && !parts) {
                    const float add = a.row ? bt[sp.entry] : 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) S[i] = __builtin_amdgcn_exp2f(S[i] * a.c + (add - lr[8 * (i >> 2) + (i & 3)]));
                } else {
                    const int l = sa_here(threadIdx.x) & 63;
                    const float* be = bt + (sp.apart ? sa_flat_entry(a, sp) : sa_entry(a, r0 + 4 * (l >> 5) + sq.shift - wfirst - (l & 31)));
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        S[i] = __builtin_amdgcn_exp2f((S[i] * a.c + be[8 * (i >> 2) + (i & 3)]) - lr[8 * (i >> 2) + (i & 3)]);
                    if (parts) {
                        const SaArgs n = sa_again();
                        const float* second = n->lse + static_cast<int64_t>(n->Hq + h) * n->Tq + sq.q0;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            // (one after the other: this rare path takes no registers from the others)
                            float p = S[i] * second[min(r0 + ((sa_here(threadIdx.x) >> 3) & 4) + 8 * (i >> 2) + (i & 3), sq.lq - 1)];
                            asm volatile("" : "+v"(p) : : "memory");
                            S[i] = p;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) dP[i] = S[i] * (dP[i] - dr[8 * (i >> 2) + (i & 3)]);
                sa_ahead<4, false>(cols, [&](int buf, int i) {
                    float f[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = i & 1 ? dP[8 * (i >> 1) + j] : S[8 * (i >> 1) + j];
                    bf16x8 P[NP];
                    sa_planes_f(f, P);
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) {
                        if (i & 1) dK[db] = sa_mma(T[buf][db], P, dK[db]);
                        else dV[db] = sa_mma(T[buf][db], P, dV[db]);
                    }
                });
            }
        }
        if (exists) {
            const int64_t o = ((sq.k0 + wfirst + (sa_here(threadIdx.x) & 31)) * a.Hk + hk) * a.D;       // (places made anew: no registers spill)
            const int hi4 = sa_here(4 * hi);
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const int d = db * 32 + 2 * i + hi4;
                    float x[4], y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[j] = live ? dK[db][i + j] * a.scale : 0.f;
                        y[j] = live ? dV[db][i + j] : 0.f;
                    }
                    sa_store4<NP>(a.dk, o, d, a.D, x);
                    sa_store4<NP>(a.dv, o, d, a.D, y);
                }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------- host
struct SaBwdPlan {
    SaK q, kv;
    int nw_q, nw_kv;
    size_t delta, bytes;
    bool fits;
};
static SaBwdPlan sa_bwd_plan(const swr_seq_attention_args* p) {
    SaBwdPlan pl{};
    pl.q = pl.kv = sa_args(p);
    pl.nw_q = sa_waves(p->max_q, pl.q, p->dtype == SWR_F32);
    pl.nw_kv = sa_waves(p->max_k, pl.kv, p->dtype == SWR_F32);
    sa_set_grid(pl.q, std::max<int64_t>(1, swr_ceil_div(p->max_q, pl.nw_q * 32)), pl.q.G, 0, pl.nw_q);
    sa_set_grid(pl.kv, std::max<int64_t>(1, swr_ceil_div(p->max_k, pl.nw_kv * 32)), 1, 0, pl.nw_kv);
    pl.fits = pl.q.blocks && pl.kv.blocks && static_cast<int64_t>(p->Hq) * p->n_buckets <= sa_most_blocks(256);
    const int64_t slots = static_cast<int64_t>(p->B) * pl.q.tiles;
    pl.q.bias_slots = static_cast<int>(slots);
    pl.delta = static_cast<size_t>(p->Hq) * p->Tq * sizeof(float);
    pl.bytes = pl.delta + (p->dbias && p->n_dist ? static_cast<size_t>(p->Hq) * p->n_buckets * slots * sizeof(float) : 0) + 256;
    return pl;
}

extern "C" size_t swr_seq_attention_bwd_workspace_bytes(const swr_seq_attention_args* p) {
    return sa_check(p, true) == SWR_OK ? sa_bwd_plan(p).bytes : 0;
}

template <int NP, int DP, int NW, bool FAST>
static int sa_dq_launch(SaK& a, hipStream_t st) {
    const int lds = SaDq<NP, DP, NW, FAST>::lds(a);
    SWR_REQUIRE(lds <= 160 * 1024, SWR_ERR_UNSUPPORTED);
    if (lds > 64 * 1024 && !swr_raise_lds(reinterpret_cast<const void*>(seq_attention_dq_kernel<NP, DP, NW, FAST>), 160 * 1024)) return SWR_ERR_LAUNCH;
    hipLaunchKernelGGL((seq_attention_dq_kernel<NP, DP, NW, FAST>), dim3(a.blocks), dim3(NW * 64), lds, st, a);
    return SWR_OK;
}
template <int NP, int DP, int NW, bool FAST>
static int sa_dkv_launch(SaK& a, hipStream_t st) {
    const int lds = SaDkv<NP, DP, NW, FAST>::lds(a);
    SWR_REQUIRE(lds <= 160 * 1024, SWR_ERR_UNSUPPORTED);
    if (lds > 64 * 1024 && !swr_raise_lds(reinterpret_cast<const void*>(seq_attention_dkv_kernel<NP, DP, NW, FAST>), 160 * 1024)) return SWR_ERR_LAUNCH;
    hipLaunchKernelGGL((seq_attention_dkv_kernel<NP, DP, NW, FAST>), dim3(a.blocks), dim3(NW * 64), lds, st, a);
    return SWR_OK;
}
template <int NP, int DP>
static int sa_bwd_dp(SaBwdPlan& pl, hipStream_t st) {
    SaK &q = pl.q, &kv = pl.kv;
    if (!q.fast) {
        const int rc = sa_dq_launch<NP, DP, 4, false>(q, st);
        return rc != SWR_OK ? rc : sa_dkv_launch<NP, DP, 4, false>(kv, st);
    }
    if constexpr (NP * DP >= 384) {
        const int rc = sa_dq_launch<NP, DP, 4, true>(q, st);
        return rc != SWR_OK ? rc : sa_dkv_launch<NP, DP, 4, true>(kv, st);
    } else {
        const int rc = pl.nw_q == 1 ? sa_dq_launch<NP, DP, 1, true>(q, st)
                                    : (pl.nw_q == 2 ? sa_dq_launch<NP, DP, 2, true>(q, st) : sa_dq_launch<NP, DP, 4, true>(q, st));
        if (rc != SWR_OK) return rc;
        return pl.nw_kv == 1 ? sa_dkv_launch<NP, DP, 1, true>(kv, st)
                             : (pl.nw_kv == 2 ? sa_dkv_launch<NP, DP, 2, true>(kv, st) : sa_dkv_launch<NP, DP, 4, true>(kv, st));
    }
}

extern "C" int swr_seq_attention_bwd(const swr_seq_attention_args* p, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = sa_check(p, true);
    if (rc != SWR_OK) return rc;
    SaBwdPlan pl = sa_bwd_plan(p);
    SWR_REQUIRE(pl.fits, SWR_ERR_UNSUPPORTED);
    SWR_REQUIRE(workspace && workspace_bytes >= pl.bytes, SWR_ERR_WORKSPACE);
    SWR_REQUIRE(swr_aligned16(workspace), SWR_ERR_ALIGN);
    SaK &q = pl.q, &kv = pl.kv;
    q.delta = kv.delta = static_cast<float*>(workspace);
    if (p->dbias && p->n_dist) q.bias_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + (pl.delta + 255) / 256 * 256);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int r = p->dtype == SWR_F32 ? (p->D <= 32 ? sa_bwd_dp<3, 32>(pl, st) : (p->D <= 64 ? sa_bwd_dp<3, 64>(pl, st) : sa_bwd_dp<3, 128>(pl, st)))
                                      : (p->D <= 32 ? sa_bwd_dp<1, 32>(pl, st) : (p->D <= 64 ? sa_bwd_dp<1, 64>(pl, st) : sa_bwd_dp<1, 128>(pl, st)));
    if (r != SWR_OK) return r;
    if (q.bias_part) hipLaunchKernelGGL(seq_attention_dbias_kernel, dim3(static_cast<unsigned>(p->Hq) * p->n_buckets), dim3(256), 0, st, q);
    return swr_launch_status();
}
