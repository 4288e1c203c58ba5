// The norms before and after a block fused with its gate and residual: one pass each way over the rows.
//
//   t = y rms(y) w_post (w_post NULL: t = y),   t *= sigmoid(gate) (gate NULL: 1),   z = x + scale t (y NULL: z = x)
//   u = z rms(z) w_pre (w_pre NULL: no u)       rms(a) = (mean a^2 + eps)^-1/2
//
// z is the residual stream behind the block, u the next block's normalised input.  Backward, with rows' statistics ry, rz saved and
// z recomputed from x, y, gate in fp32 (the stored z is rounded):
//   zh = z rz, a = du w_pre:   dx = dz + rz (a - zh mean(a zh)),   dw_pre = sum du zh
//   yh = y ry, dn = dx scale sigmoid(gate):   dgate = dx scale (yh w_post) s (1 - s),   dw_post = sum dn yh
//   e = dn w_post:             dy = ry (e - yh mean(e yh))
//
// HBM-bound: every operand is read once and every result written once, a row stays in registers between its two sums.  LPR lanes hold a
// row (8 elements a lane and chunk, 8 .. 64 lanes by width; above 1 024 columns the whole workgroup).  All loads of a row are issued
// before its first sum.  The weight gradients are column sums: a workgroup walks a fixed set of rows and leaves one partial per
// column, a second launch adds them in order (no atomics).
#include <algorithm>

#include "vec8.h"

#define NG_THREADS 256
#define NG_MAX_WGS 512

struct NgK {
    int64_t M;
    int N, n_wgs, accumulate;
    float eps, scale;
    const void *x, *y, *gate; int64_t ldx, ldy, ldg;
    const float *w_post, *w_pre;
    void *z, *u;                            // contiguous [M, N]
    float *ry, *rz;                         // [M], NULL: not kept
    const void *dz, *du; int64_t lddz, lddu;
    void *dx, *dy, *dg;                     // contiguous [M, N]
    float* part;                            // [n_wgs][2][N]
    float *dw_post, *dw_pre;
    int vx, vy, vg, vdz, vdu, vo, vw;
};

template <int LPR>
__device__ __forceinline__ float ng_sum(float v, float* sm) {
#pragma unroll
    for (int o = 1; o < (LPR < 64 ? LPR : 64); o <<= 1) v += __shfl_xor(v, o);
    if (LPR > 64) {
        if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (sm[0] + sm[1]) + (sm[2] + sm[3]);
        // (the next sum uses another array: no barrier protects this one's reuse inside a row; rows alternate two sets)
    }
    return v;
}

template <typename T, int MAXC>
struct NgRow {
    Raw8<T> r[MAXC];
    template <int LPR>
    __device__ __forceinline__ void load(const void* base, int64_t row, int64_t ld, int j0, int N, int vw) {
#pragma unroll
        for (int c = 0; c < MAXC; ++c) {
            const int col = (j0 + c * LPR) * 8;
            r[c] = load8(static_cast<const T*>(base) + row * ld + col, N - col, vw);
        }
    }
};
template <int LPR, int MAXC>
__device__ __forceinline__ void ng_weights(const float* w, int j0, int N, int vw, float (&o)[MAXC][8]) {
#pragma unroll
    for (int c = 0; c < MAXC; ++c) {
        const int col = (j0 + c * LPR) * 8;
        floats8(load8(w + col, w ? N - col : 0, vw), o[c]);
    }
}
template <typename T, int LPR, int MAXC>
__device__ __forceinline__ void ng_store(void* base, int64_t row, int j0, int N, int vw, const float (&x)[MAXC][8]) {
#pragma unroll
    for (int c = 0; c < MAXC; ++c) {
        const int col = (j0 + c * LPR) * 8;
        store8(static_cast<T*>(base) + row * N + col, N - col, vw, x[c]);
    }
}

template <typename T, int LPR, int MAXC>
__global__ __launch_bounds__(NG_THREADS) void norm_gate_fwd_kernel(const NgK k) {
    __shared__ float sm[2][2][4];
    constexpr int SLOTS = NG_THREADS / LPR;
    const int j0 = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const float inv_n = 1.f / static_cast<float>(k.N);
    float wp[MAXC][8], wn[MAXC][8];
    ng_weights<LPR, MAXC>(k.w_post, j0, k.N, k.vw, wp);
    ng_weights<LPR, MAXC>(k.w_pre, j0, k.N, k.vw, wn);
    int turn = 0;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * SLOTS + slot; r < k.M; r += static_cast<int64_t>(gridDim.x) * SLOTS, turn ^= 1) {
        NgRow<T, MAXC> rx, ry, rg;
        rx.template load<LPR>(k.x, r, k.ldx, j0, k.N, k.vx);
        if (k.y) ry.template load<LPR>(k.y, r, k.ldy, j0, k.N, k.vy);
        if (k.gate) rg.template load<LPR>(k.gate, r, k.ldg, j0, k.N, k.vg);
        float z[MAXC][8];
#pragma unroll
        for (int c = 0; c < MAXC; ++c) floats8(rx.r[c], z[c]);
        if (k.y) {
            float t[MAXC][8];
#pragma unroll
            for (int c = 0; c < MAXC; ++c) floats8(ry.r[c], t[c]);
            if (k.w_post) {
                float q = 0.f;
#pragma unroll
                for (int c = 0; c < MAXC; ++c)
#pragma unroll
                    for (int v = 0; v < 8; ++v) q += t[c][v] * t[c][v];
                const float s = rsqrtf(ng_sum<LPR>(q, sm[turn][0]) * inv_n + k.eps);
                if (k.ry && j0 == 0) k.ry[r] = s;
#pragma unroll
                for (int c = 0; c < MAXC; ++c)
#pragma unroll
                    for (int v = 0; v < 8; ++v) t[c][v] = t[c][v] * s * wp[c][v];
            }
            if (k.gate) {
#pragma unroll
                for (int c = 0; c < MAXC; ++c) {
                    float g[8];
                    floats8(rg.r[c], g);
#pragma unroll
                    for (int v = 0; v < 8; ++v) t[c][v] *= swr_sigmoid(g[v]);
                }
            }
#pragma unroll
            for (int c = 0; c < MAXC; ++c)
#pragma unroll
                for (int v = 0; v < 8; ++v) z[c][v] += k.scale * t[c][v];
            ng_store<T, LPR, MAXC>(k.z, r, j0, k.N, k.vo, z);
        }
        if (k.w_pre) {
            float q = 0.f;
#pragma unroll
            for (int c = 0; c < MAXC; ++c)
#pragma unroll
                for (int v = 0; v < 8; ++v) q += z[c][v] * z[c][v];
            const float s = rsqrtf(ng_sum<LPR>(q, sm[turn][1]) * inv_n + k.eps);
            if (k.rz && j0 == 0) k.rz[r] = s;
#pragma unroll
            for (int c = 0; c < MAXC; ++c)
#pragma unroll
                for (int v = 0; v < 8; ++v) z[c][v] = z[c][v] * s * wn[c][v];
            ng_store<T, LPR, MAXC>(k.u, r, j0, k.N, k.vo, z);
        }
    }
}

template <typename T, int LPR, int MAXC>
__global__ __launch_bounds__(NG_THREADS) void norm_gate_bwd_kernel(const NgK k) {
    __shared__ float sm[2][2][4];
    __shared__ float red[LPR < NG_THREADS ? NG_THREADS * 8 : 1];
    constexpr int SLOTS = NG_THREADS / LPR;
    const int j0 = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const float inv_n = 1.f / static_cast<float>(k.N);
    float wp[MAXC][8], wn[MAXC][8], ap[MAXC][8], an[MAXC][8];
    ng_weights<LPR, MAXC>(k.w_post, j0, k.N, k.vw, wp);
    ng_weights<LPR, MAXC>(k.w_pre, j0, k.N, k.vw, wn);
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
#pragma unroll
        for (int v = 0; v < 8; ++v) ap[c][v] = an[c][v] = 0.f;
    int turn = 0;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * SLOTS + slot; r < k.M; r += static_cast<int64_t>(gridDim.x) * SLOTS, turn ^= 1) {
        NgRow<T, MAXC> rx, ry, rg, rdz, rdu;
        rx.template load<LPR>(k.x, r, k.ldx, j0, k.N, k.vx);
        if (k.y) ry.template load<LPR>(k.y, r, k.ldy, j0, k.N, k.vy);
        if (k.gate) rg.template load<LPR>(k.gate, r, k.ldg, j0, k.N, k.vg);
        if (k.dz) rdz.template load<LPR>(k.dz, r, k.lddz, j0, k.N, k.vdz);
        if (k.du) rdu.template load<LPR>(k.du, r, k.lddu, j0, k.N, k.vdu);
        const float sy = k.w_post ? k.ry[r] : 1.f, sz = k.w_pre ? k.rz[r] : 0.f;
        float d[MAXC][8], y[MAXC][8], g[MAXC][8];
#pragma unroll
        for (int c = 0; c < MAXC; ++c) {
            if (k.dz) floats8(rdz.r[c], d[c]);
            if (k.y) floats8(ry.r[c], y[c]);
            if (k.gate) floats8(rg.r[c], g[c]);
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                if (!k.dz) d[c][v] = 0.f;
                y[c][v] = k.y ? y[c][v] * sy : 0.f;                        // yh (y itself without a post-norm)
                g[c][v] = k.gate ? swr_sigmoid(g[c][v]) : 1.f;
                if (!k.w_post) wp[c][v] = 1.f;
            }
        }
        if (k.du) {                                                        // (the host passes du only with w_pre)
            float z[MAXC][8], du[MAXC][8], q = 0.f;
#pragma unroll
            for (int c = 0; c < MAXC; ++c) {
                floats8(rx.r[c], z[c]);
                floats8(rdu.r[c], du[c]);
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    z[c][v] = (z[c][v] + k.scale * (y[c][v] * wp[c][v] * g[c][v])) * sz;
                    an[c][v] += du[c][v] * z[c][v];
                    du[c][v] *= wn[c][v];
                    q += du[c][v] * z[c][v];
                }
            }
            q = ng_sum<LPR>(q, sm[turn][0]) * inv_n;
#pragma unroll
            for (int c = 0; c < MAXC; ++c)
#pragma unroll
                for (int v = 0; v < 8; ++v) d[c][v] += sz * (du[c][v] - z[c][v] * q);
        }
        ng_store<T, LPR, MAXC>(k.dx, r, j0, k.N, k.vo, d);
        if (!k.y) continue;
        if (k.gate) {
            float dg[MAXC][8];
#pragma unroll
            for (int c = 0; c < MAXC; ++c)
#pragma unroll
                for (int v = 0; v < 8; ++v) dg[c][v] = d[c][v] * k.scale * (y[c][v] * wp[c][v]) * (g[c][v] * (1.f - g[c][v]));
            ng_store<T, LPR, MAXC>(k.dg, r, j0, k.N, k.vo, dg);
        }
        float q = 0.f;
#pragma unroll
        for (int c = 0; c < MAXC; ++c)
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                const float dn = d[c][v] * k.scale * g[c][v];
                ap[c][v] += dn * y[c][v];
                d[c][v] = dn * wp[c][v];
                q += d[c][v] * y[c][v];
            }
        if (k.w_post) {
            q = ng_sum<LPR>(q, sm[turn][1]) * inv_n;
#pragma unroll
            for (int c = 0; c < MAXC; ++c)
#pragma unroll
                for (int v = 0; v < 8; ++v) d[c][v] = sy * (d[c][v] - y[c][v] * q);
        }
        ng_store<T, LPR, MAXC>(k.dy, r, j0, k.N, k.vo, d);
    }
    if (!k.part) return;
    // one partial per column: the slots of the workgroup in order
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float* p = k.part + (static_cast<int64_t>(blockIdx.x) * 2 + w) * k.N;
            if (LPR == NG_THREADS) {
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    const int col = (j0 + c * LPR) * 8 + v;
                    if (col < k.N) p[col] = w ? an[c][v] : ap[c][v];
                }
            } else {
                __syncthreads();
#pragma unroll
                for (int v = 0; v < 8; ++v) red[(slot * 8 + v) * LPR + j0] = w ? an[c][v] : ap[c][v];
                __syncthreads();
                for (int i = threadIdx.x; i < LPR * 8; i += NG_THREADS) {
                    float s = 0.f;
                    for (int t = 0; t < SLOTS; ++t) s += red[(t * 8 + i / LPR) * LPR + i % LPR];
                    const int col = (i % LPR + c * LPR) * 8 + i / LPR;
                    if (col < k.N) p[col] = s;
                }
            }
        }
}

// dw[c] = sum of the workgroups' partials: 16 columns x 16 groups of partials per workgroup, groups joined in order
__global__ __launch_bounds__(256) void norm_gate_dw_kernel(const NgK k) {
    __shared__ double sm[16][17];
    const int c = threadIdx.x & 15, grp = threadIdx.x >> 4, col = blockIdx.x * 16 + c, w = blockIdx.y;
    double s = 0.;
    if (col < k.N) {
#pragma unroll 8
        for (int b = grp; b < k.n_wgs; b += 16) s += static_cast<double>(k.part[(static_cast<int64_t>(b) * 2 + w) * k.N + col]);
    }
    sm[grp][c] = s;
    __syncthreads();
    if (grp == 0 && col < k.N) {
        for (int g = 1; g < 16; ++g) s += sm[g][c];
        float* out = w ? k.dw_pre : k.dw_post;
        if (out) out[col] = static_cast<float>(k.accumulate ? out[col] + s : s);
    }
}

// ------------------------------------------------------------------------------------------------------------------- host
static int ng_lanes(int N) {
    if (N > 1024) return NG_THREADS;
    int l = 8;
    while (l < 64 && l * 8 < N) l <<= 1;
    return l;
}
static int ng_wgs(int64_t M, int N, bool backward) {
    const int64_t rows = NG_THREADS / ng_lanes(N), need = std::max<int64_t>(1, swr_ceil_div(M, rows));
    // two workgroups a CU keep HBM busy in the backward (eight operands' loads in flight) and bound the partials; the forward, with
    // fewer loads a row, takes four
    return static_cast<int>(std::min<int64_t>(need, backward ? NG_MAX_WGS : 2 * NG_MAX_WGS));
}
static int ng_check(const swr_norm_gate_args* p, bool backward) {
    SWR_REQUIRE(p && p->M >= 0 && p->N >= 1, SWR_ERR_ARG);
    SWR_REQUIRE(p->dtype == SWR_F32 || p->dtype == SWR_BF16, SWR_ERR_DTYPE);
    SWR_REQUIRE(p->N <= SWR_NORM_GATE_MAX_WIDTH, SWR_ERR_UNSUPPORTED);
    SWR_REQUIRE(p->x && (p->y || p->w_pre), SWR_ERR_ARG);
    SWR_REQUIRE(p->y || (!p->gate && !p->w_post), SWR_ERR_ARG);
    if (!backward) {
        SWR_REQUIRE((!p->y || p->z) && (!p->w_pre || p->u), SWR_ERR_ARG);
    } else {
        SWR_REQUIRE(p->dx && (!p->y || p->dy) && (!p->gate || p->dgate) && (p->dz || p->du), SWR_ERR_ARG);
        SWR_REQUIRE((!p->du || p->w_pre) && (!p->w_pre || p->rz) && (!p->w_post || p->ry), SWR_ERR_ARG);
    }
    return SWR_OK;
}
static NgK ng_args(const swr_norm_gate_args* p, bool backward) {
    NgK k{};
    const int e = p->dtype == SWR_F32 ? 4 : 2;
    k.M = p->M; k.N = p->N; k.accumulate = p->accumulate; k.eps = p->eps; k.scale = p->scale;
    k.x = p->x; k.y = p->y; k.gate = p->gate; k.ldx = p->ldx; k.ldy = p->ldy; k.ldg = p->ldg;
    k.w_post = p->w_post; k.w_pre = p->w_pre; k.z = p->z; k.u = p->u; k.ry = p->ry; k.rz = p->rz;
    k.dz = p->dz; k.du = p->du; k.lddz = p->lddz; k.lddu = p->lddu;
    k.dx = p->dx; k.dy = p->dy; k.dg = p->dgate; k.dw_post = p->dw_post; k.dw_pre = p->dw_pre;
    k.vx = swr_vec8(p->x, p->ldx, 0, p->N, e);
    k.vy = swr_vec8(p->y, p->ldy, 0, p->N, e);
    k.vg = swr_vec8(p->gate, p->ldg, 0, p->N, e);
    k.vdz = swr_vec8(p->dz, p->lddz, 0, p->N, e);
    k.vdu = swr_vec8(p->du, p->lddu, 0, p->N, e);
    k.vw = std::min(swr_vec8(p->w_post, 0, 0, p->N, 4), swr_vec8(p->w_pre, 0, 0, p->N, 4));
    k.vo = 8;
    void* outs[5] = {p->z, p->u, p->dx, p->dy, p->dgate};
    for (void* o : outs) k.vo = std::min(k.vo, swr_vec8(o, p->N, 0, p->N, e));
    k.n_wgs = ng_wgs(p->M, p->N, backward);
    return k;
}

template <typename T, int LPR, int MAXC>
static void ng_launch(const NgK& k, bool backward, hipStream_t st) {
    if (backward) hipLaunchKernelGGL((norm_gate_bwd_kernel<T, LPR, MAXC>), dim3(k.n_wgs), dim3(NG_THREADS), 0, st, k);
    else hipLaunchKernelGGL((norm_gate_fwd_kernel<T, LPR, MAXC>), dim3(k.n_wgs), dim3(NG_THREADS), 0, st, k);
}
template <typename T>
static void ng_dispatch(const NgK& k, bool backward, hipStream_t st) {
    switch (ng_lanes(k.N)) {
        case 8: return ng_launch<T, 8, 1>(k, backward, st);
        case 16: return ng_launch<T, 16, 1>(k, backward, st);
        case 32: return ng_launch<T, 32, 1>(k, backward, st);
        case 64: return k.N <= 512 ? ng_launch<T, 64, 1>(k, backward, st) : ng_launch<T, 64, 2>(k, backward, st);
        default:
            return k.N <= 2048 ? ng_launch<T, NG_THREADS, 1>(k, backward, st)
                               : (k.N <= 4096 ? ng_launch<T, NG_THREADS, 2>(k, backward, st) : ng_launch<T, NG_THREADS, 4>(k, backward, st));
    }
}

extern "C" int swr_norm_gate_fwd(const swr_norm_gate_args* p, void* stream) {
    const int rc = ng_check(p, false);
    if (rc != SWR_OK) return rc;
    if (p->M == 0) return SWR_OK;
    const NgK k = ng_args(p, false);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (p->dtype == SWR_F32) ng_dispatch<float>(k, false, st);
    else ng_dispatch<uint16_t>(k, false, st);
    return swr_launch_status();
}

extern "C" size_t swr_norm_gate_bwd_workspace_bytes(int64_t M, int N) {
    if (M < 0 || N < 1 || N > SWR_NORM_GATE_MAX_WIDTH) return 0;
    return static_cast<size_t>(ng_wgs(M, N, true)) * 2 * N * sizeof(float);
}

extern "C" int swr_norm_gate_bwd(const swr_norm_gate_args* p, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = ng_check(p, true);
    if (rc != SWR_OK) return rc;
    NgK k = ng_args(p, true);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (p->dw_post || p->dw_pre) {
        SWR_REQUIRE(workspace && workspace_bytes >= swr_norm_gate_bwd_workspace_bytes(p->M, p->N), SWR_ERR_WORKSPACE);
        SWR_REQUIRE(swr_aligned16(workspace), SWR_ERR_ALIGN);
        k.part = static_cast<float*>(workspace);
    }
    if (p->dtype == SWR_F32) ng_dispatch<float>(k, true, st);
    else ng_dispatch<uint16_t>(k, true, st);
    if (k.part) hipLaunchKernelGGL(norm_gate_dw_kernel, dim3((k.N + 15) / 16, 2), dim3(256), 0, st, k);
    return swr_launch_status();
}
