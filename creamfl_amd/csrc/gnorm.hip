// gnorm.hip -- group normalisation (+ residual add) (+ activation) of channels_last feature maps, forward and backward.
//
//   mu = sum x / M, v = sum (x - mu)^2 / M over a group's M = (C / G) H W values of one sample, r = (v + eps)^-1/2, xh = (x - mu) r
//   z = xh gamma_c + beta_c (+ residual),  y = act(z),  act in {identity, relu, silu}
//   backward: dz = dy act'(z) (= the residual's gradient),  dbeta_c = sum dz,  dgamma_c = sum dz xh  over all samples,
//             g = dz gamma_c,  s1 = sum_group g / M,  s2 = sum_group g xh / M,  dx = r (g - s1 - xh s2)
//
// Where it sits: the normalisation of the image trunks (src/networks/models/image_encoder.py:27-36, src/networks/resnet_client.py:60-98
// use BatchNorm there), for federations whose clients' batch statistics do not average.
// HBM-bound.  A sample is a row-major [H W, C] matrix; a thread owns 8 consecutive channels of its rows (one 16-byte access in bf16).
// Statistics: a thread keeps its RPT rows in registers and forms mean and squared deviations of what it holds in two passes; partial
// (mean, M2) pairs are then merged by sum n (mean - mu)^2, so that a mean much larger than the deviation costs no digits (a running
// sum of squares would).  Everything is summed in 32 bits and in a fixed order: two runs give the same bits.
#include "common.h"
#include "colmap.h"

namespace {

constexpr int GN_T = 256;          // threads of a workgroup
constexpr int GN_RPT = 8;          // rows a thread holds
constexpr int GN_MAXC = 2048;      // channels: one row is at most one access per thread

enum { GN_NONE = 0, GN_RELU = 1, GN_SILU = 2 };

// thread -> (first channel, row phase): C / 8 threads per row, `rpp` rows per pass; threads behind the last whole row idle
struct GMap { int tpr, rpp, c0, rsub; bool active; };
__device__ __forceinline__ GMap gn_map(int C) {
    GMap m;
    m.tpr = C >> 3;
    m.rpp = GN_T / m.tpr;
    m.rsub = threadIdx.x / m.tpr;
    m.c0 = (threadIdx.x % m.tpr) * 8;
    m.active = m.rsub < m.rpp;
    return m;
}

template <int ACT> __device__ __forceinline__ float gn_act(float z) {
    if (ACT == GN_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
    if (ACT == GN_SILU) return z / (1.f + __expf(-z));
    return z;
}
template <int ACT> __device__ __forceinline__ float gn_act_grad(float z) {
    if (ACT == GN_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == GN_SILU) { const float s = 1.f / (1.f + __expf(-z)); return s * (1.f + z * (1.f - s)); }
    return 1.f;
}

// ---- forward, pass 1: (mean, M2) of every group over a chunk of rows.  grid = (chunks, N); part: [N][chunks][G][2]
template <class E>
__global__ __launch_bounds__(GN_T) void cfl_gn_stats_kernel(const E* __restrict__ x, int HW, int C, int G, int rows, float* __restrict__ part) {
    __shared__ float sm[GN_T * 8], sq[GN_T * 8];               // [rpp][C] mean / M2 of a thread's rows of one channel
    const GMap m = gn_map(C);
    const int r0 = blockIdx.x * rows, r1 = min(HW, r0 + rows);
    const int C8 = C >> 3;
    const E* p = x + ((long long)blockIdx.y * HW + r0 + m.rsub) * C8 + (m.c0 >> 3);
    if (m.active) {
        float f[GN_RPT][8];
        int cnt = 0;
#pragma unroll
        for (int k = 0; k < GN_RPT; ++k) {
            if (r0 + m.rsub + k * m.rpp < r1) {
                unpack8(p[(long long)k * m.rpp * C8], f[k]);
                ++cnt;
            }
        }
        const float inv = cnt ? 1.f / (float)cnt : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float s = 0.f, q = 0.f;
#pragma unroll
            for (int k = 0; k < GN_RPT; ++k) if (k < cnt) s += f[k][j];
            const float mean = s * inv;
#pragma unroll
            for (int k = 0; k < GN_RPT; ++k) if (k < cnt) { const float d = f[k][j] - mean; q = fmaf(d, d, q); }
            sm[m.rsub * C + m.c0 + j] = mean;
            sq[m.rsub * C + m.c0 + j] = q;
        }
    }
    __syncthreads();
    const int cpg = C / G;
    for (int g = threadIdx.x; g < G; g += GN_T) {
        // rows of phase s: those r0 + s + k rpp below r1
        float sum = 0.f;
        for (int s = 0; s < m.rpp; ++s) {
            const int cnt = (r1 - r0 - s + m.rpp - 1) / m.rpp;
            if (r1 - r0 > s) for (int c = 0; c < cpg; ++c) sum = fmaf((float)cnt, sm[s * C + g * cpg + c], sum);
        }
        const float mean = sum / (float)((r1 - r0) * cpg);
        float m2 = 0.f;
        for (int s = 0; s < m.rpp; ++s) {
            const int cnt = (r1 - r0 - s + m.rpp - 1) / m.rpp;
            if (r1 - r0 > s) for (int c = 0; c < cpg; ++c) {
                const float d = sm[s * C + g * cpg + c] - mean;
                m2 += fmaf((float)cnt * d, d, sq[s * C + g * cpg + c]);
            }
        }
        float* o = part + (((long long)blockIdx.y * gridDim.x + blockIdx.x) * G + g) * 2;
        o[0] = mean; o[1] = m2;
    }
}

// merge of the chunks' pairs: mean and 1 / sqrt(var + eps) of every group of sample n into LDS
__device__ __forceinline__ void gn_merge(const float* __restrict__ part, int n, int chunks, int rows, int HW, int cpg, int G, float eps,
                                         float* mu, float* rs) {
    for (int g = threadIdx.x; g < G; g += GN_T) {
        const float* p = part + ((long long)n * chunks * G + g) * 2;
        float sum = 0.f;
        for (int k = 0; k < chunks; ++k) sum = fmaf((float)min(rows, HW - k * rows), p[(long long)k * G * 2], sum);
        const float mean = sum / (float)HW;
        float m2 = 0.f;
        for (int k = 0; k < chunks; ++k) {
            const float d = p[(long long)k * G * 2] - mean;
            m2 += fmaf((float)(min(rows, HW - k * rows) * cpg) * d, d, p[(long long)k * G * 2 + 1]);
        }
        mu[g] = mean;
        rs[g] = 1.f / sqrtf(m2 / ((float)HW * (float)cpg) + eps);
    }
}

// ---- forward, pass 2: y = act(xh gamma + beta (+ res)); the first chunk keeps mean / rstd for the backward
template <class E, int ACT, bool RES>
__global__ __launch_bounds__(GN_T) void cfl_gn_apply_kernel(const E* __restrict__ x, const E* __restrict__ res, const float* __restrict__ gamma,
                                                            const float* __restrict__ beta, const float* __restrict__ part, int HW, int C,
                                                            int G, int rows, float eps, E* __restrict__ y, float* __restrict__ mean,
                                                            float* __restrict__ rstd) {
    __shared__ float mu[GN_MAXC], rs[GN_MAXC];
    const GMap m = gn_map(C);
    const int n = blockIdx.y, cpg = C / G;
    gn_merge(part, n, gridDim.x, rows, HW, cpg, G, eps, mu, rs);
    __syncthreads();
    if (blockIdx.x == 0 && mean) for (int g = threadIdx.x; g < G; g += GN_T) { mean[(long long)n * G + g] = mu[g]; rstd[(long long)n * G + g] = rs[g]; }
    if (!m.active) return;
    float sc[8], sh[8], mv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int g = (m.c0 + j) / cpg;
        sc[j] = rs[g] * gamma[m.c0 + j]; sh[j] = beta[m.c0 + j]; mv[j] = mu[g];
    }
    const int r0 = blockIdx.x * rows, r1 = min(HW, r0 + rows), C8 = C >> 3;
    for (int r = r0 + m.rsub; r < r1; r += m.rpp) {
        const long long at = ((long long)n * HW + r) * C8 + (m.c0 >> 3);
        float f[8], h[8];
        unpack8(x[at], f);
        if (RES) unpack8(res[at], h);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float z = fmaf(f[j] - mv[j], sc[j], sh[j]);
            if (RES) z += h[j];
            f[j] = gn_act<ACT>(z);
        }
        y[at] = pack8g<E>(f);
    }
}

// the gradient of one 8-channel record: the sum of the two that may arrive (added in 32 bits)
template <class E> __device__ __forceinline__ void gn_dy(const E* __restrict__ dy, const E* __restrict__ dy2, long long at, float (&d)[8]) {
    unpack8(dy[at], d);
    if (dy2) {
        float w[8];
        unpack8(dy2[at], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] += w[j];
    }
}
// xh of one record, and its gradient through the activation in place
template <class E, int ACT, bool RES>
__device__ __forceinline__ void gn_dz(const E& xv, const E& rv, const float (&mv)[8], const float (&rv8)[8], const float (&ga)[8],
                                      const float (&be)[8], float (&xh)[8], float (&dz)[8]) {
    float h[8];
    unpack8(xv, xh);
    if (RES && ACT != GN_NONE) unpack8(rv, h);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        xh[j] = (xh[j] - mv[j]) * rv8[j];
        if (ACT != GN_NONE) {
            float z = fmaf(xh[j], ga[j], be[j]);
            if (RES) z += h[j];
            dz[j] *= gn_act_grad<ACT>(z);
        }
    }
}

// ---- backward, pass 1: per chunk, sum dz and sum dz xh of every channel -> pc [N][chunks][2][C], and of every group, weighted with
// gamma -> pg [N][chunks][G][2]
template <class E, int ACT, bool RES>
__global__ __launch_bounds__(GN_T) void cfl_gn_bwd_reduce_kernel(const E* __restrict__ x, const E* __restrict__ dy, const E* __restrict__ dy2,
                                                                 const E* __restrict__ res, const float* __restrict__ gamma,
                                                                 const float* __restrict__ beta, const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd, int HW, int C, int G, int rows,
                                                                 float* __restrict__ pc, float* __restrict__ pg) {
    __shared__ float sa[GN_T * 8], sb[GN_T * 8];
    const GMap m = gn_map(C);
    const int n = blockIdx.y, cpg = C / G, C8 = C >> 3;
    const int r0 = blockIdx.x * rows, r1 = min(HW, r0 + rows);
    if (m.active) {
        float mv[8], rv[8], ga[8], be[8], a[8], b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int g = (m.c0 + j) / cpg;
            mv[j] = mean[(long long)n * G + g]; rv[j] = rstd[(long long)n * G + g];
            ga[j] = gamma[m.c0 + j]; be[j] = beta[m.c0 + j];
            a[j] = 0.f; b[j] = 0.f;
        }
        for (int r = r0 + m.rsub; r < r1; r += m.rpp) {
            const long long at = ((long long)n * HW + r) * C8 + (m.c0 >> 3);
            float xh[8], dz[8];
            E rr{};
            if (RES && ACT != GN_NONE) rr = res[at];
            gn_dy(dy, dy2, at, dz);
            gn_dz<E, ACT, RES>(x[at], rr, mv, rv, ga, be, xh, dz);
#pragma unroll
            for (int j = 0; j < 8; ++j) { a[j] += dz[j]; b[j] = fmaf(dz[j], xh[j], b[j]); }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) { sa[m.rsub * C + m.c0 + j] = a[j]; sb[m.rsub * C + m.c0 + j] = b[j]; }
    }
    __syncthreads();
    const long long blk = (long long)n * gridDim.x + blockIdx.x;
    for (int c = threadIdx.x; c < C; c += GN_T) {
        float a = 0.f, b = 0.f;
        for (int s = 0; s < m.rpp; ++s) { a += sa[s * C + c]; b += sb[s * C + c]; }
        pc[blk * 2 * C + c] = a;
        pc[blk * 2 * C + C + c] = b;
        sa[c] = a * gamma[c]; sb[c] = b * gamma[c];            // (row phase 0's place: read above by this thread alone)
    }
    __syncthreads();
    for (int g = threadIdx.x; g < G; g += GN_T) {
        float a = 0.f, b = 0.f;
        for (int c = 0; c < cpg; ++c) { a += sa[g * cpg + c]; b += sb[g * cpg + c]; }
        pg[(blk * G + g) * 2] = a;
        pg[(blk * G + g) * 2 + 1] = b;
    }
}

// ---- backward, pass 2: dx (and dz = dres)
template <class E, int ACT, bool RES>
__global__ __launch_bounds__(GN_T) void cfl_gn_bwd_apply_kernel(const E* __restrict__ x, const E* __restrict__ dy, const E* __restrict__ dy2,
                                                                const E* __restrict__ res, const float* __restrict__ gamma,
                                                                const float* __restrict__ beta, const float* __restrict__ mean,
                                                                const float* __restrict__ rstd, const float* __restrict__ pg, int HW, int C,
                                                                int G, int rows, E* __restrict__ dx, E* __restrict__ dres) {
    __shared__ float s1[GN_MAXC], s2[GN_MAXC];
    const GMap m = gn_map(C);
    const int n = blockIdx.y, cpg = C / G, C8 = C >> 3;
    for (int g = threadIdx.x; g < G; g += GN_T) {
        const float* p = pg + ((long long)n * gridDim.x * G + g) * 2;
        float a = 0.f, b = 0.f;
        for (int k = 0; k < (int)gridDim.x; ++k) { a += p[(long long)k * G * 2]; b += p[(long long)k * G * 2 + 1]; }
        const float inv = 1.f / ((float)HW * (float)cpg);
        s1[g] = a * inv; s2[g] = b * inv;
    }
    __syncthreads();
    if (!m.active) return;
    float mv[8], rv[8], ga[8], be[8], c1[8], c2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int g = (m.c0 + j) / cpg;
        mv[j] = mean[(long long)n * G + g]; rv[j] = rstd[(long long)n * G + g];
        ga[j] = gamma[m.c0 + j]; be[j] = beta[m.c0 + j];
        c1[j] = s1[g]; c2[j] = s2[g];
    }
    const int r0 = blockIdx.x * rows, r1 = min(HW, r0 + rows);
    for (int r = r0 + m.rsub; r < r1; r += m.rpp) {
        const long long at = ((long long)n * HW + r) * C8 + (m.c0 >> 3);
        float xh[8], dz[8];
        E rr{};
        if (RES && ACT != GN_NONE) rr = res[at];
        gn_dy(dy, dy2, at, dz);
        gn_dz<E, ACT, RES>(x[at], rr, mv, rv, ga, be, xh, dz);
        if (dres) dres[at] = pack8g<E>(dz);
#pragma unroll
        for (int j = 0; j < 8; ++j) dz[j] = rv[j] * (fmaf(dz[j], ga[j], -c1[j]) - xh[j] * c2[j]);
        dx[at] = pack8g<E>(dz);
    }
}

// ---- dgamma / dbeta: sum of pc over samples and chunks, 16 channels x 64 partial groups per workgroup
__global__ __launch_bounds__(1024) void cfl_gn_bwd_final_kernel(const float* __restrict__ pc, int nblk, int C, float* __restrict__ dgamma,
                                                                float* __restrict__ dbeta) {
    __shared__ float sa[64][16], sb[64][16];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), grp = threadIdx.x >> 4;
    float a, b;
    reduce_partials<64>(pc, pc + C, nblk, 2 * C, c < C ? c : 2 * C, grp, a, b, sa, sb);
    if (grp == 0 && c < C) { dbeta[c] = a; dgamma[c] = b; }
}

// rows per chunk: one register load per thread (RPT rows), the chunk count bounded so that its merge stays short
inline int gn_rows(int HW, int C) {
    const int rpp = GN_T / (C >> 3);
    return rpp * GN_RPT;
}
inline bool gn_bad(const void* x, int N, int HW, int C, int G) { return !x || N < 1 || HW < 1 || C < 1 || G < 1 || C % G != 0; }
inline bool gn_limit(int N, int HW, int C) { return C % 8 != 0 || C > GN_MAXC || N > 65535; }

}  // namespace

extern "C" {

size_t cfl_gn_ws_bytes(int N, int HW, int C, int G) {
    if (N < 1 || HW < 1 || C < 8 || G < 1 || C % G || gn_limit(N, HW, C)) return 0;
    const size_t chunks = cfl_cdiv(HW, gn_rows(HW, C));
    return cfl_align256((size_t)N * chunks * G * 2 * 4) + cfl_align256((size_t)N * chunks * C * 2 * 4);
}

#define GN_SWITCH(E, LAUNCH)                                                                            \
    do {                                                                                                \
        if (act == GN_NONE && !res) { LAUNCH(E, GN_NONE, false); }                                      \
        else if (act == GN_NONE) { LAUNCH(E, GN_NONE, true); }                                          \
        else if (act == GN_RELU && !res) { LAUNCH(E, GN_RELU, false); }                                 \
        else if (act == GN_RELU) { LAUNCH(E, GN_RELU, true); }                                          \
        else if (!res) { LAUNCH(E, GN_SILU, false); }                                                   \
        else { LAUNCH(E, GN_SILU, true); }                                                              \
    } while (0)

int cfl_gn_fwd(const void* x, const void* res, const float* gamma, const float* beta, int dtype, int N, int HW, int C, int G, float eps,
               int act, void* y, float* mean, float* rstd, void* ws, void* stream_) {
    if (gn_bad(x, N, HW, C, G) || !gamma || !beta || !y || !ws || dtype < 0 || dtype > 1 || act < 0 || act > 2 || !(eps >= 0.f) ||
        (mean == nullptr) != (rstd == nullptr)) return CFL_EINVAL;
    if (((uintptr_t)x | (uintptr_t)res | (uintptr_t)y) & 15) return CFL_EALIGN;
    if (gn_limit(N, HW, C)) return CFL_ELIMIT;
    hipStream_t stream = (hipStream_t)stream_;
    const int rows = gn_rows(HW, C);
    const dim3 grid(cfl_cdiv(HW, rows), N);
    float* part = (float*)ws;
#define GN_FWD(E, A, R)                                                                                                               \
    CFL_LAUNCH(K_GN_APPLY, (cfl_gn_apply_kernel<E, A, R>), grid, dim3(GN_T), 0, stream, (const E*)x, (const E*)res, gamma, beta, part, \
               HW, C, G, rows, eps, (E*)y, mean, rstd)
    if (dtype == 0) {
        CFL_LAUNCH(K_GN_STATS, cfl_gn_stats_kernel<F8>, grid, dim3(GN_T), 0, stream, (const F8*)x, HW, C, G, rows, part);
        GN_SWITCH(F8, GN_FWD);
    } else {
        CFL_LAUNCH(K_GN_STATS, cfl_gn_stats_kernel<U4>, grid, dim3(GN_T), 0, stream, (const U4*)x, HW, C, G, rows, part);
        GN_SWITCH(U4, GN_FWD);
    }
#undef GN_FWD
    return 0;
}

int cfl_gn_bwd(const void* dy, const void* dy2, const void* x, const void* res, const float* gamma, const float* beta, const float* mean,
               const float* rstd, int dtype, int N, int HW, int C, int G, int act, int want_dres, void* dx, void* dres, float* dgamma,
               float* dbeta, void* ws, void* stream_) {
    if (gn_bad(x, N, HW, C, G) || !dy || !gamma || !beta || !mean || !rstd || !dx || !dgamma || !dbeta || !ws || dtype < 0 || dtype > 1 ||
        act < 0 || act > 2 || (want_dres && !dres)) return CFL_EINVAL;
    if (((uintptr_t)x | (uintptr_t)res | (uintptr_t)dy | (uintptr_t)dy2 | (uintptr_t)dx | (uintptr_t)dres) & 15) return CFL_EALIGN;
    if (gn_limit(N, HW, C)) return CFL_ELIMIT;
    hipStream_t stream = (hipStream_t)stream_;
    const int rows = gn_rows(HW, C), chunks = cfl_cdiv(HW, rows);
    const dim3 grid(chunks, N);
    float* pg = (float*)ws;
    float* pc = (float*)((char*)ws + cfl_align256((size_t)N * chunks * G * 2 * 4));
#define GN_BWD(E, A, R)                                                                                                                 \
    CFL_LAUNCH(K_GN_BWD_REDUCE, (cfl_gn_bwd_reduce_kernel<E, A, R>), grid, dim3(GN_T), 0, stream, (const E*)x, (const E*)dy,            \
               (const E*)dy2, (const E*)res, gamma, beta, mean, rstd, HW, C, G, rows, pc, pg);                                          \
    CFL_LAUNCH(K_GN_BWD_APPLY, (cfl_gn_bwd_apply_kernel<E, A, R>), grid, dim3(GN_T), 0, stream, (const E*)x, (const E*)dy,              \
               (const E*)dy2, (const E*)res, gamma, beta, mean, rstd, pg, HW, C, G, rows, (E*)dx, want_dres ? (E*)dres : (E*)nullptr)
    if (dtype == 0) { GN_SWITCH(F8, GN_BWD); } else { GN_SWITCH(U4, GN_BWD); }
#undef GN_BWD
    CFL_LAUNCH(K_GN_BWD_FINAL, cfl_gn_bwd_final_kernel, dim3(cfl_cdiv(C, 16)), dim3(1024), 0, stream, pc, N * chunks, C, dgamma, dbeta);
    return 0;
}

}  // extern "C"
