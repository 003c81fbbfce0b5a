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

// ---- one pass: a workgroup holds all H W rows of a slice of S channels (whole groups) of one sample in registers, so the activation is
// read once.  Record: 8 channels of one row; a thread holds up to V of them, rows rsub, rsub + rpp, ...  NG = 1: a thread's 8 channels
// lie in one group; NG = 8: each is treated by itself.
struct ResPlan { int S, T; };                                  // channels of a slice (0: does not fit), threads
constexpr int RES_V16 = 14, RES_V32 = 8;                       // records a thread holds in the forward: bf16 / fp32
constexpr int RES_B16 = 13, RES_B32 = 9;                       // ... in the backward: x and the 32-bit gradient
constexpr int RES_TF = 1024, RES_TB = 512;                     // most threads: 128 registers each / 256

// (count, mean, M2) of the workgroup's groups from per-thread pairs in LDS: lds[rsub * slots + slot] = (mean, M2) over cnt(rsub) rows of the
// slot's `w` channels.  Two levels, both exact merges; results in mu[], rs[] (GS groups, `spg` slots each).
__device__ __forceinline__ void gn_block_stats(float2* lds, int T, int slots, int spg, int GS, int rpp, int HW, float w, float eps, float* mu,
                                               float* rs) {
    const int t = threadIdx.x;
    // level 1: part `part` of P merges rows part, part + P, ... of its slot; its pair takes the place of row `part`
    const int P = min(min(T / slots, 16), rpp), slot = t % slots, part = t / slots;
    float n1 = 0.f, mean = 0.f, m2 = 0.f;
    if (part < P) {
        float sum = 0.f;
        for (int r = part; r < rpp && r < HW; r += P) {
            const float c = (float)((HW - r + rpp - 1) / rpp) * w;
            sum = fmaf(c, lds[r * slots + slot].x, sum);
            n1 += c;
        }
        mean = n1 > 0.f ? sum / n1 : 0.f;
        for (int r = part; r < rpp && r < HW; r += P) {
            const float c = (float)((HW - r + rpp - 1) / rpp) * w;
            const float2 v = lds[r * slots + slot];
            const float d = v.x - mean;
            m2 += fmaf(c * d, d, v.y);
        }
    }
    __syncthreads();
    if (part < P) {
        lds[part * slots + slot] = make_float2(mean, m2);
        if (slot == 0) rs[part] = n1;                          // (counts: the same for every slot; rs is free until the end)
    }
    __syncthreads();
    // level 2: L lanes of one wave per group
    int L = 1;
    while (L < 64 && 2 * L * GS <= T) L *= 2;
    float cnt[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) cnt[k] = k < P ? rs[k] : 0.f;
    __syncthreads();
    for (int g0 = 0; g0 < GS; g0 += T / L) {
        const int g = g0 + t / L, l = t % L;
        const bool on = g < GS;
        const int E = on ? P * spg : 0;
        float n = 0.f, sum = 0.f;
        for (int e = l; e < E; e += L) {
            const int k = e / spg;
            float c = 0.f;
#pragma unroll
            for (int q = 0; q < 16; ++q) c = q == k ? cnt[q] : c;
            n += c;
            sum = fmaf(c, lds[k * slots + g * spg + e % spg].x, sum);
        }
        for (int o = L >> 1; o > 0; o >>= 1) { n += __shfl_xor(n, o, 64); sum += __shfl_xor(sum, o, 64); }
        const float gm = n > 0.f ? sum / n : 0.f;
        float q2 = 0.f;
        for (int e = l; e < E; e += L) {
            const int k = e / spg;
            float c = 0.f;
#pragma unroll
            for (int q = 0; q < 16; ++q) c = q == k ? cnt[q] : c;
            const float2 v = lds[k * slots + g * spg + e % spg];
            const float d = v.x - gm;
            q2 += fmaf(c * d, d, v.y);
        }
        for (int o = L >> 1; o > 0; o >>= 1) q2 += __shfl_xor(q2, o, 64);
        if (on && l == 0) { mu[g] = gm; rs[g] = 1.f / sqrtf(q2 / n + eps); }
    }
    __syncthreads();
}

template <class E, int NG, int V>
__global__ __launch_bounds__(RES_TF) void cfl_gn_res_fwd_kernel(const E* __restrict__ x, const E* __restrict__ res, const float* __restrict__ gamma,
                                                              const float* __restrict__ beta, int HW, int C, int G, int S, float eps, int act,
                                                              E* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    extern __shared__ __attribute__((aligned(16))) float gl[];
    const int T = blockDim.x, t = threadIdx.x, cpg = C / G, GS = S / cpg, tpr = S >> 3, rpp = T / tpr, C8 = C >> 3, nsl = C / S;
    const int slots = NG == 1 ? tpr : S, nrs = max(GS, 16);
    float* mu = gl;
    float* rs = gl + nrs;
    float2* lds = reinterpret_cast<float2*>(gl + 2 * nrs);
    const int id = xcd_remap(blockIdx.x, gridDim.x), n = id / nsl, s0 = (id % nsl) * S;
    const int rsub = t / tpr, cl = (t % tpr) * 8, c0 = s0 + cl;
    const bool active = rsub < rpp;
    const long long at0 = ((long long)n * HW + rsub) * C8 + (c0 >> 3), step = (long long)rpp * C8;
    E v[V];
    int cnt = 0;
    if (active) {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (rsub + k * rpp < HW) { v[k] = x[at0 + k * step]; ++cnt; }
        float m8[8], q8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { m8[j] = 0.f; q8[j] = 0.f; }
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k < cnt) {
                float f[8];
                unpack8(v[k], f);
#pragma unroll
                for (int j = 0; j < 8; ++j) m8[j] += f[j];
            }
        const float inv = cnt ? 1.f / (float)cnt : 0.f;
        if (NG == 1) {
            float a = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) a += m8[j];
            a *= inv * 0.125f;
#pragma unroll
            for (int j = 0; j < 8; ++j) m8[j] = a;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) m8[j] *= inv;
        }
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k < cnt) {
                float f[8];
                unpack8(v[k], f);
#pragma unroll
                for (int j = 0; j < 8; ++j) { const float d = f[j] - m8[j]; q8[j] = fmaf(d, d, q8[j]); }
            }
        if (NG == 1) {
            lds[rsub * slots + (cl >> 3)] = make_float2(m8[0], ((q8[0] + q8[1]) + (q8[2] + q8[3])) + ((q8[4] + q8[5]) + (q8[6] + q8[7])));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) lds[rsub * slots + cl + j] = make_float2(m8[j], q8[j]);
        }
    }
    __syncthreads();
    gn_block_stats(lds, T, slots, NG == 1 ? cpg >> 3 : cpg, GS, rpp, HW, NG == 1 ? 8.f : 1.f, eps, mu, rs);
    if (mean && t < GS) { mean[(long long)n * G + s0 / cpg + t] = mu[t]; rstd[(long long)n * G + s0 / cpg + t] = rs[t]; }
    if (!active) return;
    float sc[8], sh[8], mv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int g = (cl + j) / cpg;
        sc[j] = rs[g] * gamma[c0 + j]; sh[j] = beta[c0 + j]; mv[j] = mu[g];
    }
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (k < cnt) {
            float f[8], h[8];
            unpack8(v[k], f);
            if (res) unpack8(res[at0 + k * step], h);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float z = fmaf(f[j] - mv[j], sc[j], sh[j]);
                if (res) z += h[j];
                f[j] = act == GN_RELU ? gn_act<GN_RELU>(z) : act == GN_SILU ? gn_act<GN_SILU>(z) : z;
            }
            y[at0 + k * step] = pack8g<E>(f);
        }
}

// backward in one pass over x, dy (dy2, res): x stays packed, dz in 32 bits.  pc [N][2][C]: the sample's sums of dz and dz xh.
template <class E, int V>
__global__ __launch_bounds__(RES_TB) void cfl_gn_res_bwd_kernel(const E* __restrict__ x, const E* __restrict__ dy, const E* __restrict__ dy2,
                                                              const E* __restrict__ res, const float* __restrict__ gamma,
                                                              const float* __restrict__ beta, const float* __restrict__ mean,
                                                              const float* __restrict__ rstd, int HW, int C, int G, int S, int act,
                                                              E* __restrict__ dx, E* __restrict__ dres, float* __restrict__ pc) {
    extern __shared__ __attribute__((aligned(16))) float gl[];
    const int T = blockDim.x, t = threadIdx.x, cpg = C / G, GS = S / cpg, tpr = S >> 3, rpp = T / tpr, C8 = C >> 3, nsl = C / S;
    float* s1 = gl;                                            // [GS]
    float* s2 = gl + GS;
    float* ta = gl + 2 * GS;                                   // [S] channel totals, weighted with gamma
    float* tb = ta + S;
    float* la = tb + S;                                        // [rpp][S]
    float* lb = la + rpp * S;
    const int id = xcd_remap(blockIdx.x, gridDim.x), n = id / nsl, s0 = (id % nsl) * S;
    const int rsub = t / tpr, cl = (t % tpr) * 8, c0 = s0 + cl;
    const bool active = rsub < rpp;
    const long long at0 = ((long long)n * HW + rsub) * C8 + (c0 >> 3), step = (long long)rpp * C8;
    E v[V];
    float dz[V][8], mv[8], rv[8], ga[8];
    int cnt = 0;
    if (active) {
        float be[8], a8[8], b8[8];
        E d[V];
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (rsub + k * rpp < HW) { v[k] = x[at0 + k * step]; d[k] = dy[at0 + k * step]; ++cnt; }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int g = s0 / cpg + (cl + j) / cpg;
            mv[j] = mean[(long long)n * G + g]; rv[j] = rstd[(long long)n * G + g];
            ga[j] = gamma[c0 + j]; be[j] = beta[c0 + j];
            a8[j] = 0.f; b8[j] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k < cnt) {
                float xh[8], h[8];
                unpack8(v[k], xh);
                unpack8(d[k], dz[k]);
                if (dy2) {
                    unpack8(dy2[at0 + k * step], h);
#pragma unroll
                    for (int j = 0; j < 8; ++j) dz[k][j] += h[j];
                }
                if (res) unpack8(res[at0 + k * step], h);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    xh[j] = (xh[j] - mv[j]) * rv[j];
                    if (act != GN_NONE) {
                        float z = fmaf(xh[j], ga[j], be[j]);
                        if (res) z += h[j];
                        dz[k][j] *= act == GN_RELU ? gn_act_grad<GN_RELU>(z) : gn_act_grad<GN_SILU>(z);
                    }
                    a8[j] += dz[k][j];
                    b8[j] = fmaf(dz[k][j], xh[j], b8[j]);
                }
            }
#pragma unroll
        for (int j = 0; j < 8; ++j) { la[rsub * S + cl + j] = a8[j]; lb[rsub * S + cl + j] = b8[j]; }
    }
    __syncthreads();
    // level 1: part of the row phases of one channel; level 2: the parts of a channel, then the channels of a group
    const int P = min(min(T / S, 32), rpp), c = t % S, part = t / S;
    float a = 0.f, b = 0.f;
    if (part < P) for (int r = part; r < rpp; r += P) { a += la[r * S + c]; b += lb[r * S + c]; }
    __syncthreads();
    if (part < P) { la[part * S + c] = a; lb[part * S + c] = b; }
    __syncthreads();
    if (t < S) {
        float ca = 0.f, cb = 0.f;
        for (int r = 0; r < P; ++r) { ca += la[r * S + t]; cb += lb[r * S + t]; }
        pc[(long long)n * 2 * C + s0 + t] = ca;
        pc[(long long)n * 2 * C + C + s0 + t] = cb;
        ta[t] = ca * gamma[s0 + t]; tb[t] = cb * gamma[s0 + t];
    }
    __syncthreads();
    if (t < GS) {
        const float inv = 1.f / ((float)HW * (float)cpg);
        float ga_ = 0.f, gb_ = 0.f;
        for (int k = 0; k < cpg; ++k) { ga_ += ta[t * cpg + k]; gb_ += tb[t * cpg + k]; }
        s1[t] = ga_ * inv; s2[t] = gb_ * inv;
    }
    __syncthreads();
    if (!active) return;
    float c1[8], c2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { const int g = (cl + j) / cpg; c1[j] = s1[g]; c2[j] = s2[g]; }
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (k < cnt) {
            float xh[8];
            unpack8(v[k], xh);
            if (dres) dres[at0 + k * step] = pack8g<E>(dz[k]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                xh[j] = (xh[j] - mv[j]) * rv[j];
                xh[j] = rv[j] * (fmaf(dz[k][j], ga[j], -c1[j]) - xh[j] * c2[j]);
            }
            dx[at0 + k * step] = pack8g<E>(xh);
        }
}

inline int gn_gcd(int a, int b) { while (b) { const int r = a % b; a = b; b = r; } return a; }

// Slice width and threads of the one-pass kernels for records of `size` bytes an element and at most V records a thread, or S = 0.
// Slices are whole groups and whole records; the widest one up to 128 bytes a row that fits (a row's neighbours then share no cache
// line), else the narrowest possible.  `words`: 32-bit words of LDS per channel and row phase.
inline ResPlan gn_plan(int HW, int C, int G, int size, int V, bool bwd) {
    const int cpg = C / G, unit = cpg / gn_gcd(cpg, 8) * 8;     // lcm(cpg, 8)
    ResPlan best{0, 0};
    for (int S = unit; S <= C; S += unit) {
        if (C % S) continue;
        if (best.S && S * size > 128) break;
        const int tpr = S >> 3;
        const int most = bwd ? RES_TB : RES_TF;
        if (tpr > most || (bwd || cpg % 8 ? S : tpr) > most) break;
        if ((long long)(most / tpr) * V < HW) break;
        const long long rec = (long long)HW * tpr;
        int T = 128;
        while (T < most && (T * 4 < rec || (long long)(T / tpr) * V < HW || (bwd || cpg % 8 ? S : tpr) > T)) T *= 2;
        best.S = S; best.T = T;
    }
    return best;
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
    const ResPlan rp = gn_plan(HW, C, G, dtype ? 2 : 4, dtype ? RES_V16 : RES_V32, false);
    if (rp.S && (long long)N * (C / rp.S) <= 0x7fffffffll) {
        const int ng = (C / G) % 8 ? 8 : 1, gs = rp.S / (C / G), nrs = gs < 16 ? 16 : gs;
        const size_t lds = (size_t)2 * nrs * 4 + (size_t)rp.T * ng * 8;
        const dim3 rg((unsigned)(N * (C / rp.S)));
#define GN_RES(E, NG, V)                                                                                                                   \
    do {                                                                                                                                   \
        CFL_SET_LDS((cfl_gn_res_fwd_kernel<E, NG, V>), 96 * 1024);                                                                         \
        CFL_LAUNCH(K_GN_RES, (cfl_gn_res_fwd_kernel<E, NG, V>), rg, dim3(rp.T), lds, stream, (const E*)x, (const E*)res, gamma, beta, HW, C, \
                   G, rp.S, eps, act, (E*)y, mean, rstd);                                                                                  \
    } while (0)
        if (dtype == 0 && ng == 1) { GN_RES(F8, 1, RES_V32); } else if (dtype == 0) { GN_RES(F8, 8, RES_V32); }
        else if (ng == 1) { GN_RES(U4, 1, RES_V16); } else { GN_RES(U4, 8, RES_V16); }
#undef GN_RES
        return 0;
    }
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
    const ResPlan rp = gn_plan(HW, C, G, dtype ? 2 : 4, dtype ? RES_B16 : RES_B32, true);
    if (rp.S && (long long)N * (C / rp.S) <= 0x7fffffffll) {
        const int rpp = rp.T / (rp.S >> 3);
        const size_t lds = (size_t)2 * (rp.S / (C / G) + rp.S + rpp * rp.S) * 4;
        const dim3 rg((unsigned)(N * (C / rp.S)));
        float* pcr = (float*)ws;
#define GN_RES(E, V)                                                                                                                        \
    do {                                                                                                                                    \
        CFL_SET_LDS((cfl_gn_res_bwd_kernel<E, V>), 96 * 1024);                                                                              \
        CFL_LAUNCH(K_GN_RES, (cfl_gn_res_bwd_kernel<E, V>), rg, dim3(rp.T), lds, stream, (const E*)x, (const E*)dy, (const E*)dy2,          \
                   (const E*)res, gamma, beta, mean, rstd, HW, C, G, rp.S, act, (E*)dx, want_dres ? (E*)dres : (E*)nullptr, pcr);           \
    } while (0)
        if (dtype == 0) { GN_RES(F8, RES_B32); } else { GN_RES(U4, RES_B16); }
#undef GN_RES
        CFL_LAUNCH(K_GN_BWD_FINAL, cfl_gn_bwd_final_kernel, dim3(cfl_cdiv(C, 16)), dim3(1024), 0, stream, pcr, N, C, dgamma, dbeta);
        return 0;
    }
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
