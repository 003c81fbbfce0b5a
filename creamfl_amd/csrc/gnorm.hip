// gnorm.hip -- group normalisation (+ residual add) (+ activation) of channels_last feature maps, forward and backward.
//
//   mu = sum x / M, v = sum (x - mu)^2 / M over a group's M = (C / G) H W values of one sample, r = (v + eps)^-1/2, xh = (x - mu) r
//   z = xh gamma_c + beta_c (+ residual),  y = act(z),  act in {identity, relu, silu}
//   backward: dz = dy act'(z) (= the residual's gradient),  dbeta_c = sum dz,  dgamma_c = sum dz xh  over all samples,
//             g = dz gamma_c,  s1 = sum_group g / M,  s2 = sum_group g xh / M,  dx = r (g - s1 - xh s2)
//
// Where it sits: the normalisation of the image trunks (src/networks/models/image_encoder.py:27-36, src/networks/resnet_client.py:60-98
// use BatchNorm there), for federations whose clients' batch statistics do not average.
// HBM-bound: bf16 256 x 56 x 56 x 256 with a residual takes 266 us forward (290 before what fits registers and LDS was kept for the second
// pass) and 605 backward (everything read twice, 5.4 TB/s; the same keeping there, three records of 25, gave 1 %); fp32 128 x 28 x 28 x 128,
// read once, 24 and 38 us (4.2 and 4.0 TB/s).  A one-pass form that kept slices of 200 KB in registers, one workgroup a CU, lost: its loads and
// stores do not overlap (261 us without, 329 with a residual).
// A sample is a row-major [H W, C] matrix; a thread owns 8 consecutive channels of its rows (one 16-byte access in bf16).
// Statistics: a thread keeps its RPT rows in registers and forms mean and squared deviations of what it holds in two passes; partial
// (mean, M2) pairs are then merged by sum n (mean - mu)^2, so that a mean much larger than the deviation costs no digits (a running
// sum of squares would).  Everything is summed in 32 bits and in a fixed order: two runs give the same bits.
#include <type_traits>
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

// 1 / (1 + e^-z) on the hardware's exp2 and reciprocal (one unit in the last place each; an IEEE division would cost more than all the rest
// of the pass: the forward has 28 vector operations per element at the memory's pace, and a division takes ten)
__device__ __forceinline__ float gn_sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}
__device__ __forceinline__ float gn_act(int act, float z) {
    if (act == GN_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
    if (act == GN_SILU) return z * gn_sigmoid(z);
    return z;
}
// d act'(z).  ReLU selects: where it is closed the result is 0 whatever the gradient holds (a product would make NaN of an infinite one, and
// the group's sums would carry it into the whole group)
__device__ __forceinline__ float gn_act_grad(int act, float z, float d) {
    if (act == GN_RELU) return z > 0.f ? d : 0.f;
    if (act == GN_SILU) { const float s = gn_sigmoid(z); return d * (s * fmaf(z, 1.f - s, 1.f)); }
    return d;
}
// 8 channels rounded once (hardware conversion, two values an instruction)
__device__ __forceinline__ void gn_store(U4* p, const float (&f)[8]) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef float w8 __attribute__((ext_vector_type(8)));
    w8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = f[j];
    *reinterpret_cast<v8*>(p) = __builtin_convertvector(o, v8);
}
__device__ __forceinline__ void gn_store(F8* p, const float (&f)[8]) { *p = pack8g<F8>(f); }
// group (from the slice's first) of each of a thread's 8 channels cl .. cl + 7
__device__ __forceinline__ void gn_groups(int cl, int cpg, int (&g)[8]) {
    g[0] = cl / cpg;
    int r = cl - g[0] * cpg;
#pragma unroll
    for (int j = 1; j < 8; ++j) {
        const bool next = ++r == cpg;
        g[j] = g[j - 1] + (next ? 1 : 0);
        r = next ? 0 : r;
    }
}

// lanes (a power of two) of a wave for each of G groups of `work` items, GN_T threads in all (one thread a group took 175 us of a map of 64 channels
// in one group, 32 row phases)
__device__ __forceinline__ int gn_lanes(int G, int work) {
    int L = 1;
    while (L < 64 && 2 * L * G <= GN_T && L < work) L *= 2;
    return L;
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
    // L lanes of a wave to a group, over its (row phase, channel) pairs
    const int cpg = C / G, pairs = m.rpp * cpg, L = gn_lanes(G, pairs), l = threadIdx.x & (L - 1);
    for (int g0 = 0; g0 < G; g0 += GN_T / L) {
        const int g = g0 + threadIdx.x / L;
        const bool on = g < G;
        float sum = 0.f;
        for (int k = l; on && k < pairs; k += L) {
            const int s = k / cpg, cnt = (r1 - r0 - s + m.rpp - 1) / m.rpp;      // rows of phase s: those r0 + s + i rpp below r1
            if (r1 - r0 > s) sum = fmaf((float)cnt, sm[s * C + g * cpg + k - s * cpg], sum);
        }
        for (int o = L >> 1; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        const float mean = sum / (float)((r1 - r0) * cpg);
        float m2 = 0.f;
        for (int k = l; on && k < pairs; k += L) {
            const int s = k / cpg, cnt = (r1 - r0 - s + m.rpp - 1) / m.rpp, at = s * C + g * cpg + k - s * cpg;
            if (r1 - r0 > s) {
                const float d = sm[at] - mean;
                m2 += fmaf((float)cnt * d, d, sq[at]);
            }
        }
        for (int o = L >> 1; o > 0; o >>= 1) m2 += __shfl_xor(m2, o, 64);
        if (on && l == 0) {
            float* o = part + (((long long)blockIdx.y * gridDim.x + blockIdx.x) * G + g) * 2;
            o[0] = mean; o[1] = m2;
        }
    }
}

// merge of the chunks' pairs: mean and 1 / sqrt(var + eps) of every group of sample n into mu, rs.  Thread t of T takes every T-th group, L lanes
// of a wave to a group, their partial merges by the same formula.
template <int T, int L>
__device__ __forceinline__ void gn_merge(const float* __restrict__ part, int n, int chunks, int rows, int HW, int cpg, int G, float eps,
                                         float* mu, float* rs) {
    const int l = threadIdx.x % L;
    for (int g0 = 0; g0 < G; g0 += T / L) {
        const int g = g0 + threadIdx.x / L;
        const float* p = part + ((long long)n * chunks * G + min(g, G - 1)) * 2;
        float sum = 0.f;
        for (int k = l; k < chunks; k += L) sum = fmaf((float)min(rows, HW - k * rows), p[(long long)k * G * 2], sum);
        for (int o = L >> 1; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        const float mean = sum / (float)HW;
        float m2 = 0.f;
        for (int k = l; k < chunks; k += L) {
            const float d = p[(long long)k * G * 2] - mean;
            m2 += fmaf((float)(min(rows, HW - k * rows) * cpg) * d, d, p[(long long)k * G * 2 + 1]);
        }
        for (int o = L >> 1; o > 0; o >>= 1) m2 += __shfl_xor(m2, o, 64);
        if (g < G && l == 0) {
            mu[g] = mean;
            rs[g] = 1.f / sqrtf(m2 / ((float)HW * (float)cpg) + eps);
        }
    }
}
// More than GN_MERGE chunks: every workgroup of the second pass merging them for itself would cost their number squared; one small launch does it
// once, a workgroup a sample.  stats: [2][N][G].
constexpr int GN_MERGE = 64;
__global__ __launch_bounds__(1024) void cfl_gn_merge_kernel(const float* __restrict__ part, int chunks, int rows, int HW, int cpg, int G, float eps,
                                                            float* __restrict__ stats) {
    float* mu = stats + (long long)blockIdx.x * G;
    gn_merge<1024, 64>(part, blockIdx.x, chunks, rows, HW, cpg, G, eps, mu, mu + (long long)gridDim.x * G);
}

// ---- forward, pass 2: y = act(xh gamma + beta (+ res)); the first chunk keeps mean / rstd for the backward
template <class E, int ACT, bool RES>
__global__ __launch_bounds__(GN_T) void cfl_gn_apply_kernel(const E* __restrict__ x, const E* __restrict__ res, const float* __restrict__ gamma,
                                                            const float* __restrict__ beta, const float* __restrict__ part, int HW, int C,
                                                            int G, int rows, float eps, E* __restrict__ y, float* __restrict__ mean,
                                                            float* __restrict__ rstd, const float* __restrict__ stats) {
    __shared__ float mu[GN_MAXC], rs[GN_MAXC];
    const GMap m = gn_map(C);
    const int n = blockIdx.y, cpg = C / G;
    if (stats) {
        const float* p = stats + (long long)n * G;
        for (int g = threadIdx.x; g < G; g += GN_T) { mu[g] = p[g]; rs[g] = p[(long long)gridDim.y * G + g]; }
    } else {
        gn_merge<GN_T, 1>(part, n, gridDim.x, rows, HW, cpg, G, eps, mu, rs);
    }
    __syncthreads();
    if (blockIdx.x == 0 && mean) for (int g = threadIdx.x; g < G; g += GN_T) { mean[(long long)n * G + g] = mu[g]; rstd[(long long)n * G + g] = rs[g]; }
    if (!m.active) return;
    float sc[8], sh[8], mv[8];
    int gi[8];
    gn_groups(m.c0, cpg, gi);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int g = gi[j];
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
            f[j] = gn_act(ACT, z);
        }
        gn_store(y + at, f);
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
            dz[j] = gn_act_grad(ACT, z, dz[j]);
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
        int gi[8];
        gn_groups(m.c0, cpg, gi);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int g = gi[j];
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
        float p[4] = {0.f, 0.f, 0.f, 0.f}, q[4] = {0.f, 0.f, 0.f, 0.f};      // (four chains: one of 256 equal terms is off by up to 64 halves of a last place)
        int s = 0;
        for (; s + 3 < m.rpp; s += 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { p[i] += sa[(s + i) * C + c]; q[i] += sb[(s + i) * C + c]; }
        }
        for (; s < m.rpp; ++s) { p[0] += sa[s * C + c]; q[0] += sb[s * C + c]; }
        const float a = (p[0] + p[1]) + (p[2] + p[3]), b = (q[0] + q[1]) + (q[2] + q[3]);
        pc[blk * 2 * C + c] = a;
        pc[blk * 2 * C + C + c] = b;
        sa[c] = a * gamma[c]; sb[c] = b * gamma[c];            // (row phase 0's place: read above by this thread alone)
    }
    __syncthreads();
    const int L = gn_lanes(G, cpg), l = threadIdx.x & (L - 1);
    for (int g0 = 0; g0 < G; g0 += GN_T / L) {
        const int g = g0 + threadIdx.x / L;
        float a = 0.f, b = 0.f;
        for (int c = l; g < G && c < cpg; c += L) { a += sa[g * cpg + c]; b += sb[g * cpg + c]; }
        for (int o = L >> 1; o > 0; o >>= 1) { a += __shfl_xor(a, o, 64); b += __shfl_xor(b, o, 64); }
        if (g < G && l == 0) { pg[(blk * G + g) * 2] = a; pg[(blk * G + g) * 2 + 1] = b; }
    }
}

// the chunks' group sums of a sample added up, where they are many (as cfl_gn_merge_kernel): to the place of its chunk 0.  grid = (G, N)
__global__ __launch_bounds__(64) void cfl_gn_bwd_merge_kernel(float* __restrict__ pg, int chunks, int G) {
    float* p = pg + ((long long)blockIdx.y * chunks * G + blockIdx.x) * 2;
    float a = 0.f, b = 0.f;
    for (int k = threadIdx.x; k < chunks; k += 64) { a += p[(long long)k * G * 2]; b += p[(long long)k * G * 2 + 1]; }
    a = wave_sum(a);
    b = wave_sum(b);
    if (threadIdx.x == 0) { p[0] = a; p[1] = b; }
}

// ---- backward, pass 2: dx (and dz = dres)
template <class E, int ACT, bool RES>
__global__ __launch_bounds__(GN_T) void cfl_gn_bwd_apply_kernel(const E* __restrict__ x, const E* __restrict__ dy, const E* __restrict__ dy2,
                                                                const E* __restrict__ res, const float* __restrict__ gamma,
                                                                const float* __restrict__ beta, const float* __restrict__ mean,
                                                                const float* __restrict__ rstd, const float* __restrict__ pg, int HW, int C,
                                                                int G, int rows, int sums, E* __restrict__ dx, E* __restrict__ dres) {
    __shared__ float s1[GN_MAXC], s2[GN_MAXC];
    const GMap m = gn_map(C);
    const int n = blockIdx.y, cpg = C / G, C8 = C >> 3;
    for (int g = threadIdx.x; g < G; g += GN_T) {
        const float* p = pg + ((long long)n * gridDim.x * G + g) * 2;
        float a = 0.f, b = 0.f;
        for (int k = 0; k < sums; ++k) { a += p[(long long)k * G * 2]; b += p[(long long)k * G * 2 + 1]; }
        const float inv = 1.f / ((float)HW * (float)cpg);
        s1[g] = a * inv; s2[g] = b * inv;
    }
    __syncthreads();
    if (!m.active) return;
    float mv[8], rv[8], ga[8], be[8], c1[8], c2[8];
    int gi[8];
    gn_groups(m.c0, cpg, gi);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int g = gi[j];
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
        if (dres) gn_store(dres + at, dz);
#pragma unroll
        for (int j = 0; j < 8; ++j) dz[j] = rv[j] * (fmaf(dz[j], ga[j], -c1[j]) - xh[j] * c2[j]);
        gn_store(dx + at, dz);
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
constexpr int RES_V16 = 14, RES_V32 = 8;                       // records a thread holds in the forward: bf16 / fp32
constexpr int RES_B16 = 13, RES_B32 = 9;                       // ... in the backward: x and the 32-bit gradient
constexpr int RES_F16 = 4, RES_F32 = 3;                        // ... in the variants for few records
constexpr int STR_T = 1024;                                    // threads of the two-pass kernels
constexpr int STR_KEEP = 8;                                    // records a thread keeps in the forward of bf16
constexpr int RES_T = 512;                                     // most threads of the one-pass kernels

// (count, mean, M2) of the workgroup's groups from per-thread pairs in LDS: lds[rsub * slots + slot] = (mean, M2) over cnt(rsub) rows of the
// slot's `w` channels.  Two levels, both exact merges; results in mu[], rs[] (GS groups, `spg` slots each).
__device__ __forceinline__ void gn_block_stats(float2* lds, float* cn, int T, int slots, int spg, int GS, int rpp, int HW, float w, float eps,
                                               float* mu, float* rs) {
    const int t = threadIdx.x;
    // level 1: part `part` of P merges rows part, part + P, ... of its slot; its pair takes the place of row `part`, its count cn[part]
    const int q = T / slots, P = min(min(q, 16), rpp), part = t / slots, slot = t - part * slots, rows = min(rpp, HW);
    const int full = HW / rpp, more = HW - full * rpp;         // a row phase r has full + (r < more) rows
    float n1 = 0.f, mean = 0.f, m2 = 0.f;
    if (part < P) {
        float sum = 0.f;
        for (int r = part; r < rows; r += P) {
            const float c = (float)(full + (r < more)) * w;
            sum = fmaf(c, lds[r * slots + slot].x, sum);
            n1 += c;
        }
        mean = n1 > 0.f ? sum / n1 : 0.f;
        for (int r = part; r < rows; r += P) {
            const float c = (float)(full + (r < more)) * w;
            const float2 v = lds[r * slots + slot];
            const float d = v.x - mean;
            m2 += fmaf(c * d, d, v.y);
        }
    }
    __syncthreads();
    if (part < P) {
        lds[part * slots + slot] = make_float2(mean, m2);
        if (slot == 0) cn[part] = n1;
    }
    __syncthreads();
    // level 2: L lanes of one wave per group
    int L = 1;
    while (L < 64 && 2 * L * GS <= T && L < P * spg) L *= 2;
    for (int g0 = 0; g0 < GS; g0 += T / L) {
        const int g = g0 + t / L, l = t & (L - 1);
        const bool on = g < GS;
        float n = 0.f, sum = 0.f;
        if (on)
            for (int k = l / spg, s = l - k * spg; k < P; ) {
                const float c = cn[k];
                n += c;
                sum = fmaf(c, lds[k * slots + g * spg + s].x, sum);
                for (s += L; s >= spg && k < P; s -= spg) ++k;
            }
        for (int o = L >> 1; o > 0; o >>= 1) { n += __shfl_xor(n, o, 64); sum += __shfl_xor(sum, o, 64); }
        const float gm = n > 0.f ? sum / n : 0.f;
        float q2 = 0.f;
        if (on)
            for (int k = l / spg, s = l - k * spg; k < P; ) {
                const float2 v = lds[k * slots + g * spg + s];
                const float d = v.x - gm;
                q2 += fmaf(cn[k] * d, d, v.y);
                for (s += L; s >= spg && k < P; s -= spg) ++k;
            }
        for (int o = L >> 1; o > 0; o >>= 1) q2 += __shfl_xor(q2, o, 64);
        if (on && l == 0) { mu[g] = gm; rs[g] = 1.f / sqrtf(q2 / n + eps); }
    }
    __syncthreads();
}

template <class E, int NG, int V>
__global__ __launch_bounds__(V <= 4 ? 256 : RES_T) void cfl_gn_res_fwd_kernel(const E* __restrict__ x, const E* __restrict__ res, const float* __restrict__ gamma,
                                                              const float* __restrict__ beta, int HW, int C, int G, int S, float eps, int act,
                                                              E* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    extern __shared__ __attribute__((aligned(16))) float gl[];
    const int T = blockDim.x, t = threadIdx.x, cpg = C / G, GS = S / cpg, tpr = S >> 3, rpp = T / tpr, C8 = C >> 3, nsl = C / S;
    const int slots = NG == 1 ? tpr : S;
    float* cn = gl;                                            // [16]
    float2* lds = reinterpret_cast<float2*>(gl + 16);          // [T NG]
    float* mu = gl + 16 + 2 * T * NG;
    float* rs = mu + GS;
    const int id = xcd_remap(blockIdx.x, gridDim.x), n = id / nsl, s0 = (id % nsl) * S;
    const int rsub = t / tpr, cl = (t - rsub * tpr) * 8, c0 = s0 + cl;
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
    gn_block_stats(lds, cn, T, slots, NG == 1 ? cpg >> 3 : cpg, GS, rpp, HW, NG == 1 ? 8.f : 1.f, eps, mu, rs);
    if (mean) for (int g = t; g < GS; g += T) { mean[(long long)n * G + s0 / cpg + g] = mu[g]; rstd[(long long)n * G + s0 / cpg + g] = rs[g]; }
    if (!active) return;
    float sc[8], sh[8], mv[8];
    int gi[8];
    gn_groups(cl, cpg, gi);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int g = gi[j];
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
                f[j] = gn_act(act, z);
            }
            gn_store(y + at0 + k * step, f);
        }
}

// the workgroup's channel sums from its row phases' (la, lb: [rpp][S]): to pc[0 .. S), pc[C .. C + S), and, weighted with gamma, their groups'
// means s1, s2.  Two levels over the row phases, then L lanes of a wave per group; S <= T.
__device__ __forceinline__ void gn_block_sums(float* la, float* lb, float* ta, float* tb, float* s1, float* s2, int T, int S, int GS, int cpg,
                                              int rpp, int HW, const float* __restrict__ gamma, float* __restrict__ pc, int C) {
    const int t = threadIdx.x, part = t / S, c = t - part * S, P = min(min(T / S, 16), rpp);
    float a = 0.f, b = 0.f;
    if (part < P) for (int r = part; r < rpp; r += P) { a += la[r * S + c]; b += lb[r * S + c]; }
    __syncthreads();
    if (part < P) { la[part * S + c] = a; lb[part * S + c] = b; }
    __syncthreads();
    if (t < S) {
        float ca = 0.f, cb = 0.f;
        for (int r = 0; r < P; ++r) { ca += la[r * S + t]; cb += lb[r * S + t]; }
        pc[t] = ca;
        pc[C + t] = cb;
        ta[t] = ca * gamma[t]; tb[t] = cb * gamma[t];
    }
    __syncthreads();
    int L = 1;
    while (L < 64 && 2 * L * GS <= T && L < cpg) L *= 2;
    const float inv = 1.f / ((float)HW * (float)cpg);
    for (int g0 = 0; g0 < GS; g0 += T / L) {
        const int g = g0 + t / L, l = t & (L - 1);
        float x = 0.f, y = 0.f;
        if (g < GS) for (int k = l; k < cpg; k += L) { x += ta[g * cpg + k]; y += tb[g * cpg + k]; }
        for (int o = L >> 1; o > 0; o >>= 1) { x += __shfl_xor(x, o, 64); y += __shfl_xor(y, o, 64); }
        if (g < GS && l == 0) { s1[g] = x * inv; s2[g] = y * inv; }
    }
    __syncthreads();
}

// backward in one pass over x, dy (dy2, res): x stays packed, dz in 32 bits.  pc [N][2][C]: the sample's sums of dz and dz xh.
template <class E, int V>
__global__ __launch_bounds__(V <= 4 ? 256 : RES_T) void cfl_gn_res_bwd_kernel(const E* __restrict__ x, const E* __restrict__ dy, const E* __restrict__ dy2,
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
    const int rsub = t / tpr, cl = (t - rsub * tpr) * 8, c0 = s0 + cl, g0 = s0 / cpg;
    const bool active = rsub < rpp;
    const long long at0 = ((long long)n * HW + rsub) * C8 + (c0 >> 3), step = (long long)rpp * C8;
    E v[V];
    float dz[V][8], mv[8], rv[8], ga[8];
    int cnt = 0, gi[8];
    gn_groups(cl, cpg, gi);
    if (active) {
        float be[8], a8[8], b8[8];
        E d[V], w[V];                                          // (everything is requested before anything is used)
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (rsub + k * rpp < HW) { v[k] = x[at0 + k * step]; d[k] = dy[at0 + k * step]; ++cnt; }
        constexpr bool AHEAD = sizeof(E) == 16 || V <= 3;      // (the 32-byte records of fp32 leave no registers for it)
        if (AHEAD && res) {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (k < cnt) w[k] = res[at0 + k * step];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int g = g0 + gi[j];
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
                if (res) unpack8(AHEAD ? w[k] : res[at0 + k * step], h);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    xh[j] = (xh[j] - mv[j]) * rv[j];
                    if (act != GN_NONE) {
                        float z = fmaf(xh[j], ga[j], be[j]);
                        if (res) z += h[j];
                        dz[k][j] = gn_act_grad(act, z, dz[k][j]);
                    }
                    a8[j] += dz[k][j];
                    b8[j] = fmaf(dz[k][j], xh[j], b8[j]);
                }
            }
#pragma unroll
        for (int j = 0; j < 8; ++j) { la[rsub * S + cl + j] = a8[j]; lb[rsub * S + cl + j] = b8[j]; }
    }
    __syncthreads();
    gn_block_sums(la, lb, ta, tb, s1, s2, T, S, GS, cpg, rpp, HW, gamma + s0, pc + (long long)n * 2 * C + s0, C);
    if (!active) return;
    float c1[8], c2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { c1[j] = s1[gi[j]]; c2[j] = s2[gi[j]]; }
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (k < cnt) {
            float xh[8];
            unpack8(v[k], xh);
            if (dres) gn_store(dres + at0 + k * step, dz[k]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                xh[j] = (xh[j] - mv[j]) * rv[j];
                xh[j] = rv[j] * (fmaf(dz[k][j], ga[j], -c1[j]) - xh[j] * c2[j]);
            }
            gn_store(dx + at0 + k * step, xh);
        }
}

// ---- the same in two passes of one workgroup over its slice, for slices that do not fit the registers: the second pass finds most of the
// slice in the caches (L2 and the 256 MB behind it), and runs from the last row to the first, the most recently read ones.
// Statistics: the records that a thread has in registers together give a mean and squared deviations of their own, which join the thread's by
// the formula of all merges (gn_join).  A value far from the rest -- a corner, a border -- costs no digits wherever it stands; one running sum of
// squares from a fixed shift would lose them where it is the shift: 2e-3 to 6e-2 of the variance at 512 x 512 (restated on the CPU; this: 6e-7).
// KEEP of a thread's last records stay in registers and `kl` before them in LDS (its own place): the second pass does not read them again (17 of
// 25 at 56 x 56 x 256 bf16: 290 -> 266 us with a residual; ten in registers 275).
template <class E, int B>
__device__ __forceinline__ void gn_join(const E (&v)[B], int c, float& n, float (&mean)[8], float (&m2)[8]) {      // the first c of v; c >= 1
    float f[B][8];
#pragma unroll
    for (int u = 0; u < B; ++u) unpack8(v[u], f[u]);
    const float cf = (float)c, inv = c == B ? 1.f / B : __builtin_amdgcn_rcpf(cf), all = n + cf, w = cf * __builtin_amdgcn_rcpf(all), nw = n * w;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int u = 0; u < B; ++u) s += u < c ? f[u][j] : 0.f;
        s *= inv;
#pragma unroll
        for (int u = 0; u < B; ++u) { const float d = u < c ? f[u][j] - s : 0.f; q = fmaf(d, d, q); }
        const float d = s - mean[j];
        mean[j] = fmaf(d, w, mean[j]);
        m2[j] += fmaf(d * nw, d, q);                             // (in this order: a first mean of 1e20 must not meet 0 as infinity)
    }
    n = all;
}
template <class E, int NG, int U, int KEEP>
__global__ __launch_bounds__(STR_T) void cfl_gn_str_fwd_kernel(const E* __restrict__ x, const E* __restrict__ res, const float* __restrict__ gamma,
                                                               const float* __restrict__ beta, int HW, int C, int G, int S, float eps, int act, int kl,
                                                               E* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    extern __shared__ __attribute__((aligned(16))) float gl[];
    const int T = blockDim.x, t = threadIdx.x, cpg = C / G, GS = S / cpg, tpr = S >> 3, rpp = T / tpr, C8 = C >> 3, nsl = C / S;
    const int slots = NG == 1 ? tpr : S;
    float* cn = gl;
    float2* lds = reinterpret_cast<float2*>(gl + 16);
    float* mu = gl + 16 + 2 * T * NG;
    float* rs = mu + GS;
    E* kept = reinterpret_cast<E*>(gl + (16 + 2 * T * NG + 2 * GS + 3) / 4 * 4);      // [kl][T]
    const int id = xcd_remap(blockIdx.x, gridDim.x), n = id / nsl, s0 = (id % nsl) * S;
    const int rsub = t / tpr, cl = (t - rsub * tpr) * 8, c0 = s0 + cl;
    const bool active = rsub < rpp;
    const long long step = (long long)rpp * C8;
    const E* px = x + ((long long)n * HW + rsub) * C8 + (c0 >> 3);
    const int cnt = active && rsub < HW ? (HW - rsub + rpp - 1) / rpp : 0;
    const int tail = max(cnt - KEEP, 0), body = max(tail - kl, 0);       // records from `body` on: LDS, from `tail` on: registers
    E own[KEEP > 0 ? KEEP : 1];
    if (active) {
        float have = 0.f, s[8], q[8];                           // rows taken; their mean and squared deviations
#pragma unroll
        for (int j = 0; j < 8; ++j) { s[j] = 0.f; q[j] = 0.f; }
        const auto pass = [&](int from, int to, auto keep) {
            for (int k0 = from; k0 < to; k0 += U) {
                E v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) v[u] = px[min(k0 + u, to - 1) * step];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (keep && k0 + u < to) kept[(k0 + u - from) * T + t] = v[u];
                if (to - k0 >= U) gn_join(v, U, have, s, q);
                else gn_join(v, to - k0, have, s, q);
            }
        };
        pass(0, body, std::false_type{});
        pass(body, tail, std::true_type{});
        if (KEEP > 0 && cnt) {
#pragma unroll
            for (int i = 0; i < KEEP; ++i) own[i] = px[min(tail + i, cnt - 1) * step];
            gn_join(own, min(KEEP, cnt), have, s, q);
        }
        if (NG == 1) {
            float m = 0.f, m2 = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) m += s[j];
            m *= 0.125f;
#pragma unroll
            for (int j = 0; j < 8; ++j) { const float d = s[j] - m; m2 += fmaf((float)cnt * d, d, q[j]); }
            lds[rsub * slots + (cl >> 3)] = make_float2(m, m2);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) lds[rsub * slots + cl + j] = make_float2(s[j], q[j]);
        }
    }
    __syncthreads();
    gn_block_stats(lds, cn, T, slots, NG == 1 ? cpg >> 3 : cpg, GS, rpp, HW, NG == 1 ? 8.f : 1.f, eps, mu, rs);
    if (mean) for (int g = t; g < GS; g += T) { mean[(long long)n * G + s0 / cpg + g] = mu[g]; rstd[(long long)n * G + s0 / cpg + g] = rs[g]; }
    if (!cnt) return;
    float sc[8], sh[8], mv[8];
    int gi[8];
    gn_groups(cl, cpg, gi);
#pragma unroll
    for (int j = 0; j < 8; ++j) { sc[j] = rs[gi[j]] * gamma[c0 + j]; sh[j] = beta[c0 + j]; mv[j] = mu[gi[j]]; }
    const E* pr = res ? res + (px - x) : nullptr;
    E* py = y + (px - x);
    const auto put = [&](const E& v, const E& w, int at) {
        float f[8], h[8];
        unpack8(v, f);
        if (res) unpack8(w, h);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float z = fmaf(f[j] - mv[j], sc[j], sh[j]);
            if (res) z += h[j];
            f[j] = gn_act(act, z);
        }
        gn_store(py + at * step, f);
    };
#pragma unroll
    for (int i0 = 0; i0 < KEEP; i0 += U) {
        E w[U];
        if (res) {
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = pr[min(tail + i0 + u, cnt - 1) * step];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (tail + i0 + u < cnt) put(own[i0 + u], w[u], tail + i0 + u);
    }
    const auto back = [&](int from, int to, auto keep) {           // records to - 1 .. from
        for (int k0 = to - 1; k0 >= from; k0 -= U) {
            E v[U], w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = keep ? kept[(max(k0 - u, from) - from) * T + t] : px[max(k0 - u, from) * step];
            if (res) {
#pragma unroll
                for (int u = 0; u < U; ++u) w[u] = pr[max(k0 - u, from) * step];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (k0 - u < from) break;
                put(v[u], w[u], k0 - u);
            }
        }
    };
    back(body, tail, std::true_type{});
    back(0, body, std::false_type{});
}

template <class E, int U>
__global__ __launch_bounds__(STR_T) void cfl_gn_str_bwd_kernel(const E* __restrict__ x, const E* __restrict__ dy, const E* __restrict__ dy2,
                                                               const E* __restrict__ res, const float* __restrict__ gamma,
                                                               const float* __restrict__ beta, const float* __restrict__ mean,
                                                               const float* __restrict__ rstd, int HW, int C, int G, int S, int act,
                                                               E* __restrict__ dx, E* __restrict__ dres, float* __restrict__ pc) {
    extern __shared__ __attribute__((aligned(16))) float gl[];
    const int T = blockDim.x, t = threadIdx.x, cpg = C / G, GS = S / cpg, tpr = S >> 3, rpp = T / tpr, C8 = C >> 3, nsl = C / S;
    float* s1 = gl;
    float* s2 = gl + GS;
    float* ta = gl + 2 * GS;
    float* tb = ta + S;
    float* la = tb + S;
    float* lb = la + rpp * S;
    const int id = xcd_remap(blockIdx.x, gridDim.x), n = id / nsl, s0 = (id % nsl) * S;
    const int rsub = t / tpr, cl = (t - rsub * tpr) * 8, c0 = s0 + cl, g0 = s0 / cpg;
    const bool active = rsub < rpp;
    const long long at0 = ((long long)n * HW + rsub) * C8 + (c0 >> 3), step = (long long)rpp * C8;
    const int cnt = active && rsub < HW ? (HW - rsub + rpp - 1) / rpp : 0;
    float mv[8], rv[8], ga[8], be[8];
    int gi[8];
    gn_groups(cl, cpg, gi);
    const auto load = [&](int k, E& xv, float (&dz)[8], E& hv) {
        const long long at = at0 + k * step;
        xv = x[at];
        gn_dy(dy, dy2, at, dz);
        if (res) hv = res[at];
    };
    const auto form = [&](const E& xv, const E& hv, float (&xh)[8], float (&dz)[8]) {
        float h[8];
        unpack8(xv, xh);
        if (res) unpack8(hv, h);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            xh[j] = (xh[j] - mv[j]) * rv[j];
            if (act != GN_NONE) {
                float z = fmaf(xh[j], ga[j], be[j]);
                if (res) z += h[j];
                dz[j] = gn_act_grad(act, z, dz[j]);
            }
        }
    };
    if (active) {
        float* pa = la + rsub * S + cl;
        float* pb = lb + rsub * S + cl;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            mv[j] = mean[(long long)n * G + g0 + gi[j]]; rv[j] = rstd[(long long)n * G + g0 + gi[j]];
            ga[j] = gamma[c0 + j]; be[j] = beta[c0 + j];
            pa[j] = 0.f; pb[j] = 0.f;
        }
        // sums of 16 records join the thread's in LDS (its own words): equal terms round the same way, and a chain of 512 would be off by up to 127
        // halves of a last place, of 2048 by 508
        for (int b0 = 0; b0 < cnt; b0 += 16) {
            const int to = min(b0 + 16, cnt);
            float a[8], b[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) { a[j] = 0.f; b[j] = 0.f; }
            for (int k0 = b0; k0 < to; k0 += U) {
                E xv[U], hv[U];
                float dz[U][8];
#pragma unroll
                for (int u = 0; u < U; ++u) load(min(k0 + u, to - 1), xv[u], dz[u], hv[u]);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (k0 + u >= to) break;
                    float xh[8];
                    form(xv[u], hv[u], xh, dz[u]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) { a[j] += dz[u][j]; b[j] = fmaf(dz[u][j], xh[j], b[j]); }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) { pa[j] += a[j]; pb[j] += b[j]; }
        }
    }
    __syncthreads();
    gn_block_sums(la, lb, ta, tb, s1, s2, T, S, GS, cpg, rpp, HW, gamma + s0, pc + (long long)n * 2 * C + s0, C);
    if (!cnt) return;
    float c1[8], c2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { c1[j] = s1[gi[j]]; c2[j] = s2[gi[j]]; }
    for (int k0 = cnt - 1; k0 >= 0; k0 -= U) {
        E xv[U], hv[U];
        float dz[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) load(max(k0 - u, 0), xv[u], dz[u], hv[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 - u < 0) break;
            const long long at = at0 + (k0 - u) * step;
            float xh[8];
            form(xv[u], hv[u], xh, dz[u]);
            if (dres) gn_store(dres + at, dz[u]);
#pragma unroll
            for (int j = 0; j < 8; ++j) xh[j] = rv[j] * (fmaf(dz[u][j], ga[j], -c1[j]) - xh[j] * c2[j]);
            gn_store(dx + at, xh);
        }
    }
}

inline int gn_gcd(int a, int b) { while (b) { const int r = a % b; a = b; b = r; } return a; }

// How a call is run: slices of S channels (whole groups, whole records) by workgroups of T threads, in one pass over registers (kind 1) or
// two passes (2), or all channels in chunks of rows by several launches (0).
struct Plan { int kind, S, T; bool few; };
// One pass where a slice of 64 or 128 bytes a row (a narrower one shares its cache lines with its neighbours) fits half a CU's threads at
// V records each, so that one workgroup's loads run beside another's stores; else two passes where there is a slice for every CU; else
// (few samples, large maps) chunks.  Measured, forward / forward with residual / backward with residual, microseconds:
//   bf16 256 x 56 x 56 x 256: one pass 242 / 307 / 684 (32-byte slices), two passes 218 / 266 / 609
//   bf16 128 x 28 x 28 x 512: one pass 47 / 67 / 139, two passes 64 / 81 / 155;  fp32 128 x 28 x 28 x 128: 23 / 28 / 52, 27 / 34 / 66
//   bf16 64 x 112 x 112 x 64 (128 slices): two passes 68 / 113 / 247, chunks 86 / 160 / 222
inline Plan gn_plan(int N, int HW, int C, int G, int size, bool bwd) {
    const int cpg = C / G, unit = cpg / gn_gcd(cpg, 8) * 8;     // lcm(cpg, 8)
    const int V = bwd ? (size == 2 ? RES_B16 : RES_B32) : (size == 2 ? RES_V16 : RES_V32);
    const int few = size == 2 ? RES_F16 : RES_F32;
    Plan best{0, 0, 0, false};
    int wide = 0;                                              // the widest slice up to 128 bytes (or the narrowest possible)
    for (int S = unit; S <= C; S += unit) {
        if (C % S) continue;
        if (wide && S * size > 128) break;
        // (a wider slice than 64 bytes only where workgroups are plenty: fp32 128 x 28 x 28 x 128 backward 40 against 44)
        if (wide * size >= 64 && (long long)N * (C / S) < (best.kind ? 1024 : 256)) break;
        wide = S;
        const int tpr = S >> 3, slots = bwd || cpg % 8 ? S : tpr;
        if (slots > 512 || (long long)(512 / tpr) * V < HW || (S * size < 64 && S < C && HW > 64)) continue;
        int T = 64;
        while ((long long)(T / tpr) * V < HW || slots > T) T *= 2;
        best.kind = 1; best.S = S; best.T = T;
        // rows of a few records a thread: leaner registers, more workgroups at a time
        while (T < 512 && (long long)(T / tpr) * few < HW && (long long)T * few < (long long)HW * tpr * 2) T *= 2;
        best.few = (long long)(T / tpr) * few >= HW && T <= 256;
        if (best.few) best.T = T;
    }
    if (best.kind == 0 && wide && (bwd || cpg % 8 ? wide : wide >> 3) <= STR_T && (long long)N * (C / wide) >= (bwd ? 256 : 128)) {
        best.kind = 2; best.S = wide; best.T = STR_T;
        while (best.T > 256 && (long long)(best.T >> 1) * 8 >= (long long)HW * (wide >> 3) && (bwd || cpg % 8 ? wide : wide >> 3) <= best.T >> 1)
            best.T >>= 1;                                      // (eight records a thread are enough)
    }
    if (best.kind && (long long)N * (C / best.S) > 0x7fffffffll) best.kind = 0;
    return best;
}

// rows per chunk: one register load per thread (RPT rows)
inline int gn_rows(int HW, int C) { return GN_T / (C >> 3) * GN_RPT; }
inline bool gn_bad(const void* x, int N, int HW, int C, int G) { return !x || N < 1 || HW < 1 || C < 1 || G < 1 || C % G != 0; }
// (rows are counted in 32 bits, a step of at most GN_T GN_RPT beyond the last: GN_MAXHW leaves room for it)
constexpr int GN_MAXHW = 1 << 30;
inline bool gn_limit(int N, int HW, int C) { return C % 8 != 0 || C > GN_MAXC || N > 65535 || HW > GN_MAXHW; }

}  // namespace

extern "C" {

size_t cfl_gn_ws_bytes(int N, int HW, int C, int G) {
    if (N < 1 || HW < 1 || C < 8 || G < 1 || C % G || gn_limit(N, HW, C)) return 0;
    const size_t chunks = cfl_cdiv(HW, gn_rows(HW, C));        // (also enough for the one-workgroup kernels: [N][2][C])
    return cfl_align256((size_t)N * chunks * G * 2 * 4) + cfl_align256((size_t)N * chunks * C * 2 * 4);      // (second: also the merged [2][N][G])
}

int cfl_gn_plan(int N, int HW, int C, int G, int dtype, int bwd) {
    if (N < 1 || HW < 1 || C < 8 || G < 1 || C % G || dtype < 0 || dtype > 1) return CFL_EINVAL;
    if (gn_limit(N, HW, C)) return CFL_ELIMIT;
    const Plan p = gn_plan(N, HW, C, G, dtype ? 2 : 4, bwd != 0);
    return p.kind | (p.kind && p.few ? 4 : 0) | (p.kind && !bwd && (C / G) % 8 ? 8 : 0) | (p.kind ? p.T << 4 : 0);
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
    const Plan p = gn_plan(N, HW, C, G, dtype ? 2 : 4, false);
    if (p.kind) {
        const int ng = (C / G) % 8 ? 8 : 1, gs = p.S / (C / G);
        size_t lds = (size_t)(16 + 2 * gs) * 4 + (size_t)p.T * ng * 8;
        int kl = 0;
        if (p.kind == 2) {                                     // (1024 threads have the CU's LDS for themselves, 512 half of it)
            lds = (lds + 15) / 16 * 16;
            const int rows = cfl_cdiv(HW, p.T / (p.S >> 3)) - (dtype ? STR_KEEP : 0), fit = ((160 * 1024 / STR_T) * p.T - (int)lds) / (p.T * (dtype ? 16 : 32));
            kl = rows < fit ? rows : fit;
            kl = kl > 0 ? kl : 0;
            lds += (size_t)kl * p.T * (dtype ? 16 : 32);
        }
        const dim3 rg((unsigned)(N * (C / p.S)));
#define GN_ONE(KERN, ...)                                                                                                                \
    do {                                                                                                                                 \
        CFL_SET_LDS(KERN, 160 * 1024);                                                                                                   \
        CFL_LAUNCH(K_GN_RES, KERN, rg, dim3(p.T), lds, stream, (const GE*)x, (const GE*)res, gamma, beta, HW, C, G, p.S, eps, act,       \
                   __VA_ARGS__ (GE*)y, mean, rstd);                                                                                      \
    } while (0)
#define GN_KIND(NG, VF, V)                                                                \
    do {                                                                                  \
        if (p.kind == 2) { GN_ONE((cfl_gn_str_fwd_kernel<GE, NG, 4, sizeof(GE) == 16 ? STR_KEEP : 0>), kl, ); } \
        else if (p.few) { GN_ONE((cfl_gn_res_fwd_kernel<GE, NG, VF>)); }                  \
        else { GN_ONE((cfl_gn_res_fwd_kernel<GE, NG, V>)); }                              \
    } while (0)
        if (dtype == 0) {
            typedef F8 GE;
            if (ng == 1) { GN_KIND(1, RES_F32, RES_V32); } else { GN_KIND(8, RES_F32, RES_V32); }
        } else {
            typedef U4 GE;
            if (ng == 1) { GN_KIND(1, RES_F16, RES_V16); } else { GN_KIND(8, RES_F16, RES_V16); }
        }
#undef GN_ONE
#undef GN_KIND
        return 0;
    }
    const int rows = gn_rows(HW, C);
    const dim3 grid(cfl_cdiv(HW, rows), N);
    float* part = (float*)ws;
    float* stats = (int)grid.x > GN_MERGE ? (float*)((char*)ws + cfl_align256((size_t)N * grid.x * G * 2 * 4)) : nullptr;
#define GN_FWD(E, A, R)                                                                                                               \
    CFL_LAUNCH(K_GN_APPLY, (cfl_gn_apply_kernel<E, A, R>), grid, dim3(GN_T), 0, stream, (const E*)x, (const E*)res, gamma, beta, part, \
               HW, C, G, rows, eps, (E*)y, mean, rstd, stats)
    if (dtype == 0) {
        CFL_LAUNCH(K_GN_STATS, cfl_gn_stats_kernel<F8>, grid, dim3(GN_T), 0, stream, (const F8*)x, HW, C, G, rows, part);
    } else {
        CFL_LAUNCH(K_GN_STATS, cfl_gn_stats_kernel<U4>, grid, dim3(GN_T), 0, stream, (const U4*)x, HW, C, G, rows, part);
    }
    if (stats)
        CFL_LAUNCH(K_GN_STATS, cfl_gn_merge_kernel, dim3(N), dim3(1024), 0, stream, part, (int)grid.x, rows, HW, C / G, G, eps, stats);
    if (dtype == 0) { GN_SWITCH(F8, GN_FWD); } else { GN_SWITCH(U4, GN_FWD); }
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
    const Plan p = gn_plan(N, HW, C, G, dtype ? 2 : 4, true);
    if (p.kind) {
        const int rpp = p.T / (p.S >> 3);
        const size_t lds = (size_t)2 * (p.S / (C / G) + p.S + rpp * p.S) * 4;
        const dim3 rg((unsigned)(N * (C / p.S)));
        float* pcr = (float*)ws;
#define GN_ONE(KERN)                                                                                                                    \
    do {                                                                                                                                \
        CFL_SET_LDS(KERN, 96 * 1024);                                                                                                   \
        CFL_LAUNCH(K_GN_RES, KERN, rg, dim3(p.T), lds, stream, (const GE*)x, (const GE*)dy, (const GE*)dy2, (const GE*)res, gamma, beta, \
                   mean, rstd, HW, C, G, p.S, act, (GE*)dx, want_dres ? (GE*)dres : (GE*)nullptr, pcr);                                 \
    } while (0)
#define GN_KIND(VF, V)                                                                    \
    do {                                                                                  \
        if (p.kind == 2) { GN_ONE((cfl_gn_str_bwd_kernel<GE, 2>)); }                      \
        else if (p.few) { GN_ONE((cfl_gn_res_bwd_kernel<GE, VF>)); }                      \
        else { GN_ONE((cfl_gn_res_bwd_kernel<GE, V>)); }                                  \
    } while (0)
        if (dtype == 0) { typedef F8 GE; GN_KIND(RES_F32, RES_B32); } else { typedef U4 GE; GN_KIND(RES_F16, RES_B16); }
#undef GN_ONE
#undef GN_KIND
        CFL_LAUNCH(K_GN_BWD_FINAL, cfl_gn_bwd_final_kernel, dim3(cfl_cdiv(C, 16)), dim3(1024), 0, stream, pcr, N, C, dgamma, dbeta);
        return 0;
    }
    const int rows = gn_rows(HW, C), chunks = cfl_cdiv(HW, rows);
    const dim3 grid(chunks, N);
    float* pg = (float*)ws;
    float* pc = (float*)((char*)ws + cfl_align256((size_t)N * chunks * G * 2 * 4));
    const int sums = chunks > GN_MERGE ? 1 : chunks;
#define GN_BWD(E, A, R)                                                                                                                 \
    CFL_LAUNCH(K_GN_BWD_REDUCE, (cfl_gn_bwd_reduce_kernel<E, A, R>), grid, dim3(GN_T), 0, stream, (const E*)x, (const E*)dy,            \
               (const E*)dy2, (const E*)res, gamma, beta, mean, rstd, HW, C, G, rows, pc, pg);                                          \
    if (chunks > GN_MERGE) CFL_LAUNCH(K_GN_BWD_REDUCE, cfl_gn_bwd_merge_kernel, dim3(G, N), dim3(64), 0, stream, pg, chunks, G);        \
    CFL_LAUNCH(K_GN_BWD_APPLY, (cfl_gn_bwd_apply_kernel<E, A, R>), grid, dim3(GN_T), 0, stream, (const E*)x, (const E*)dy,              \
               (const E*)dy2, (const E*)res, gamma, beta, mean, rstd, pg, HW, C, G, rows, sums, (E*)dx, want_dres ? (E*)dres : (E*)nullptr)
    if (dtype == 0) { GN_SWITCH(F8, GN_BWD); } else { GN_SWITCH(U4, GN_BWD); }
#undef GN_BWD
    CFL_LAUNCH(K_GN_BWD_FINAL, cfl_gn_bwd_final_kernel, dim3(cfl_cdiv(C, 16)), dim3(1024), 0, stream, pc, N * chunks, C, dgamma, dbeta);
    return 0;
}

}  // extern "C"
