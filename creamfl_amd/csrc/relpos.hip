// relpos.hip -- self-attention with a learned relative position bias by buckets, head dim 64, any length; forward and backward.
//
//   s_ij = scale q_i . k_j + table[bucket[clip(j - i, -R, R) + R]][h]   (keys that the mask drops: -inf),  p = softmax_j(s),  o_i = sum_j p_ij v_j
//   backward: D_i = sum_d do_id o_id,  ds_ij = p_ij (do_i . v_j - D_i),  dv_j = sum_i p_ij do_i,  dq_i = scale sum_j ds_ij k_j,
//             dk_j = scale sum_i ds_ij q_i,  dtable[b][h] = sum of ds_ij over all texts and pairs (i, j) whose bucket is b
//   A row whose mask leaves no key has o = 0 and no gradient.
//
// Where it sits: the text tower at src/networks/models/pcme.py:36-44, with distances in place of that BERT's absolute positions.
// The bias depends on j - i alone, so a head's bias is a vector over distances: it is expanded into LDS once per workgroup, and tiles
// whose distances all lie beyond R take one constant.  dtable's sums run over diagonals; see the dQ kernel.
// Nothing of size L x L reaches memory: one pass over the keys with the running maximum and sum of the softmax (in units of log2);
// the backward recomputes p from the row's log-sum.  dQ (a wave owns queries) and dK / dV (a wave owns keys) are separate kernels, so
// no gradient is accumulated by atomics across workgroups: results are the same bits on every run.
//
// Matrix instructions: v_mfma_f32_32x32x16_bf16; scores are formed TRANSPOSED (S^T = K Q^T) where a wave owns queries, so a lane owns
// one query and its keys sit in the lane's registers; registers 8 kk .. 8 kk + 7 are then, packed to bf16, the second operand of the
// following product (o^T = V^T P^T) whose first operand is read transposed out of LDS in the same key order (ds_read_b64_tr_b16).
// P and ds are rounded to bf16 there (2^-9 relative, the precision of v and k themselves); sums stay in 32 bits.
#include "common.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16;
typedef unsigned int u32;
typedef unsigned long long u64;

constexpr int TP = 72;                      // LDS row pitch in bf16 (144 bytes: 16-byte rows and both kinds of reads spread over the banks)
constexpr int KT = 64;                      // rows of a staged tile
constexpr int BPAD = 64;                    // the bias vector reaches this far beyond +-R: a tile that touches |d| <= R needs no clipping
constexpr int MAXR = 512;                   // largest R (LDS)
constexpr float LOG2E = 1.4426950408889634f;

struct RpArgs {
    const u16 *q, *k, *v, *o, *dout;        // element (row, h * 64 + d) of a text's rows: base + row * ld + ...
    long long ldq, ldk, ldo;                // row strides of q / (k, v) / (o, dout)
    u16 *out, *dq, *dk, *dv;
    long long lddq, lddk;
    const unsigned char* mask;              // [B][Lk] key mask (non-zero = takes part) or NULL
    const int* cu;                          // packed form: text b = rows cu[b] .. cu[b + 1] - 1 of [T] rows; NULL = padded
    int B, Lq, Lk, T, heads;                // Lq = 0: the queries are the packed rows themselves; Lk: (about) the longest text
    float scale2;                           // scale * log2(e)
    float scale;
    const void* table;                      // [nb][heads]
    int table_bf16, nb, R;
    const int* bucket;                      // [2 R + 1]
    float* lse;                             // [heads][rows]: log2-sum of a row's scores (+inf: no key)
    float* dsum;                            // [heads][rows]: D
    float* diag;                            // [heads][slots][2 Rr + 1]
    int Rr;                                 // min(R, longest distance): distances that occur
    int nqb;                                // query blocks of the longest text
    long long rows;                         // query rows in all (B Lq or T)
};

// rows of text b
struct Text { long long q0, k0; int lq, lk; };
__device__ __forceinline__ Text text_of(const RpArgs& a, int b) {
    Text t;
    if (a.cu) {
        const int r0 = min(max(a.cu[b], 0), a.T), r1 = min(max(a.cu[b + 1], r0), a.T);
        t.k0 = r0; t.lk = r1 - r0;
        t.q0 = a.Lq ? (long long)b * a.Lq : r0; t.lq = a.Lq ? a.Lq : t.lk;
    } else {
        t.q0 = (long long)b * a.Lq; t.k0 = (long long)b * a.Lk; t.lq = a.Lq; t.lk = a.Lk;
    }
    return t;
}

__device__ __forceinline__ int acc_r(int r, int lane) { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }
__device__ __forceinline__ void zero16(f32x16& a) {
#pragma unroll
    for (int r = 0; r < 16; ++r) a[r] = 0.f;
}
__device__ __forceinline__ u32 pack2(float a, float b) {
    union { __bf16 h[2]; u32 u; } x;
    x.h[0] = (__bf16)a; x.h[1] = (__bf16)b;
    return x.u;
}
__device__ __forceinline__ bf16x8 pack_acc(const f32x16& a, int kk) {
    f32x4 v;
#pragma unroll
    for (int t = 0; t < 4; ++t) v[t] = __uint_as_float(pack2(a[8 * kk + 2 * t], a[8 * kk + 2 * t + 1]));
    return __builtin_bit_cast(bf16x8, v);
}
// operand whose lane owns row `row0 + (lane & 31)` of a staged tile, contraction over d: 16 kk + 8 (lane >> 5) .. + 7
__device__ __forceinline__ bf16x8 frag_rows(const u16* t, int row0, int kk, int lane) {
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const f32x4*>(t + (row0 + (lane & 31)) * TP + kk * 16 + (lane >> 5) * 8));
}
// operand whose lane owns column 32 dt + (lane & 31) of a staged tile, contraction over rows in the accumulators' order:
// row0 + 4 (lane >> 5) + {0..3} and + 8 (a 16-lane group's transposing read takes a [4 rows x 16 columns] block)
__device__ __forceinline__ bf16x8 frag_cols(const u16* t, int row0, int dt, int lane) {
    const int p = lane & 15, g = lane >> 4;
    const u16* a = t + (row0 + 4 * (g >> 1) + (p >> 2)) * TP + 32 * dt + 16 * (g & 1) + 4 * (p & 3);
    union { s16x4 h[2]; bf16x8 v; } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 8 * TP));
    return u.v;
}
// a wave's 32 rows straight from memory as an operand (rows >= n repeat the last one: their results are not used)
__device__ __forceinline__ void load_rows(const u16* base, long long ld, int row0, int n, int lane, bf16x8 (&f)[4]) {
    const int r = min(row0 + (lane & 31), n - 1);
    const u16* p = base + (long long)r * ld + (lane >> 5) * 8;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) f[kk] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const f32x4*>(p + kk * 16));
}
// rows r0 .. r0 + 63 of a [n][64] matrix into a tile; rows >= n and rows whose keep flag is 0 become zeros (whatever stands there,
// infinities and NaN included, must not reach a product)
template <int NT>
__device__ __forceinline__ void stage(const u16* base, long long ld, int r0, int n, const unsigned char* keep, u16* tile) {
#pragma unroll
    for (int it = 0; it < KT * 8 / NT; ++it) {
        const int c = it * NT + threadIdx.x, row = c >> 3, cc = c & 7;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (r0 + row < n && (!keep || keep[r0 + row])) v = *reinterpret_cast<const f32x4*>(base + (long long)(r0 + row) * ld + cc * 8);
        *reinterpret_cast<f32x4*>(tile + row * TP + cc * 8) = v;
    }
}
// the 64 keep flags of keys k0 .. k0 + 63
__device__ __forceinline__ u64 key_bits(const unsigned char* mask, int k0, int lk, int lane) {
    const int j = k0 + lane;
    return __ballot(j < lk && (!mask || mask[j]));
}
// head h's bias over distances, in units of log2: bl[d + R + BPAD], |d| <= R + BPAD
template <int NT>
__device__ __forceinline__ void fill_bias(const RpArgs& a, int h, float* bl) {
    for (int i = threadIdx.x; i < 2 * (a.R + BPAD) + 1; i += NT) {
        const int d = min(max(i - BPAD, 0), 2 * a.R);
        const int b = min(max(a.bucket[d], 0), a.nb - 1);
        const float t = a.table_bf16 ? __uint_as_float((u32)((const u16*)a.table)[(long long)b * a.heads + h] << 16)
                                     : ((const float*)a.table)[(long long)b * a.heads + h];
        bl[i] = t * LOG2E;
    }
}
// bias of a 32 x 32 block: distances key - query with d0 = (first key) - (first query); near = the block touches |d| < R
struct BlockBias { bool near; float c; const float* p; };
template <bool KEY_LANE>
__device__ __forceinline__ BlockBias block_bias(const float* bl, int R, int d0, int lane) {
    BlockBias x;
    x.near = d0 - 31 < R && d0 + 31 > -R;
    x.c = bl[(d0 > 0 ? R : -R) + R + BPAD];
    // lane = query: d = d0 + key - lane, key = acc_r; lane = key: d = d0 + lane - query, query = acc_r
    x.p = bl + R + BPAD + (x.near ? d0 : 0) + (KEY_LANE ? (lane & 31) - 4 * (lane >> 5) : 4 * (lane >> 5) - (lane & 31));
    return x;
}

// ---- forward.  A wave owns 32 queries of one (text, head); NW waves share the staged keys.
template <int NW>
__global__ __launch_bounds__(NW * 64) void cfl_relpos_fwd_kernel(RpArgs a) {
    constexpr int NT = NW * 64;
    __shared__ __attribute__((aligned(16))) u16 Kt[KT * TP], Vt[KT * TP];
    extern __shared__ float bl[];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int qb = id % a.nqb, h = (id / a.nqb) % a.heads, b = id / (a.nqb * a.heads);
    const Text t = text_of(a, b);
    fill_bias<NT>(a, h, bl);
    const unsigned char* mask = a.mask ? a.mask + (long long)b * a.Lk : nullptr;
    const u16* kp = a.k + t.k0 * a.ldk + h * 64;
    const u16* vp = a.v + t.k0 * a.ldk + h * 64;
    for (int blk = qb; blk * NW * 32 < t.lq; blk += a.nqb) {
        const int q0 = blk * NW * 32 + w * 32;
        bf16x8 qf[4];
        load_rows(a.q + t.q0 * a.ldq + h * 64, a.ldq, q0, t.lq, lane, qf);
        f32x16 o[2];
        zero16(o[0]); zero16(o[1]);
        float m = -INFINITY, l = 0.f;
        for (int k0 = 0; k0 < t.lk; k0 += KT) {
            const u64 bits = key_bits(mask, k0, t.lk, lane);
            if (bits == 0) continue;                           // (the same for every wave of the workgroup)
            __syncthreads();
            stage<NT>(kp, a.ldk, k0, t.lk, mask, Kt);
            stage<NT>(vp, a.ldk, k0, t.lk, mask, Vt);
            __syncthreads();
            f32x16 s[2];
            float top = m;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                zero16(s[u]);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows(Kt, 32 * u, kk, lane), qf[kk], s[u], 0, 0, 0);
                const BlockBias bb = block_bias<false>(bl, a.R, k0 + 32 * u - q0, lane);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float bias = bb.near ? bb.p[(r & 3) + 8 * (r >> 2)] : bb.c;
                    const float v = fmaf(s[u][r], a.scale2, bias);
                    s[u][r] = (bits >> (32 * u + acc_r(r, lane))) & 1 ? v : -INFINITY;
                    top = fmaxf(top, s[u][r]);
                }
            }
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float shrink = m == -INFINITY ? 0.f : exp2f(m - top);
            l *= shrink;
#pragma unroll
            for (int r = 0; r < 16; ++r) { o[0][r] *= shrink; o[1][r] *= shrink; }
            m = top;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[u][r] = exp2f(s[u][r] - m);
                    l += s[u][r];
                }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const bf16x8 p = pack_acc(s[u], kk);
#pragma unroll
                    for (int dt = 0; dt < 2; ++dt)
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_cols(Vt, 32 * u + 16 * kk, dt, lane), p, o[dt], 0, 0, 0);
                }
        }
        l += __shfl_xor(l, 32, 64);
        const int row = q0 + (lane & 31);
        if (row < t.lq) {
            const float inv = m == -INFINITY ? 0.f : 1.f / l;
            u16* op = a.out + (t.q0 + row) * a.ldo + h * 64 + 4 * (lane >> 5);
#pragma unroll
            for (int dt = 0; dt < 2; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint2 v;
                    v.x = pack2(o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv);
                    v.y = pack2(o[dt][4 * g + 2] * inv, o[dt][4 * g + 3] * inv);
                    *reinterpret_cast<uint2*>(op + 32 * dt + 8 * g) = v;
                }
            if (a.lse && lane < 32) a.lse[h * a.rows + t.q0 + row] = m == -INFINITY ? INFINITY : m + log2f(l);
        }
    }
}

// rows behind the last text of a packed batch: zeros (grid-stride over 16-byte pieces of `width` bf16 per row)
__global__ __launch_bounds__(256) void cfl_relpos_tail_kernel(const int* __restrict__ cu, int B, int T, u16* p, long long ld, int width) {
    const int r0 = min(max(cu[B], 0), T), per = width / 8;
    const long long n = (long long)(T - r0) * per;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
        *reinterpret_cast<f32x4*>(p + (r0 + i / per) * ld + (i % per) * 8) = z;
    }
}

// ---- backward, queries: D, dQ and the bias gradient.  Same ownership as the forward.
// The bias gradient of a distance is the sum of ds along a diagonal.  A lane's 16 values of a near block lie on 16 diagonals: each wave
// adds them to LDS words of its own, one word per distance and lane half -- the addresses of one instruction are distinct and a wave's
// LDS operations stay in order, so the sum's order is fixed.  Far blocks are summed in registers.
template <int NW>
__global__ __launch_bounds__(NW * 64) void cfl_relpos_dq_kernel(RpArgs a) {
    constexpr int NT = NW * 64;
    __shared__ __attribute__((aligned(16))) u16 Kt[KT * TP], Vt[KT * TP];
    extern __shared__ float dyn[];
    const int nd = 2 * (a.R + BPAD) + 1;
    float* bl = dyn;
    float* dg = dyn + nd;                                      // [2 NW][nd]
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int qb = id % a.nqb, h = (id / a.nqb) % a.heads, b = id / (a.nqb * a.heads);
    const Text t = text_of(a, b);
    fill_bias<NT>(a, h, bl);
    for (int i = threadIdx.x; i < 2 * NW * nd; i += NT) dg[i] = 0.f;
    float far_lo = 0.f, far_hi = 0.f;
    float* mine = dg + (2 * w + (lane >> 5)) * nd;
    const unsigned char* mask = a.mask ? a.mask + (long long)b * a.Lk : nullptr;
    const u16* kp = a.k + t.k0 * a.ldk + h * 64;
    const u16* vp = a.v + t.k0 * a.ldk + h * 64;
    __syncthreads();
    for (int blk = qb; blk * NW * 32 < t.lq; blk += a.nqb) {
        const int q0 = blk * NW * 32 + w * 32;
        const int row = q0 + (lane & 31);
        const bool live = row < t.lq;
        bf16x8 qf[4], gf[4];
        load_rows(a.q + t.q0 * a.ldq + h * 64, a.ldq, q0, t.lq, lane, qf);
        load_rows(a.dout + t.q0 * a.ldo + h * 64, a.ldo, q0, t.lq, lane, gf);
        float D = 0.f;
        {
            bf16x8 of[4];
            load_rows(a.o + t.q0 * a.ldo + h * 64, a.ldo, q0, t.lq, lane, of);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                for (int j = 0; j < 8; ++j) D = fmaf((float)of[kk][j], (float)gf[kk][j], D);
            D += __shfl_xor(D, 32, 64);
        }
        const float lse = live ? a.lse[h * a.rows + t.q0 + row] : INFINITY;
        if (live && lane < 32) a.dsum[h * a.rows + t.q0 + row] = D;
        f32x16 dq[2];
        zero16(dq[0]); zero16(dq[1]);
        for (int k0 = 0; k0 < t.lk; k0 += KT) {
            const u64 bits = key_bits(mask, k0, t.lk, lane);
            if (bits == 0) continue;
            __syncthreads();
            stage<NT>(kp, a.ldk, k0, t.lk, mask, Kt);
            stage<NT>(vp, a.ldk, k0, t.lk, mask, Vt);
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                f32x16 s, dp;
                zero16(s); zero16(dp);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows(Kt, 32 * u, kk, lane), qf[kk], s, 0, 0, 0);
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows(Vt, 32 * u, kk, lane), gf[kk], dp, 0, 0, 0);
                }
                const int d0 = k0 + 32 * u - q0;
                const BlockBias bb = block_bias<false>(bl, a.R, d0, lane);
                float* dst = mine + (bb.p - bl);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float bias = bb.near ? bb.p[(r & 3) + 8 * (r >> 2)] : bb.c;
                    const bool ok = live && ((bits >> (32 * u + acc_r(r, lane))) & 1);
                    const float p = ok ? exp2f(fmaf(s[r], a.scale2, bias) - lse) : 0.f;
                    s[r] = p == 0.f ? 0.f : p * (dp[r] - D);
                }
                if (bb.near) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        __hip_atomic_fetch_add(dst + (r & 3) + 8 * (r >> 2), s[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                } else {
                    float x = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) x += s[r];
                    if (d0 > 0) far_hi += x; else far_lo += x;
                }
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const bf16x8 p = pack_acc(s, kk);
#pragma unroll
                    for (int dt = 0; dt < 2; ++dt)
                        dq[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_cols(Kt, 32 * u + 16 * kk, dt, lane), p, dq[dt], 0, 0, 0);
                }
            }
        }
        if (live) {
            u16* op = a.dq + (t.q0 + row) * a.lddq + h * 64 + 4 * (lane >> 5);
#pragma unroll
            for (int dt = 0; dt < 2; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint2 v;
                    v.x = pack2(dq[dt][4 * g] * a.scale, dq[dt][4 * g + 1] * a.scale);
                    v.y = pack2(dq[dt][4 * g + 2] * a.scale, dq[dt][4 * g + 3] * a.scale);
                    *reinterpret_cast<uint2*>(op + 32 * dt + 8 * g) = v;
                }
        }
    }
    // the workgroup's sums per distance, clipped to +-Rr
    far_lo = wave_sum(far_lo);
    far_hi = wave_sum(far_hi);
    if (lane == 0) {                                           // (distances at the vector's ends belong to +-R as well)
        dg[2 * w * nd] += far_lo;
        dg[2 * w * nd + nd - 1] += far_hi;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nd; i += NT) {
        float x = 0.f;
#pragma unroll
        for (int c = 0; c < 2 * NW; ++c) x += dg[c * nd + i];
        dg[i] = x;                                             // (read above by this thread alone)
    }
    __syncthreads();
    float* out = a.diag + ((long long)h * a.B * a.nqb + (long long)b * a.nqb + qb) * (2 * a.Rr + 1);
    const int mid = a.R + BPAD;
    for (int i = threadIdx.x; i < 2 * a.Rr + 1; i += NT) {
        float x = dg[mid - a.Rr + i];
        if (i == 0) for (int j = mid - a.Rr - 1; j >= 0; --j) x += dg[j];
        if (i == 2 * a.Rr) for (int j = mid + a.Rr + 1; j < nd; ++j) x += dg[j];
        out[i] = x;
    }
}

// ---- backward, keys: dK and dV.  A wave owns 32 keys; the staged rows are queries.
template <int NW>
__global__ __launch_bounds__(NW * 64) void cfl_relpos_dkv_kernel(RpArgs a, int nkb) {
    constexpr int NT = NW * 64;
    __shared__ __attribute__((aligned(16))) u16 Qt[KT * TP], Gt[KT * TP];
    __shared__ float ls[KT], ds[KT];
    extern __shared__ float bl[];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int kb = id % nkb, h = (id / nkb) % a.heads, b = id / (nkb * a.heads);
    const Text t = text_of(a, b);
    fill_bias<NT>(a, h, bl);
    const unsigned char* mask = a.mask ? a.mask + (long long)b * a.Lk : nullptr;
    const u16* qp = a.q + t.q0 * a.ldq + h * 64;
    const u16* gp = a.dout + t.q0 * a.ldo + h * 64;
    for (int blk = kb; blk * NW * 32 < t.lk; blk += nkb) {
        const int k0 = blk * NW * 32 + w * 32;
        const int key = k0 + (lane & 31);
        const bool live = key < t.lk && (!mask || mask[key]);
        bf16x8 kf[4], vf[4];
        load_rows(a.k + t.k0 * a.ldk + h * 64, a.ldk, k0, t.lk, lane, kf);
        load_rows(a.v + t.k0 * a.ldk + h * 64, a.ldk, k0, t.lk, lane, vf);
        f32x16 dk[2], dv[2];
        zero16(dk[0]); zero16(dk[1]); zero16(dv[0]); zero16(dv[1]);
        for (int q0 = 0; q0 < t.lq; q0 += KT) {
            __syncthreads();
            stage<NT>(qp, a.ldq, q0, t.lq, nullptr, Qt);
            stage<NT>(gp, a.ldo, q0, t.lq, nullptr, Gt);
            for (int i = threadIdx.x; i < KT; i += NT) {
                const bool in = q0 + i < t.lq;
                ls[i] = in ? a.lse[h * a.rows + t.q0 + q0 + i] : INFINITY;
                ds[i] = in ? a.dsum[h * a.rows + t.q0 + q0 + i] : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                f32x16 s, dp;
                zero16(s); zero16(dp);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows(Qt, 32 * u, kk, lane), kf[kk], s, 0, 0, 0);
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_rows(Gt, 32 * u, kk, lane), vf[kk], dp, 0, 0, 0);
                }
                const BlockBias bb = block_bias<true>(bl, a.R, k0 - q0 - 32 * u, lane);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int i = 32 * u + acc_r(r, lane);
                    const float bias = bb.near ? bb.p[-((r & 3) + 8 * (r >> 2))] : bb.c;
                    const float p = live ? exp2f(fmaf(s[r], a.scale2, bias) - ls[i]) : 0.f;
                    s[r] = p;
                    dp[r] = p == 0.f ? 0.f : p * (dp[r] - ds[i]);
                }
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const bf16x8 p = pack_acc(s, kk), g = pack_acc(dp, kk);
#pragma unroll
                    for (int dt = 0; dt < 2; ++dt) {
                        dv[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_cols(Gt, 32 * u + 16 * kk, dt, lane), p, dv[dt], 0, 0, 0);
                        dk[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag_cols(Qt, 32 * u + 16 * kk, dt, lane), g, dk[dt], 0, 0, 0);
                    }
                }
            }
        }
        if (key < t.lk) {
            u16* kq = a.dk + (t.k0 + key) * a.lddk + h * 64 + 4 * (lane >> 5);
            u16* vq = a.dv + (t.k0 + key) * a.lddk + h * 64 + 4 * (lane >> 5);
#pragma unroll
            for (int dt = 0; dt < 2; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint2 v;
                    v.x = live ? pack2(dk[dt][4 * g] * a.scale, dk[dt][4 * g + 1] * a.scale) : 0u;
                    v.y = live ? pack2(dk[dt][4 * g + 2] * a.scale, dk[dt][4 * g + 3] * a.scale) : 0u;
                    *reinterpret_cast<uint2*>(kq + 32 * dt + 8 * g) = v;
                    v.x = live ? pack2(dv[dt][4 * g], dv[dt][4 * g + 1]) : 0u;
                    v.y = live ? pack2(dv[dt][4 * g + 2], dv[dt][4 * g + 3]) : 0u;
                    *reinterpret_cast<uint2*>(vq + 32 * dt + 8 * g) = v;
                }
        }
    }
}

// ---- dtable[bucket][h]: the sums of the bucket's distances over all workgroups of the dQ kernel, in a fixed order.  grid = (nb, heads)
__global__ __launch_bounds__(256) void cfl_relpos_dtable_kernel(const float* __restrict__ diag, const int* __restrict__ bucket, int R, int Rr,
                                                                int nb, int heads, long long slots, void* dtable, int bf16) {
    __shared__ float red[4];
    const int b = blockIdx.x, h = blockIdx.y, nd = 2 * Rr + 1;
    float x = 0.f;
    for (int i = 0; i < nd; ++i) {
        if (min(max(bucket[R - Rr + i], 0), nb - 1) != b) continue;
        for (long long s = threadIdx.x; s < slots; s += 256) x += diag[(h * slots + s) * nd + i];
    }
    x = block_sum_256(x, red);
    if (threadIdx.x == 0) {
        if (bf16) ((__bf16*)dtable)[b * heads + h] = (__bf16)x;
        else ((float*)dtable)[b * heads + h] = x;
    }
}

// waves per workgroup: texts of at most one wave's rows get workgroups of one wave
inline int rp_waves(int L) { return L <= 32 ? 1 : 4; }
inline int rp_blocks(int L) { return cfl_cdiv(L, 32 * rp_waves(L)); }

// distances that can occur, at most R (packed texts: whatever their lengths are)
inline int rp_reach(int Lq, int Lk, int T, int R) {
    const int far = (T > 0 ? (T > Lq ? T : Lq) : (Lq > Lk ? Lq : Lk)) - 1;
    return R < far ? R : far;
}

inline int rp_check(const RpArgs& a, int head_dim) {
    if (!a.q || !a.k || !a.v || !a.table || !a.bucket || a.B < 1 || a.Lq < 0 || a.Lk < 1 || a.heads < 1 || a.nb < 1 || a.R < 0 ||
        (a.cu ? a.T < 1 || a.mask != nullptr : a.Lq < 1)) return CFL_EINVAL;
    if (a.ldq % 8 || a.ldk % 8 || a.ldo % 8 || (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v) & 15)) return CFL_EALIGN;
    if (head_dim != 64 || a.R > MAXR || a.heads > 65535 || a.nb > 65535 ||
        (long long)a.B * a.heads * rp_blocks(a.Lq > a.Lk ? a.Lq : a.Lk) > 0x7fffffffll) return CFL_ELIMIT;
    return 0;
}

}  // namespace

extern "C" {

size_t cfl_relpos_ws_bytes(int B, int Lq, int Lk, int T, int heads, int R) {
    if (B < 1 || Lq < 0 || Lk < 1 || T < 0 || (Lq == 0 && T == 0) || heads < 1 || R < 0 || R > MAXR) return 0;
    return (size_t)B * heads * rp_blocks(Lq ? Lq : Lk) * (2 * rp_reach(Lq, Lk, T, R) + 1) * 4;
}

int cfl_relpos_fwd(const void* q, long long ldq, const void* k, const void* v, long long ldk, const unsigned char* mask, const int* cu,
                   int B, int Lq, int Lk, int T, int heads, int head_dim, float scale, const void* table, int table_bf16, int nb,
                   const int* bucket, int R, void* o, long long ldo, float* lse, void* stream_) {
    RpArgs a{};
    a.q = (const u16*)q; a.k = (const u16*)k; a.v = (const u16*)v; a.ldq = ldq; a.ldk = ldk; a.ldo = ldo; a.out = (u16*)o;
    a.mask = mask; a.cu = cu; a.B = B; a.Lq = Lq; a.Lk = Lk; a.T = T; a.heads = heads; a.scale = scale; a.scale2 = scale * LOG2E;
    a.table = table; a.table_bf16 = table_bf16; a.nb = nb; a.R = R; a.bucket = bucket; a.lse = lse;
    a.rows = Lq ? (long long)B * Lq : T;
    const int rc = rp_check(a, head_dim);
    if (rc) return rc;
    if (!o) return CFL_EINVAL;
    if ((uintptr_t)o & 15) return CFL_EALIGN;
    hipStream_t stream = (hipStream_t)stream_;
    const int L = Lq ? Lq : Lk;
    a.nqb = rp_blocks(L);
    const dim3 grid((unsigned)(B * heads * a.nqb));
    const size_t lds = (2 * (R + BPAD) + 1) * 4;
    if (rp_waves(L) == 1) { CFL_LAUNCH(K_RELPOS_FWD, cfl_relpos_fwd_kernel<1>, grid, dim3(64), lds, stream, a); }
    else { CFL_LAUNCH(K_RELPOS_FWD, cfl_relpos_fwd_kernel<4>, grid, dim3(256), lds, stream, a); }
    if (cu && !Lq) CFL_LAUNCH(K_RELPOS_TAIL, cfl_relpos_tail_kernel, dim3(64), dim3(256), 0, stream, cu, B, T, (u16*)o, ldo, heads * 64);
    return 0;
}

int cfl_relpos_bwd(const void* q, long long ldq, const void* k, const void* v, long long ldk, const unsigned char* mask, const int* cu,
                   int B, int Lq, int Lk, int T, int heads, int head_dim, float scale, const void* table, int table_bf16, int nb,
                   const int* bucket, int R, const void* o, const void* dout, long long ldo, const float* lse, float* dsum, void* dq,
                   long long lddq, void* dk, void* dv, long long lddk, void* dtable, void* ws, void* stream_) {
    RpArgs a{};
    a.q = (const u16*)q; a.k = (const u16*)k; a.v = (const u16*)v; a.ldq = ldq; a.ldk = ldk; a.ldo = ldo;
    a.o = (const u16*)o; a.dout = (const u16*)dout; a.dq = (u16*)dq; a.dk = (u16*)dk; a.dv = (u16*)dv; a.lddq = lddq; a.lddk = lddk;
    a.mask = mask; a.cu = cu; a.B = B; a.Lq = Lq; a.Lk = Lk; a.T = T; a.heads = heads; a.scale = scale; a.scale2 = scale * LOG2E;
    a.table = table; a.table_bf16 = table_bf16; a.nb = nb; a.R = R; a.bucket = bucket; a.lse = const_cast<float*>(lse); a.dsum = dsum;
    a.rows = Lq ? (long long)B * Lq : T;
    const int rc = rp_check(a, head_dim);
    if (rc) return rc;
    if (!o || !dout || !lse || !dsum || !dq || !dk || !dv || !dtable || !ws) return CFL_EINVAL;
    if (lddq % 8 || lddk % 8 || (((uintptr_t)o | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15)) return CFL_EALIGN;
    hipStream_t stream = (hipStream_t)stream_;
    const int L = Lq ? Lq : Lk;
    a.Rr = rp_reach(Lq, Lk, cu ? T : 0, R);
    a.diag = (float*)ws;
    a.nqb = rp_blocks(L);
    const int nkb = rp_blocks(Lk), nd = 2 * (R + BPAD) + 1;
    const dim3 gq((unsigned)(B * heads * a.nqb)), gk((unsigned)(B * heads * nkb));
    if (rp_waves(L) == 1) { CFL_LAUNCH(K_RELPOS_DQ, cfl_relpos_dq_kernel<1>, gq, dim3(64), (size_t)nd * 3 * 4, stream, a); }
    else { CFL_LAUNCH(K_RELPOS_DQ, cfl_relpos_dq_kernel<4>, gq, dim3(256), (size_t)nd * 9 * 4, stream, a); }
    if (rp_waves(Lk) == 1) { CFL_LAUNCH(K_RELPOS_DKV, cfl_relpos_dkv_kernel<1>, gk, dim3(64), (size_t)nd * 4, stream, a, nkb); }
    else { CFL_LAUNCH(K_RELPOS_DKV, cfl_relpos_dkv_kernel<4>, gk, dim3(256), (size_t)nd * 4, stream, a, nkb); }
    CFL_LAUNCH(K_RELPOS_DTABLE, cfl_relpos_dtable_kernel, dim3(nb, heads), dim3(256), 0, stream, a.diag, bucket, R, a.Rr, nb, heads,
               (long long)B * a.nqb, dtable, table_bf16);
    if (cu) {
        if (!Lq) CFL_LAUNCH(K_RELPOS_TAIL, cfl_relpos_tail_kernel, dim3(64), dim3(256), 0, stream, cu, B, T, (u16*)dq, lddq, heads * 64);
        CFL_LAUNCH(K_RELPOS_TAIL, cfl_relpos_tail_kernel, dim3(64), dim3(256), 0, stream, cu, B, T, (u16*)dk, lddk, heads * 64);
        CFL_LAUNCH(K_RELPOS_TAIL, cfl_relpos_tail_kernel, dim3(64), dim3(256), 0, stream, cu, B, T, (u16*)dv, lddk, heads * 64);
    }
    return 0;
}

}  // extern "C"
