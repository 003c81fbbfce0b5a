// relpos.hip -- self-attention with a learned relative position bias by buckets, head dim 64, any length; forward and backward.
//
//   s_ij = scale q_i . k_j + table[bucket[clip(j - i, -R, R) + R]][h]   (keys that the mask drops, or whose bias is -1e30 or less: -inf),  p = softmax_j(s),  o_i = sum_j p_ij v_j
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
// P and ds are rounded to bf16 there (by up to 2^-8 relative, as v and k are): o is then 2.3e-3 off at 512 tokens, its own rounding being 1.7e-3.
// Where a text has at most 32 queries they are taken as two bf16 terms, and o is off by its own rounding alone: captions 9.6 -> 10.0 us, 128 texts'
// [CLS] over 512 tokens 28.2 -> 29.6.  For long texts that would cost 40 -> 48 us at 32 x 512 tokens, 127 -> 178 at 2 x 4096.  Sums stay in 32 bits.
//
// What bounds it.  A score takes 3.5 vector instructions and an exp2 at a quarter of their rate in the forward, 5.5 and one in dQ, 6 to 8 and one in
// dK / dV, against 2, 3 and 4 products of 64.  At 2 texts of 4096 tokens the vector pipes are busy 0.64 / 0.63 / 0.48 of the CUs' busy time in the
// forward / dQ / dK dV, the matrix pipes 0.40 / 0.47 / 0.42 (the clock settles near 1.8 GHz): the first two are near their vector pipes' pace, while in
// dK / dV neither pipe bounds -- its registers allow two waves a SIMD, and a wave's products, exponentials and products follow one another.  At 512
// tokens both pipes wait more (vector 0.57 / 0.44 / 0.42, matrix 0.24 / 0.24 / 0.26): few tiles a workgroup behind its bias and first loads, texts of
// unequal length.  Measured, 12 heads, kernel time and rate of the products of pairs that count:
//                         32 texts of 128 to 512 tokens,   2 texts of 4096 tokens
//                         two empty, padded to 512
//   forward               38 us    440 TF/s                121 us   850 TF/s
//   dQ                    58 us    440 TF/s                164 us   940 TF/s
//   dK / dV / diagonals   74 us    450 TF/s                225 us   920 TF/s
//   table's last sums    4 + 4 us                         4 + 4 us
// Tried, without gain or worse: tiles swizzled without any bank conflict; the log-sums spread by a product with ones; three waves a SIMD for
// dK / dV (spills: 254 -> 311 us); wave priorities around the products; a loop copy per staging buffer in dK / dV.
#include <type_traits>
#include "common.h"

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16;
typedef unsigned int u32;
typedef unsigned long long u64;

constexpr int TP = 72;                      // LDS row pitch in bf16 of the kernel for short texts (144 bytes: spread over the banks)
constexpr int BPAD = 192;                   // the bias vector reaches this far beyond +-R: a tile of 128 x 64 that touches |d| < R needs no clipping
constexpr int MAXR = 512;                   // largest R (LDS)
constexpr float LOG2E = 1.4426950408889634f;

struct RpArgs {
    const u16 *q, *k, *v, *o, *dout;        // element (row, h * 64 + d) of a text's rows: base + row * ld + ...
    long long ldq, ldk, ldo;                // row strides of q / (k, v) / (o, dout)
    u16 *out, *dq, *dk, *dv;
    long long lddq, lddk;
    const unsigned char* mask;              // [B][Lk] key mask (non-zero = takes part) or NULL
    const int* cu;                          // packed form: text b = rows cu[b] .. cu[b + 1] - 1 of [T] rows; NULL = padded
    int B, Lq, Lk, T, heads;                // Lq = 0: the queries are the packed rows themselves; Lk: the longest text
    float scale2;                           // scale * log2(e)
    float scale;
    const void* table;                      // [nb][heads]
    int table_bf16, nb, R;
    const int* bucket;                      // [2 R + 1]
    float* lse;                             // [heads][rows]: log2-sum of a row's scores (+inf: no key)
    float* dsum;                            // [heads][rows]: D
    float* diag;                            // [heads][slots][nd]: the bias gradient's parts per distance
    int nqb;                                // query blocks of the longest text
    int ns;                                 // parts a text's keys (forward, dQ) or queries (dK, dV) are split into
    float *po, *pm;                         // the parts' results: [ns][heads][rows][64], and of the forward [ns][heads][rows][2] (maximum, sum)
    float* pr;                              // of dQ [ns][heads][rows]: the rows' sums of ds
    float* pv;                              // dV's
    long long rows, krows;                  // query rows, key rows in all
};

// rows of text b; a packed text longer than Lk is cut to its first Lk rows (`to`: where its rows end)
struct Text { long long q0, k0, to; int lq, lk; };
__device__ __forceinline__ Text text_of(const RpArgs& a, int b) {
    Text t;
    if (a.cu) {
        const int r0 = min(max(a.cu[b], 0), a.T), r1 = min(max(a.cu[b + 1], r0), a.T);
        t.k0 = r0; t.to = r1; t.lk = min(r1 - r0, a.Lk);
        t.q0 = a.Lq ? (long long)b * a.Lq : r0; t.lq = a.Lq ? a.Lq : t.lk;
    } else {
        t.q0 = (long long)b * a.Lq; t.k0 = (long long)b * a.Lk; t.lq = a.Lq; t.lk = a.Lk; t.to = t.k0 + a.Lk;
    }
    return t;
}
// head h's 64 columns of rows from .. to - 1: zeros
template <int NT>
__device__ __forceinline__ void zero_rows(u16* p, long long ld, int h, long long from, long long to) {
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    for (long long i = threadIdx.x; i < (to - from) * 8; i += NT) *reinterpret_cast<f32x4*>(p + (from + (i >> 3)) * ld + h * 64 + (i & 7) * 8) = z;
}
// The packed rows that belong to no text, or to a text's cut part: zeros, written by the workgroups of the text before (the first text's:
// also what stands before it).  Split: the join writes the rows before cu[B], from parts that are empty there (zeros; maximum -inf).
template <int NT>
__device__ __forceinline__ void clear_rest(const RpArgs& a, const Text& t, int b, int h, int sp, u16* p, u16* p2, long long ld) {
    const long long ends[3][2] = {{b == 0 ? 0 : t.k0, t.k0}, {t.k0 + t.lk, t.to}, {t.to, b == a.B - 1 ? a.T : t.to}};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const long long from = ends[i][0], to = ends[i][1];
        if (a.ns == 1 || (i == 2 && sp == 0)) {
            zero_rows<NT>(p, ld, h, from, to);
            if (p2) zero_rows<NT>(p2, ld, h, from, to);
        } else if (i < 2) {
            const long long at = ((long long)sp * a.heads + h) * a.T;
            for (long long r = (at + from) * 64 + threadIdx.x; r < (at + to) * 64; r += NT) {
                a.po[r] = 0.f;
                if (p2) a.pv[r] = 0.f;
            }
            if (a.pm) for (long long r = at + from + threadIdx.x; r < at + to; r += NT) { a.pm[2 * r] = -INFINITY; a.pm[2 * r + 1] = 0.f; }
        }
    }
}

__device__ __forceinline__ int acc_r(int r, int lane) { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }
__device__ __forceinline__ void zero16(f32x16& a) {
#pragma unroll
    for (int r = 0; r < 16; ++r) a[r] = 0.f;
}
// (as a vector: one instruction for two values; converted one by one they are put together by two more)
__device__ __forceinline__ u32 pack2(float a, float b) {
    const f32x2 v = {a, b};
    return __builtin_bit_cast(u32, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ bf16x8 pack_acc(const f32x16& a, int kk) {
    f32x8 v;
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = a[8 * kk + t];
    return __builtin_convertvector(v, bf16x8);
}
// what pack_acc's rounding left off
__device__ __forceinline__ bf16x8 pack_rest(const f32x16& a, const bf16x8& f, int kk) {
    const f32x8 w = __builtin_convertvector(f, f32x8);
    f32x8 v;
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = a[8 * kk + t] - w[t];
    return __builtin_convertvector(v, bf16x8);
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
// A staged tile: ROWS rows of 128 bytes, the 16-byte piece p of row r at place p ^ (r & 7) of its row: both kinds of reads below, and the
// copy, spread over the banks without padding.  The copy goes straight to LDS, 8 rows an instruction, issued from inline assembly: the
// compiler would wait for all of it before the next LDS read, while here it has a whole tile's computation to land (`landed`, then a
// barrier).  Rows past the end repeat the last one; rows whose bit in `bits` is 0 (these, and dropped keys) are cleared by the lanes that
// copied them: whatever stands there, infinities and NaN included, must not reach a product.
// APART: rows 32 .. 63 are at place p ^ 4 ^ (r & 7), for the reader that takes rows r and r + 32 together (Apart below).
template <int NW, int ROWS, bool APART = false>
struct Tile {
    static __device__ __forceinline__ void copy(const u16* base, u32 ld, int valid, const u16* tile, int w, int lane) {
        const u32 dst = (u32)(size_t)(__attribute__((address_space(3))) const u16*)tile;
#pragma unroll
        for (int i = 0; i < ROWS / 8 / NW; ++i) {
            const int ins = w + i * NW;
            const u32 off = (u32)min(ins * 8 + (lane >> 3), valid - 1) * ld * 2 +
                            (((lane & 7) ^ (lane >> 3) ^ (APART ? (ins >> 2) << 2 : 0)) << 4);
            const u32 to = __builtin_amdgcn_readfirstlane(dst + ins * 1024);
            u32 keep;
            asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                         : "=&s"(keep) : "v"(off), "s"(base), "s"(to) : "memory");
        }
    }
    static __device__ __forceinline__ void landed(u16* tile, u64 bits, int w, int lane) {
        if (bits == (ROWS == 64 ? ~0ull : 0xffffffffull)) return;
        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < ROWS / 8 / NW; ++i) {
            const int ins = w + i * NW;
            if (!((bits >> (ins * 8 + (lane >> 3))) & 1)) *reinterpret_cast<f32x4*>(tile + ins * 512 + lane * 8) = z;
        }
    }
};
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// byte offsets of a lane's reads: row (lane & 31), piece (lane >> 5); row 4 (lane >> 5) + ..., column 16 ((lane >> 4) & 1) + ...
struct Places {
    u32 row, col;
    __device__ __forceinline__ explicit Places(int lane) {
        const int p = lane & 15, g = lane >> 4, r = 4 * (g >> 1) + (p >> 2);
        row = (lane & 31) * 128 + (((lane >> 5) ^ (lane & 7)) << 4);
        col = r * 128 + (((2 * (g & 1) + ((p & 3) >> 1)) ^ r) << 4) + (p & 1) * 8;
    }
};
// Of 64 staged rows in two blocks: block u of the product S = rows x columns takes row 32 (1 - half) + 16 u + r as the one whose scores stand in
// register r of the lanes `half`, so that both halves' rows follow one another in the registers, 32 apart; byte offsets as above.
struct Apart {
    u32 row, col;
    __device__ __forceinline__ explicit Apart(int lane) {
        const int p = lane & 15, g = lane >> 4, r = (lane & 3) + 4 * ((lane & 31) >> 3), h = (lane >> 2) & 1;
        row = (32 * (1 - h) + r) * 128 + (((lane >> 5) ^ (r & 7) ^ (4 * (1 - h))) << 4);
        col = (32 * (1 - (g >> 1)) + (p >> 2)) * 128 + (((2 * (g & 1) + ((p & 3) >> 1)) ^ (p >> 2) ^ (4 * (1 - (g >> 1)))) << 4) + (p & 1) * 8;
    }
};
__device__ __forceinline__ u64 low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// The keys of a text in tiles of KT, 64 tiles at a time: which tiles have a key (bit i of `alive`: tile i from c0), which rows of a tile.
template <int NW, int KT>
struct Keys {
    const unsigned char* mask;
    int lk, c0;
    u64* tb;                                                   // [64] in LDS, used with a mask
    u64 alive;
    __device__ __forceinline__ void chunk(int c0_) {           // (all waves; a barrier inside where there is a mask)
        c0 = c0_;
        const int lane = threadIdx.x & 63, n = min(64, (lk - c0 + KT - 1) / KT);
        if (!mask) { alive = low_bits(n); return; }
        __syncthreads();
        for (int t = threadIdx.x >> 6; t < n; t += NW) {
            const int j = c0 + t * KT + lane;
            const u64 bits = __ballot(lane < KT && j < lk && mask[min(j, lk - 1)] != 0);
            if (lane == 0) tb[t] = bits;
        }
        __syncthreads();
        alive = __ballot(lane < n && tb[lane < n ? lane : 0] != 0);
    }
    __device__ __forceinline__ u64 bits(int t) const {
        if (!mask) return low_bits(min(KT, lk - c0 - t * KT));
        const u64 v = tb[t];                                   // (the same for every lane)
        return ((u64)(u32)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (u32)__builtin_amdgcn_readfirstlane((int)v);
    }
    static constexpr u64 FULL = KT == 64 ? ~0ull : 0xffffffffull;
};
__device__ __forceinline__ int next_tile(u64& alive) {         // the lowest tile left, taken out; -1: none
    if (!alive) return -1;
    const int t = __builtin_ctzll(alive);
    alive &= alive - 1;
    return t;
}

// step(buffer) for the NB buffers in turn until it is done.  The buffer is a constant in each copy of the loop: its LDS addresses are offsets in the
// instructions, where a variable one costs an addition for every read.
template <int NB, class Step>
__device__ __forceinline__ void in_turn(const Step& step) {
    while (true) {
        if (step(std::integral_constant<int, 0>{})) break;
        if constexpr (NB > 1) {
            if (step(std::integral_constant<int, 1>{})) break;
        }
    }
}

// part `sp` of `ns` of n rows in whole tiles: [from, to)
struct Part { int from, to; };
__device__ __forceinline__ Part part_of(int sp, int ns, int n, int tile) {
    const int per = ((n + tile - 1) / tile + ns - 1) / ns * tile;
    return Part{min(sp * per, n), min((sp + 1) * per, n)};
}

// the bias in units of log2; -1e30 and less (a type's lowest value, -inf) drops the key, as a mask does
__device__ __forceinline__ float bias_of(float t) { return t > -1e30f || t != t ? t * LOG2E : -INFINITY; }
// head h's bias over the distances lo .. hi, in units of log2: bl[d + R + BPAD].  Two dependent loads a distance; those of four distances
// travel together.
template <int NT>
__device__ __forceinline__ void fill_bias(const RpArgs& a, int h, float* bl, int lo, int hi) {
    const int mid = a.R + BPAD, first = max(lo, -mid), last = min(hi, mid);
    for (int d = first + (int)threadIdx.x; d <= last; d += 4 * NT) {
        int bk[4];
        float t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) bk[i] = a.bucket[min(max(min(d + i * NT, last), -a.R), a.R) + a.R];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long at = (long long)min(max(bk[i], 0), a.nb - 1) * a.heads + h;
            t[i] = a.table_bf16 ? __uint_as_float((u32)((const u16*)a.table)[at] << 16) : ((const float*)a.table)[at];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) if (d + i * NT <= last) bl[d + i * NT + mid] = bias_of(t[i]);
    }
}
// A tile of 32 queries that a wave owns against `n` staged keys, d0 = (first key) - (first query): whether it touches |d| < R
__device__ __forceinline__ bool tile_near(int R, int d0, int n) { return d0 - 31 < R && d0 + n - 1 > -R; }
// ... and, where it does not, the one bias it has
__device__ __forceinline__ float far_bias(const float* bl, int R, int d0) { return bl[(d0 > 0 ? R : -R) + R + BPAD]; }
// S += A B^T of U blocks of 32 staged rows against a wave's 32; the blocks' chains of four take turns.  The lane's operand: its row's d
// 16 kk + 8 (lane >> 5) .. + 7
template <int U>
__device__ __forceinline__ void mma_rows(const u16* tile, const Places& at, const bf16x8 (&f)[4], f32x16 (&s)[U]) {
    const char* t = reinterpret_cast<const char*>(tile);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int u = 0; u < U; ++u)
            s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(t + 4096 * u + (at.row ^ (kk << 5))), f[kk], s[u], 0, 0, 0);
}
// out^T += (tile's columns) (w packed to bf16), contraction over the 32 rows of block u; the lane's operand: column 32 dt + (lane & 31), rows
// in the accumulators' order (a 16-lane group's transposing read takes a [4 rows x 16 columns] block).  TWO: w in two bf16 terms
template <bool TWO = false>
__device__ __forceinline__ void mma_cols(const u16* tile, const Places& at, int u, const f32x16& w, f32x16 (&out)[2]) {
    const char* t = reinterpret_cast<const char*>(tile);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        const bf16x8 f = pack_acc(w, kk), rest = pack_rest(w, f, kk);
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
            const char* a = t + (2 * u + kk) * 2048 + (at.col ^ (dt << 6));
            union { s16x4 h[2]; bf16x8 v; } x;
            x.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a));
            x.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 1024));
            out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.v, f, out[dt], 0, 0, 0);
            if (TWO) out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.v, rest, out[dt], 0, 0, 0);
        }
    }
}
// ... the same two products of block u with the rows taken as by Apart
__device__ __forceinline__ void mma_rows_apart(const u16* tile, const Apart& at, int u, const bf16x8 (&f)[4], f32x16& s) {
    const char* t = reinterpret_cast<const char*>(tile) + 2048 * u;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(t + (at.row ^ (kk << 5))), f[kk], s, 0, 0, 0);
}
__device__ __forceinline__ void mma_cols_apart(const u16* tile, const Apart& at, int u, const f32x16& w, f32x16 (&out)[2]) {
    const char* t = reinterpret_cast<const char*>(tile);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        const bf16x8 f = pack_acc(w, kk);
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
            union { s16x4 h[2]; bf16x8 v; } x;
#pragma unroll
            for (int i = 0; i < 2; ++i)                        // (four rows on: the other place of a pair)
                x.h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(t + (2 * u + kk) * 1024 + i * 512 +
                                                                                                           (at.col ^ ((dt ^ i) << 6))));
            out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.v, f, out[dt], 0, 0, 0);
        }
    }
}
// dropped keys of block u: -inf (lane = query, registers = keys)
__device__ __forceinline__ void drop_keys(f32x16& s, u64 bits, int u, int lane) {
    const u32 in = (u32)(bits >> (32 * u)) >> (4 * (lane >> 5));
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = (in >> ((r & 3) + 8 * (r >> 2))) & 1 ? s[r] : -INFINITY;
}
// a lane's 32 values of its row, rounded once.  The lanes l, l ^ 32 of a row trade halves (one instruction for two values), so that each writes 16
// bytes in one piece (256 captions, 12 heads: forward 12.6 -> 11.2, backward 30.8 -> 26.6 us).
__device__ __forceinline__ void store_row(const f32x16 (&o)[2], u16* row, int lane, float c) {
    u16* op = row + 8 * (lane >> 5);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const auto x = __builtin_amdgcn_permlane32_swap(pack2(o[dt][8 * g] * c, o[dt][8 * g + 1] * c), pack2(o[dt][8 * g + 4] * c, o[dt][8 * g + 5] * c), false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(pack2(o[dt][8 * g + 2] * c, o[dt][8 * g + 3] * c), pack2(o[dt][8 * g + 6] * c, o[dt][8 * g + 7] * c), false, false);
            *reinterpret_cast<uint4*>(op + 32 * dt + 16 * g) = uint4{x[0], y[0], x[1], y[1]};
        }
}
// over the two lanes l, l ^ 32 (one VALU instruction instead of a trip through the LDS queue)
__device__ __forceinline__ float half_max(float v) {
    const u32 u = __float_as_uint(v);
    const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// a lane's 32 values of its row in 32 bits: out [64]
__device__ __forceinline__ void store_part(const f32x16 (&o)[2], float* out, int lane) {
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 v = {o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
            *reinterpret_cast<f32x4*>(out + 32 * dt + 8 * g + 4 * (lane >> 5)) = v;
        }
}

// ---- forward.  A wave owns 32 queries of one (text, head); NW waves share the staged keys, KT at a time in NB buffers.
template <int NW, int KT, int NB>
__global__ __launch_bounds__(NW * 64, 3) void cfl_relpos_fwd_kernel(RpArgs a) {
    constexpr int NT = NW * 64, U = KT / 32;
    __shared__ __attribute__((aligned(1024))) u16 Kt[NB][KT * 64], Vt[NB][KT * 64];
    __shared__ u64 tb[64];
    extern __shared__ float bl[];
    const int lane = threadIdx.x & 63, w = wave_id();
    const Places at(lane);
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int sp = id % a.ns, qb = id / a.ns % a.nqb, h = id / (a.ns * a.nqb) % a.heads, b = id / (a.ns * a.nqb * a.heads);
    const Text t = text_of(a, b);
    if (a.cu && !a.Lq && qb == 0) clear_rest<NT>(a, t, b, h, sp, a.out, nullptr, a.ldo);
    if (qb * NW * 32 >= t.lq) return;
    const Part part = part_of(sp, a.ns, t.lk, KT);
    Keys<NW, KT> keys{a.mask ? a.mask + (long long)b * a.Lk : nullptr, part.to, 0, tb, 0};
    const u16* kp = a.k + t.k0 * a.ldk + h * 64;
    const u16* vp = a.v + t.k0 * a.ldk + h * 64;
    const int q0 = (qb * NW + w) * 32;
    bf16x8 qf[4];
    load_rows(a.q + t.q0 * a.ldq + h * 64, a.ldq, q0, t.lq, lane, qf);
    f32x16 o[2];
    zero16(o[0]); zero16(o[1]);
    // l and o are relative to 2^m.  m follows the running maximum lazily: only when a score passes it by more than 8 are l and o brought
    // to the new one (p then stays below 2^8; the division by l at the end cancels whatever m is).  seen: the row has met a key; one whose
    // tiles so far were all dropped by the bias waits
    float m = 0.f, l0 = 0.f, l1 = 0.f;
    bool first = true, seen = false, filled = false;
    for (int c0 = part.from; c0 < part.to; c0 += 64 * KT) {
        keys.chunk(c0);
        u64 left = keys.alive;
        int cur = next_tile(left);
        if (cur < 0) continue;
        u64 bits = keys.bits(cur);
        const auto copy = [&](int tile, int to) {
            const int k0 = c0 + tile * KT;
            Tile<NW, KT>::copy(kp + (long long)k0 * a.ldk, (u32)a.ldk, t.lk - k0, Kt[to], w, lane);
            Tile<NW, KT>::copy(vp + (long long)k0 * a.ldk, (u32)a.ldk, t.lk - k0, Vt[to], w, lane);
        };
        __syncthreads();                                       // (the tiles' last readers)
        copy(cur, 0);
        if (!filled) fill_bias<NT>(a, h, bl, -(t.lq | (NW * 32 - 1)), t.lk | (KT - 1));      // (rows past the end are computed with as well)
        filled = true;                                         // (its loads travel with the first tile's)
        const auto step = [&](auto buf_) {                     // one tile; whether it was the last
            constexpr int buf = decltype(buf_)::value;
            const int d0 = c0 + cur * KT - q0, nxt = next_tile(left);
            wait_copies();
            Tile<NW, KT>::landed(Kt[buf], bits, w, lane);
            Tile<NW, KT>::landed(Vt[buf], bits, w, lane);
            __syncthreads();                                   // (this tile for every wave; the other buffer's readers are done)
            if (NB > 1 && nxt >= 0) copy(nxt, buf ^ 1);
            f32x16 s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) zero16(s[u]);
            mma_rows<U>(Kt[buf], at, qf, s);
            if (tile_near(a.R, d0, KT)) {
                const float* bp = bl + a.R + BPAD + d0 + 4 * (lane >> 5) - (lane & 31);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[u][r] = fmaf(s[u][r], a.scale2, bp[32 * u + (r & 3) + 8 * (r >> 2)] - m);
            } else {
                const float c = far_bias(bl, a.R, d0) - m;
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[u][r] = fmaf(s[u][r], a.scale2, c);
            }
            if (bits != Keys<NW, KT>::FULL) {
#pragma unroll
                for (int u = 0; u < U; ++u) drop_keys(s[u], bits, u, lane);
            }
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
            top = half_max(top);
            const bool met = top > -INFINITY;
            if (__any(top > 8.f || (met && !seen))) {
                const float by = !met ? 0.f : seen ? fmaxf(top, 0.f) : top, shrink = seen ? __builtin_amdgcn_exp2f(-by) : 1.f;
                if (!first) {
                    l0 *= shrink; l1 *= shrink;
#pragma unroll
                    for (int r = 0; r < 16; ++r) { o[0][r] *= shrink; o[1][r] *= shrink; }
                }
                first = false;
                seen |= met;
                m += by;
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[u][r] -= by;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    s[u][r] = __builtin_amdgcn_exp2f(s[u][r]);
                    s[u][r + 1] = __builtin_amdgcn_exp2f(s[u][r + 1]);
                    l0 += s[u][r];
                    l1 += s[u][r + 1];
                }
                mma_cols<NW == 1>(Vt[buf], at, u, s[u], o);    // (two terms for a few queries)
            }
            if (nxt < 0) return true;
            if (NB == 1) {
                __syncthreads();
                copy(nxt, 0);
            }
            cur = nxt;
            bits = keys.bits(nxt);
            return false;
        };
        in_turn<NB>(step);
    }
    float l = l0 + l1;
    l += __shfl_xor(l, 32, 64);
    const bool none = !seen && l == 0.f;                       // (not so where NaN scores made l one)
    const int row = q0 + (lane & 31);
    if (row >= t.lq) return;
    if (a.ns > 1) {
        const long long to = ((long long)sp * a.heads + h) * a.rows + t.q0 + row;
        store_part(o, a.po + to * 64, lane);
        if (lane < 32) { a.pm[2 * to] = none ? -INFINITY : m; a.pm[2 * to + 1] = l; }
    } else {
        store_row(o, a.out + (t.q0 + row) * a.ldo + h * 64, lane, none ? 0.f : 1.f / l);
        if (a.lse && lane < 32) a.lse[h * a.rows + t.q0 + row] = none ? INFINITY : m + __builtin_amdgcn_logf(l);
    }
}

// Sums of a 32 x 32 block along its diagonals.  Register r of lane (x, half) holds column x and row j = (r & 3) + 8 (r >> 2) + 4 half; the sum
// over j - x = e is added to dst[-e] in LDS.  With the columns in lanes 32 .. 63 and zeros below, the sums are  t <- (t moved down one
// lane) + v_j  for j from the highest down: lane i then holds e = 32 - i.  One instruction moves and adds; two chains of 16 rows take turns.
// The words are the wave's own, an addition's 64 addresses distinct and a wave's LDS operations in order: plain reads and writes, and a fixed
// order of every sum (with LDS atomics, some 50 clocks each, the dK / dV kernel took 100 us instead of 82 at 32 texts of 512 tokens, 12 heads).
__device__ __forceinline__ void add_own(float* p, float v) {
    *p += v;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");     // (the next addition reads words that other lanes write here)
}
__device__ __forceinline__ float down_one(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x130, 0xf, 0xf, true));
}
__device__ __forceinline__ float down_one_round(float v) {     // (lane 0's goes to lane 63)
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x134, 0xf, 0xf, true));
}
// With rows taken as by Apart no lane stands idle: register r of lane l holds e = (row) - (column) = 32 + 16 u + r - l, so after the same steps lane i
// holds e = 32 + 16 u - i; what has left at lane 0 is the difference to the same sums with the lanes in a ring: at lane i >= 49 e = 96 + 16 u - i.
// dst: the place of e = 0, places fall with e.  32 instructions for 16 rows of 64 lanes, against 80 with the zeros below.  (The difference holds to
// 2^-24 of the larger of a block's sums: a distance whose ds are 1e-8 of its neighbours' in the same block has few digits of its own.)
__device__ __forceinline__ void diag_add_apart(const f32x16& v, float* dst, int u, int lane) {
#pragma clang fp contract(off)                                  // (a fused product would take the shift out of the addition)
    float a = v[15], b = v[15];
#pragma unroll
    for (int r = 14; r >= 0; --r) { a = down_one(a) + v[r]; b = down_one_round(b) + v[r]; }
    add_own(dst + lane - 32 - 16 * u, a);
    if (lane >= 49) add_own(dst + lane - 96 - 16 * u, b - a);
}
__device__ __forceinline__ void diag_add(const f32x16& v, float* dst, int lane) {
    float hi = 0.f, lo = 0.f;
#pragma unroll
    for (int g = 1; g >= 0; --g) {
        u32 low[8], up[8];                                     // half 0's and half 1's values of the groups g + 2 and g, in lanes 32 .. 63
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const auto w = __builtin_amdgcn_permlane32_swap(0u, __float_as_uint(v[4 * (g + (k < 4 ? 2 : 0)) + (k & 3)]), false, false);
            low[k] = w[0]; up[k] = w[1];
        }
#pragma unroll
        for (int k = 3; k >= 0; --k) { hi = down_one(hi) + __uint_as_float(up[k]); lo = down_one(lo) + __uint_as_float(up[k + 4]); }
#pragma unroll
        for (int k = 3; k >= 0; --k) { hi = down_one(hi) + __uint_as_float(low[k]); lo = down_one(lo) + __uint_as_float(low[k + 4]); }
    }
    add_own(dst + lane - 48, hi);
    add_own(dst + lane - 32, lo);
}

// ---- backward, queries: dQ and D.  Same ownership as the forward.
// D is formed from the rounded o, whose error is the same for a whole row of ds: the bias gradient would add it up along every diagonal.  But a
// row of ds sums to nothing, so the row's sum here is that error, and D goes to dK / dV's kernel, which sums the diagonals, without it.
template <int NW, int KT, int NB>
__global__ __launch_bounds__(NW * 64, NW == 4 ? 3 : 2) void cfl_relpos_dq_kernel(RpArgs a) {
    constexpr int NT = NW * 64, U = KT / 32;
    __shared__ __attribute__((aligned(1024))) u16 Kt[NB][KT * 64], Vt[NB][KT * 64];
    __shared__ u64 tb[64];
    extern __shared__ float bl[];
    const int mid = a.R + BPAD;
    const int lane = threadIdx.x & 63, w = wave_id();
    const Places at(lane);
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int sp = id % a.ns, qb = id / a.ns % a.nqb, h = id / (a.ns * a.nqb) % a.heads, b = id / (a.ns * a.nqb * a.heads);
    const Text t = text_of(a, b);
    const Part part = part_of(sp, a.ns, t.lk, KT);
    if (a.cu && !a.Lq && qb == 0) clear_rest<NT>(a, t, b, h, sp, a.dq, nullptr, a.lddq);
    if (qb * NW * 32 >= t.lq) return;
    fill_bias<NT>(a, h, bl, -(t.lq | (NW * 32 - 1)), t.lk | (KT - 1));     // (rows past the end are computed with as well)
    Keys<NW, KT> keys{a.mask ? a.mask + (long long)b * a.Lk : nullptr, part.to, 0, tb, 0};
    const u16* kp = a.k + t.k0 * a.ldk + h * 64;
    const u16* vp = a.v + t.k0 * a.ldk + h * 64;
    const int q0 = (qb * NW + w) * 32, row = q0 + (lane & 31);
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
    const float lse = live ? a.lse[h * a.rows + t.q0 + row] : INFINITY;      // (+inf: p = 0 in every row that does not count)
    float r0 = 0.f, r1 = 0.f;                                  // the row's sum of ds
    f32x16 dq[2];
    zero16(dq[0]); zero16(dq[1]);
    for (int c0 = part.from; c0 < part.to; c0 += 64 * KT) {
        keys.chunk(c0);
        u64 left = keys.alive;
        int cur = next_tile(left);
        if (cur < 0) continue;
        u64 bits = keys.bits(cur);
        const auto copy = [&](int tile, int to) {
            const int k0 = c0 + tile * KT;
            Tile<NW, KT>::copy(kp + (long long)k0 * a.ldk, (u32)a.ldk, t.lk - k0, Kt[to], w, lane);
            Tile<NW, KT>::copy(vp + (long long)k0 * a.ldk, (u32)a.ldk, t.lk - k0, Vt[to], w, lane);
        };
        __syncthreads();
        copy(cur, 0);
        const auto step = [&](auto buf_) {                     // one tile; whether it was the last
            constexpr int buf = decltype(buf_)::value;
            const int d0 = c0 + cur * KT - q0, nxt = next_tile(left);
            wait_copies();
            Tile<NW, KT>::landed(Kt[buf], bits, w, lane);
            Tile<NW, KT>::landed(Vt[buf], bits, w, lane);
            __syncthreads();                                   // (this tile for every wave; the other buffer's readers are done)
            if (NB > 1 && nxt >= 0) copy(nxt, buf ^ 1);
            const bool near = tile_near(a.R, d0, KT);
            const float* bp = bl + mid + (near ? d0 : 0) + 4 * (lane >> 5) - (lane & 31);
            const float c = far_bias(bl, a.R, near ? 0 : d0) - lse;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                f32x16 s[1], dp[1];
                zero16(s[0]); zero16(dp[0]);
                mma_rows<1>(Kt[buf] + 2048 * u, at, qf, s);
                mma_rows<1>(Vt[buf] + 2048 * u, at, gf, dp);
                if (near) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[0][r] = fmaf(s[0][r], a.scale2, bp[32 * u + (r & 3) + 8 * (r >> 2)] - lse);
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[0][r] = fmaf(s[0][r], a.scale2, c);
                }
                if (bits != Keys<NW, KT>::FULL) drop_keys(s[0], bits, u, lane);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[0][r] = __builtin_amdgcn_exp2f(s[0][r]) * (dp[0][r] - D);
#pragma unroll
                for (int r = 0; r < 16; r += 2) { r0 += s[0][r]; r1 += s[0][r + 1]; }
                mma_cols<NW == 1>(Kt[buf], at, u, s[0], dq);   // (two terms for a few queries: their roundings would show, and cost nothing)
                __builtin_amdgcn_sched_barrier(0);
            }
            if (nxt < 0) return true;
            if (NB == 1) {
                __syncthreads();
                copy(nxt, 0);
            }
            cur = nxt;
            bits = keys.bits(nxt);
            return false;
        };
        in_turn<NB>(step);
    }
    r0 += r1;
    r0 += __shfl_xor(r0, 32, 64);
    if (!live) return;
    if (a.ns > 1) {
        const long long to = ((long long)sp * a.heads + h) * a.rows + t.q0 + row;
        store_part(dq, a.po + to * 64, lane);
        if (lane < 32) {
            a.pr[to] = r0;
            if (sp == 0) a.dsum[h * a.rows + t.q0 + row] = D;  // (the join adds the sums)
        }
    } else {
        store_row(dq, a.dq + (t.q0 + row) * a.lddq + h * 64, lane, a.scale);
        if (lane < 32) a.dsum[h * a.rows + t.q0 + row] = D + r0;
    }
}

// ---- backward, keys: dK, dV and the bias gradient.  A wave owns 32 keys; the staged rows are queries.
// The bias gradient of a distance is the sum of ds along a diagonal (diag_add, into words of the wave's own; adding every value with an LDS
// atomic took 240 us more at 32 texts of 512 tokens, 12 heads).  Tiles beyond +-R are summed in registers.  At the end the workgroup's sums per distance go to
// part [heads][slots][2 R + 1], one slot per (text, key block, part).
template <int NW, int KT, int NB>
__global__ __launch_bounds__(NW * 64, 2) void cfl_relpos_dkv_kernel(RpArgs a, int nkb) {
    constexpr int NT = NW * 64, U = KT / 32;
    __shared__ __attribute__((aligned(1024))) u16 Qt[NB][KT * 64], Gt[NB][KT * 64];
    __shared__ __attribute__((aligned(16))) float ls[NB][KT], ds[NB][KT];      // -log-sum and -D of the staged queries
    extern __shared__ float bl[];
    const int nd = 2 * (a.R + BPAD) + 1, mid = a.R + BPAD;
    float* gone = bl + nd;                                     // [KT] of -inf: what a lane reads whose key does not take part
    float* dg = gone + KT;                                     // [NW][nd]
    const int lane = threadIdx.x & 63, w = wave_id();
    constexpr bool APART = KT == 64;
    typedef Tile<NW, KT, APART> TileQ;
    const std::conditional_t<APART, Apart, Places> at(lane);
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int sp = id % a.ns, kb = id / a.ns % nkb, h = id / (a.ns * nkb) % a.heads, b = id / (a.ns * nkb * a.heads);
    const Text t = text_of(a, b);
    if (a.cu && kb == 0) clear_rest<NT>(a, t, b, h, sp, a.dk, a.dv, a.lddk);
    float* out = a.diag + ((((long long)h * a.B + b) * nkb + kb) * a.ns + sp) * (2 * a.R + 1);
    if (kb * NW * 32 >= t.lk) {
        for (int i = threadIdx.x; i <= 2 * a.R; i += NT) out[i] = 0.f;
        return;
    }
    const Part part = part_of(sp, a.ns, t.lq, KT);
    const int dlo = max(-(t.lq | (KT - 1)), -mid), dhi = min(t.lk | (NW * 32 - 1), mid);      // (rows past the end are computed with as well)
    for (int c = 0; c < NW; ++c)
        for (int d = dlo + (int)threadIdx.x; d <= dhi; d += NT) dg[c * nd + d + mid] = 0.f;
    float far_lo = 0.f, far_hi = 0.f;
    float* mine = dg + w * nd + mid;
    for (int i = threadIdx.x; i < KT; i += NT) gone[i] = -INFINITY;
    const unsigned char* mask = a.mask ? a.mask + (long long)b * a.Lk : nullptr;
    const u16* qp = a.q + t.q0 * a.ldq + h * 64;
    const u16* gp = a.dout + t.q0 * a.ldo + h * 64;
    const float* lp = a.lse + h * a.rows + t.q0;
    const float* dp_ = a.dsum + h * a.rows + t.q0;
    const int k0 = (kb * NW + w) * 32, key = k0 + (lane & 31);
    const bool live = key < t.lk && (!mask || mask[key]);
    bf16x8 kf[4], vf[4];
    load_rows(a.k + t.k0 * a.ldk + h * 64, a.ldk, k0, t.lk, lane, kf);
    load_rows(a.v + t.k0 * a.ldk + h * 64, a.ldk, k0, t.lk, lane, vf);
    f32x16 dk[2], dv[2];
    zero16(dk[0]); zero16(dk[1]); zero16(dv[0]); zero16(dv[1]);
    if (__syncthreads_or(live) && part.from < part.to) {       // (else no key of the workgroup takes part: zeros)
        if (!live) {
            const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) { kf[kk] = __builtin_bit_cast(bf16x8, z); vf[kk] = __builtin_bit_cast(bf16x8, z); }
        }
        float lr = 0.f, dr = 0.f;
        const auto fetch = [&](int q0, int to) {
            TileQ::copy(qp + (long long)q0 * a.ldq, (u32)a.ldq, part.to - q0, Qt[to], w, lane);
            TileQ::copy(gp + (long long)q0 * a.ldo, (u32)a.ldo, part.to - q0, Gt[to], w, lane);
            if (threadIdx.x < KT) {
                const bool in = q0 + (int)threadIdx.x < part.to;
                lr = in ? -lp[q0 + threadIdx.x] : -INFINITY;
                dr = in ? -dp_[q0 + threadIdx.x] : 0.f;
            }
        };
        int buf = 0, q0 = part.from;
        fetch(q0, 0);
        fill_bias<NT>(a, h, bl, dlo, dhi);                     // (its loads travel with the first tile's)
        __syncthreads();
        // the lane's first query in the tile, and how its registers go on from it
        const int i0 = APART ? 32 - 32 * (lane >> 5) : 4 * (lane >> 5);
        const auto query = [](int u, int r) { return APART ? 16 * u + r : 32 * u + (r & 3) + 8 * (r >> 2); };
        // the tiles up to query `until`, all near or all far for the whole workgroup, far ones with the bias c; `sum`: theirs of ds
        const auto tiles = [&](auto near_, int until, float c, float& sum) {
            constexpr bool near = decltype(near_)::value;
            for (; q0 < until; q0 += KT) {
                const bool more = q0 + KT < part.to;
                if (threadIdx.x < KT) { ls[buf][threadIdx.x] = lr; ds[buf][threadIdx.x] = dr; }
                wait_copies();
                TileQ::landed(Qt[buf], low_bits(min(KT, part.to - q0)), w, lane);
                TileQ::landed(Gt[buf], low_bits(min(KT, part.to - q0)), w, lane);
                __syncthreads();
                if (NB > 1 && more) fetch(q0 + KT, buf ^ 1);
                const int d0 = k0 - q0;
                const float* bp = live ? bl + mid + d0 + (lane & 31) - i0 : gone + KT - 1;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    f32x16 s[1], dp[1], nl;
                    zero16(s[0]);
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 x = *reinterpret_cast<const f32x4*>(&ls[buf][i0 + query(u, 4 * g)]);
                        const f32x4 y = *reinterpret_cast<const f32x4*>(&ds[buf][i0 + query(u, 4 * g)]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) { nl[4 * g + j] = x[j]; dp[0][4 * g + j] = y[j]; }
                    }
                    if constexpr (APART) {
                        mma_rows_apart(Qt[buf], at, u, kf, s[0]);
                        mma_rows_apart(Gt[buf], at, u, vf, dp[0]);
                    } else {
                        mma_rows<1>(Qt[buf], at, kf, s);
                        mma_rows<1>(Gt[buf], at, vf, dp);
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        nl[r] += near ? bp[-query(u, r)] : c;
                        s[0][r] = __builtin_amdgcn_exp2f(fmaf(s[0][r], a.scale2, nl[r]));
                        dp[0][r] *= s[0][r];
                    }
                    if constexpr (APART) mma_cols_apart(Gt[buf], at, u, s[0], dv);
                    else mma_cols<NB == 1>(Gt[buf], at, 0, s[0], dv);
                    if constexpr (APART) mma_cols_apart(Qt[buf], at, u, dp[0], dk);
                    else mma_cols<NB == 1>(Qt[buf], at, 0, dp[0], dk);
                    if constexpr (!near) {
                        float x0 = 0.f, x1 = 0.f;
#pragma unroll
                        for (int r = 0; r < 16; r += 2) { x0 += dp[0][r]; x1 += dp[0][r + 1]; }
                        sum += x0 + x1;
                    } else if constexpr (APART) {
                        diag_add_apart(dp[0], mine + d0, u, lane);
                    } else {
                        diag_add(dp[0], mine + d0, lane);
                    }
                }
                if (NB > 1) {
                    buf ^= 1;
                } else if (more) {
                    __syncthreads();
                    fetch(q0 + KT, 0);
                }
            }
        };
        // queries so far before the workgroup's keys that every distance is R or more, then the near ones, then those far behind
        const int first = kb * NW * 32, before = first - a.R - KT + 2, behind = first + NW * 32 - 1 + a.R;
        const float clo = live ? far_bias(bl, a.R, -1) : -INFINITY, chi = live ? far_bias(bl, a.R, 1) : -INFINITY;
        tiles(std::false_type{}, min(before, part.to), chi, far_hi);
        tiles(std::true_type{}, min(behind, part.to), 0.f, far_hi);
        tiles(std::false_type{}, part.to, clo, far_lo);
    }
    // the workgroup's sums per distance; what lies beyond +-R counts as +-R
    for (int d = dlo + lane; d < -a.R; d += 64) far_lo += mine[d];
    for (int d = a.R + 1 + lane; d <= dhi; d += 64) far_hi += mine[d];
    far_lo = wave_sum(far_lo);
    far_hi = wave_sum(far_hi);
    if (lane == 0) {                                           // (these words exist where there was something to add)
        if (dlo <= -a.R) mine[-a.R] += far_lo;
        if (dhi >= a.R) mine[a.R] += far_hi;
    }
    __syncthreads();
    for (int i = threadIdx.x; i <= 2 * a.R; i += NT) {
        const int d = i - a.R;
        float x = 0.f;
        if (d >= dlo && d <= dhi) {
#pragma unroll
            for (int c = 0; c < NW; ++c) x += dg[c * nd + d + mid];
        }
        out[i] = x;
    }
    if (key >= t.lk) return;
    if (!live) { zero16(dk[0]); zero16(dk[1]); zero16(dv[0]); zero16(dv[1]); }
    if (a.ns > 1) {
        const long long to = (((long long)sp * a.heads + h) * a.krows + t.k0 + key) * 64;
        store_part(dk, a.po + to, lane);
        store_part(dv, a.pv + to, lane);
    } else {
        store_row(dk, a.dk + (t.k0 + key) * a.lddk + h * 64, lane, a.scale);
        store_row(dv, a.dv + (t.k0 + key) * a.lddk + h * 64, lane, 1.f);
    }
}

// ---- backward of texts of at most 32 tokens: everything in one kernel, a wave per (text, head).  The rows come straight from memory as
// operands; K, Q and dO pass through LDS for the products that contract over rows.  D is summed from p and dp themselves, so the
// rounding of o plays no part; P and ds are taken as two bf16 terms: few products, and waiting for memory bounds this kernel.  The bias gradient's diagonals go to memory as they are: part [heads][B][64], place d + 32.
// The log-sum is taken off the score as the forward formed it: a row of one key has p = 1 and ds = 0 to the bit.
// 256 packed captions of 8 to 32 tokens, 12 heads: 21 us (2.2 TB/s), against 40 us with the kernels for long texts.  A wave's chain of loads bounds
// it: every wave is resident at once, so nothing follows to hide it.
__global__ __launch_bounds__(64) void cfl_relpos_bwd32_kernel(RpArgs a) {
    __shared__ __attribute__((aligned(16))) u16 Kt[32 * TP], Qt[32 * TP], Gt[32 * TP];
    __shared__ float bl[64], dgs[128];
    __shared__ __attribute__((aligned(16))) float ls[32], Ds[32];
    const int lane = threadIdx.x, x = lane & 31, half = lane >> 5;
    const int id = xcd_remap(blockIdx.x, gridDim.x), h = id % a.heads, b = id / a.heads;
    const int bk = a.bucket[min(max(lane - 31, -a.R), a.R) + a.R];      // (first: a second load hangs on it)
    const Text t = text_of(a, b);
    float* part = a.diag + ((long long)h * a.B + b) * 64;
    if (a.cu) {
        if (!a.Lq) clear_rest<64>(a, t, b, h, 0, a.dq, nullptr, a.lddq);
        clear_rest<64>(a, t, b, h, 0, a.dk, a.dv, a.lddk);
    }
    if (t.lq == 0 || t.lk == 0) {
        part[lane] = 0.f;
        zero_rows<64>(a.dq, a.lddq, h, t.q0, t.q0 + t.lq);
        return;
    }
    const long long ti = (long long)min(max(bk, 0), a.nb - 1) * a.heads + h;
    const float bias = a.table_bf16 ? __uint_as_float((u32)((const u16*)a.table)[ti] << 16) : ((const float*)a.table)[ti];
    const u32 bits = (u32)__ballot(lane < t.lk && (!a.mask || a.mask[(long long)b * a.Lk + min(lane, t.lk - 1)] != 0));
    const bool keep = (bits >> x) & 1;
    bf16x8 kf[4], vf[4], qf[4], gf[4];
    load_rows(a.k + t.k0 * a.ldk + h * 64, a.ldk, 0, t.lk, lane, kf);
    load_rows(a.v + t.k0 * a.ldk + h * 64, a.ldk, 0, t.lk, lane, vf);
    load_rows(a.q + t.q0 * a.ldq + h * 64, a.ldq, 0, t.lq, lane, qf);
    load_rows(a.dout + t.q0 * a.ldo + h * 64, a.ldo, 0, t.lq, lane, gf);
    const float lse = x < t.lq ? a.lse[h * a.rows + t.q0 + x] : INFINITY;
    bl[lane] = bias_of(bias);
    const f32x4 z4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        const int at = x * TP + kk * 16 + half * 8;
        if (!keep) { kf[kk] = __builtin_bit_cast(bf16x8, z4); vf[kk] = __builtin_bit_cast(bf16x8, z4); }
        *reinterpret_cast<bf16x8*>(Kt + at) = kf[kk];
        *reinterpret_cast<bf16x8*>(Qt + at) = qf[kk];
        *reinterpret_cast<bf16x8*>(Gt + at) = gf[kk];
    }
    __syncthreads();
    f32x16 s, dp;
    // lane = query
    zero16(s); zero16(dp);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk], qf[kk], s, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[kk], gf[kk], dp, 0, 0, 0);
    }
    float D = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int kr = (r & 3) + 8 * (r >> 2);
        const bool ok = (bits >> (kr + 4 * half)) & 1;
        const float p = ok ? __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, bl[31 + 4 * half - x + kr]) - lse) : 0.f;
        s[r] = p;
        dp[r] = ok ? dp[r] : 0.f;                              // (a text without a key: 0, whatever its gradient holds)
        D = fmaf(p, dp[r], D);
    }
    D += __shfl_xor(D, 32, 64);
    if (lane < 32) { ls[x] = lse; Ds[x] = D; }
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= dp[r] - D;
    dgs[lane] = 0.f;
    dgs[lane + 64] = 0.f;
    f32x16 out[2];
    const auto store = [&](u16* p, long long ld, bool on, bool live, float c) {
        if (!on) return;
        if (!live) { zero16(out[0]); zero16(out[1]); }
        store_row(out, p + x * ld, lane, c);
    };
    const auto apply = [&](const u16* tile, const f32x16& w) {
        zero16(out[0]); zero16(out[1]);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const bf16x8 f = pack_acc(w, kk), rest = pack_rest(w, f, kk);
#pragma unroll
            for (int dt = 0; dt < 2; ++dt) {
                const bf16x8 c = frag_cols(tile, 16 * kk, dt, lane);
                out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(c, f, out[dt], 0, 0, 0);
                out[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(c, rest, out[dt], 0, 0, 0);
            }
        }
    };
    apply(Kt, s);
    store(a.dq + t.q0 * a.lddq + h * 64, a.lddq, x < t.lq, true, a.scale);
    __syncthreads();
    // lane = key
    zero16(s); zero16(dp);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf[kk], kf[kk], s, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(gf[kk], vf[kk], dp, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int i = acc_r(r, lane);
        const float p = keep ? __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, bl[31 + x - i]) - ls[i]) : 0.f;
        s[r] = p;
        dp[r] = keep ? p * (dp[r] - Ds[i]) : 0.f;
    }
    apply(Gt, s);
    store(a.dv + t.k0 * a.lddk + h * 64, a.lddk, x < t.lk, keep, 1.f);
    diag_add(dp, dgs + 64, lane);                              // (distances -48 .. 31: what lies below -31 is zero)
    apply(Qt, dp);
    store(a.dk + t.k0 * a.lddk + h * 64, a.lddk, x < t.lk, keep, a.scale);
    __syncthreads();
    part[lane] = dgs[lane + 32];
}
// ---- joins of the parts: a wave per (row, head), a lane per d
__global__ __launch_bounds__(256) void cfl_relpos_join_kernel(const float* __restrict__ po, const float* __restrict__ pm, int ns, int heads,
                                                              long long rows, long long last, const int* __restrict__ end, u16* o, long long ldo,
                                                              float* __restrict__ lse) {
    const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const long long row = i / heads, h = i % heads;
    if (row >= min(rows, end ? (long long)max(*end, 0) : last)) return;
    float m = -INFINITY;
    for (int s = 0; s < ns; ++s) m = fmaxf(m, pm[2 * ((s * heads + h) * rows + row)]);
    float l = 0.f, x = 0.f;
    for (int s = 0; s < ns; ++s) {
        const long long at = (s * heads + h) * rows + row;
        const float ms = pm[2 * at], c = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - m);
        l = fmaf(pm[2 * at + 1], c, l);
        if (c != 0.f) x = fmaf(po[at * 64 + lane], c, x);
    }
    reinterpret_cast<__bf16*>(o)[row * ldo + h * 64 + lane] = (__bf16)(m == -INFINITY ? 0.f : x / l);
    if (lse && lane == 0) lse[h * rows + row] = m == -INFINITY ? INFINITY : m + __builtin_amdgcn_logf(l);
}
__global__ __launch_bounds__(256) void cfl_relpos_join_sum_kernel(const float* __restrict__ po, int ns, int heads, long long rows, long long last,
                                                                  const int* __restrict__ end, float scale, u16* o, long long ldo,
                                                                  const float* __restrict__ pr, float* dsum) {
    const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const long long row = i / heads, h = i % heads;
    if (row >= min(rows, end ? (long long)max(*end, 0) : last)) return;
    float x = 0.f;
    for (int s = 0; s < ns; ++s) x += po[((s * heads + h) * rows + row) * 64 + lane];
    reinterpret_cast<__bf16*>(o)[row * ldo + h * 64 + lane] = (__bf16)(x * scale);
    if (dsum && lane == 0) {
        float y = 0.f;
        for (int s = 0; s < ns; ++s) y += pr[(s * heads + h) * rows + row];
        dsum[h * rows + row] += y;
    }
}

// ---- the bias gradient from part [heads][slots][nd] (place i: distance i - mid): sums of 64 distances over `per` slots, then of these every
// bucket's share, in a fixed order.  grid = (heads, ceil(nd / 64), ceil(slots / per)), 64 distances x 16 strands of slots.  One workgroup a
// head: that is the table's gradient; more: share [heads][workgroups][nb], which a launch of its own adds up in order (4 us; the last
// workgroup doing it would need a fence that writes back and drops whole caches, 30 us).
__device__ __forceinline__ void put_dtable(void* dtable, int bf16, long long at, float v) {
    if (bf16) ((__bf16*)dtable)[at] = (__bf16)v;
    else ((float*)dtable)[at] = v;
}
__global__ __launch_bounds__(1024) void cfl_relpos_dtable_kernel(const float* __restrict__ part, int nd, int mid, long long slots, int per,
                                                                 const int* __restrict__ bucket, int R, int nb, int heads, float* share,
                                                                 void* dtable, int bf16) {
    __shared__ float red[16][64];
    __shared__ int bk[64];
    const int h = blockIdx.x, lane = threadIdx.x & 63, strand = threadIdx.x >> 6, i = blockIdx.y * 64 + lane;
    if (strand == 0) bk[lane] = i < nd ? min(max(bucket[min(max(i - mid, -R), R) + R], 0), nb - 1) : -1;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (i < nd) {
        const float* p = part + (long long)h * slots * nd + i;
        const long long last = min(slots, (long long)(blockIdx.z + 1) * per);
        long long s = (long long)blockIdx.z * per + strand;
        for (; s + 112 < last; s += 128) {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] += p[(s + 16 * k) * nd];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (s + 16 * k < last) x[k] += p[(s + 16 * k) * nd];
    }
    red[strand][lane] = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    __syncthreads();
    if (strand == 0) {
        float y = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) y += red[k][lane];
        red[0][lane] = y;                                      // (its own place)
    }
    __syncthreads();
    int L = 16;                                                // lanes a bucket
    while (L > 1 && (long long)nb * L > 1024) L >>= 1;
    for (int b0 = 0; b0 < nb; b0 += 1024 / L) {
        const int b = b0 + threadIdx.x / L;
        float y = 0.f;
        for (int k = threadIdx.x & (L - 1); k < 64; k += L) y += bk[k] == b ? red[0][k] : 0.f;
        for (int o = L >> 1; o > 0; o >>= 1) y += __shfl_xor(y, o, 64);
        if (b < nb && (threadIdx.x & (L - 1)) == 0) {
            if (share) share[(((long long)h * gridDim.z + blockIdx.z) * gridDim.y + blockIdx.y) * nb + b] = y;
            else put_dtable(dtable, bf16, (long long)b * heads + h, y);
        }
    }
}
// share [heads][all][nb] -> dtable; L lanes of a wave to a bucket, as above
__global__ __launch_bounds__(1024) void cfl_relpos_dtable_join_kernel(const float* __restrict__ share, int all, int nb, int heads, void* dtable,
                                                                      int bf16) {
    const int h = blockIdx.x;
    int L = 16;
    while (L > 1 && (long long)nb * L > 1024) L >>= 1;
    for (int b0 = 0; b0 < nb; b0 += 1024 / L) {
        const int b = b0 + threadIdx.x / L;
        float y = 0.f;
        if (b < nb)
            for (int k = threadIdx.x & (L - 1); k < all; k += L) y += share[((long long)h * all + k) * nb + b];
        for (int o = L >> 1; o > 0; o >>= 1) y += __shfl_xor(y, o, 64);
        if (b < nb && (threadIdx.x & (L - 1)) == 0) put_dtable(dtable, bf16, (long long)b * heads + h, y);
    }
}

// Launch shape for `L` rows that waves own (32 each) against `K` rows that are passed over, for every (text, head).  Each rule with both sides
// measured, forward / backward in microseconds:
//   texts of at most 32 tokens by their own backward kernel: 256 x 32 tokens x 12 heads 30 against 47
//   the long axis split: one text of 8192 tokens, one head 46 / 117 against 171 / 507, of 2048 tokens x 4 heads 22 / 60 against 46 / 135 (until
//   every SIMD has two waves instead of one: 43 / 116 and 27 / 60)
//   four waves a workgroup: 32 x 512 x 12 42 / 144 against 65 / 208, one text of 1000 tokens, one head 14.8 / 44 against 15.9 / 49, 64 x 33 x 12 and less
//   tie; their tiles of 64 rows against 32: 2 x 4096 x 12 129 / 420 against 141 / 466
struct Shape { int nw, kt, blocks, ns; bool small; };
inline Shape rp_shape(long long BH, int L, int K) {
    Shape p;
    p.small = L <= 32 && K <= 32;
    const long long waves = BH * cfl_cdiv(L, 32);
    // few waves against a long axis: split it, into parts of 256 rows at least, until every SIMD has a wave
    long long ns = 1024 / waves;
    const int most = K / 256 < 16 ? K / 256 : 16;
    p.ns = (int)(ns > most ? most : ns);
    if (p.ns < 1) p.ns = 1;
    p.nw = L > 32 ? 4 : 1;                                     // four waves share what is staged
    p.kt = p.nw == 1 || K <= 32 ? 32 : 64;
    p.blocks = cfl_cdiv(L, 32 * p.nw);
    return p;
}

inline int rp_check(const RpArgs& a, int head_dim) {
    if (!a.q || !a.k || !a.v || !a.table || !a.bucket || a.B < 1 || a.Lq < 0 || a.Lk < 1 || a.heads < 1 || a.nb < 1 || a.R < 0 ||
        (a.cu ? a.T < 1 || a.mask != nullptr : a.Lq < 1)) return CFL_EINVAL;
    if (a.ldq >= 1 << 24 || a.ldk >= 1 << 24 || a.ldo >= 1 << 24) return CFL_ELIMIT;
    if (a.ldq < 64 * a.heads || a.ldk < 64 * a.heads || a.ldo < 64 * a.heads) return CFL_EINVAL;
    if (a.ldq % 8 || a.ldk % 8 || a.ldo % 8 || (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v) & 15)) return CFL_EALIGN;
    const int L = a.Lq > a.Lk ? a.Lq : a.Lk;
    if (head_dim != 64 || a.R > MAXR || a.heads > 65535 || a.nb > 65535 ||
        (long long)a.B * a.heads * (cfl_cdiv(L, 32) + 16) > 0x7fffffffll) return CFL_ELIMIT;
    return 0;
}

#define RP_LAUNCH(ID, KERN, P, LDS1, ...)                                                                                              \
    do {                                                                                                                               \
        const dim3 grid_((unsigned)((long long)a.B * a.heads * (P).blocks * (P).ns));                                                  \
        if ((P).nw == 1) { CFL_LAUNCH(ID, (KERN<1, 32, 2>), grid_, dim3(64), LDS1(1), stream, __VA_ARGS__); }                          \
        else if ((P).kt == 64) { CFL_LAUNCH(ID, (KERN<4, 64, 2>), grid_, dim3(256), LDS1(4), stream, __VA_ARGS__); }                   \
        else { CFL_LAUNCH(ID, (KERN<4, 32, 1>), grid_, dim3(256), LDS1(4), stream, __VA_ARGS__); }                                     \
    } while (0)

inline int rp_nd(int R) { return 2 * (R + BPAD) + 1; }
inline size_t rp_part_bytes(const Shape& p, int heads, long long rows) {
    return p.ns > 1 ? cfl_align256((size_t)p.ns * heads * rows * 64 * 4) : 0;
}

// slots a workgroup of the table's last sums takes: 512, by at most 1024 workgroups (one query of each of 446 texts of 1959 tokens, one head: 7136
// slots take 44 us as one)
inline int rp_per(long long slots) {
    const long long parts = (slots + 511) / 512;
    return (int)((slots + (parts < 1024 ? parts : 1024) - 1) / (parts < 1024 ? parts : 1024));
}
inline size_t rp_share_bytes(int heads, int nd, long long slots, int nb) {
    return cfl_align256((size_t)heads * cfl_cdiv(nd, 64) * cfl_cdiv(slots, rp_per(slots)) * nb * 4);
}
inline size_t rp_row_bytes(const Shape& p, int heads, long long rows) { return p.ns > 1 ? cfl_align256((size_t)p.ns * heads * rows * 4) : 0; }

}  // namespace

extern "C" {

size_t cfl_relpos_fwd_ws_bytes(int B, int Lq, int Lk, int T, int heads) {
    if (B < 1 || Lq < 0 || Lk < 1 || T < 0 || heads < 1 || (Lq == 0 && T == 0)) return 0;
    const Shape p = rp_shape((long long)B * heads, Lq ? Lq : Lk, Lk);
    const long long rows = Lq ? (long long)B * Lq : T;
    return p.ns > 1 ? rp_part_bytes(p, heads, rows) + (size_t)p.ns * heads * rows * 2 * 4 : 0;
}

size_t cfl_relpos_bwd_ws_bytes(int B, int Lq, int Lk, int T, int heads, int nb, int R) {
    if (B < 1 || Lq < 0 || Lk < 1 || T < 0 || heads < 1 || nb < 1 || R < 0 || R > MAXR || (Lq == 0 && T == 0)) return 0;
    const Shape p = rp_shape((long long)B * heads, Lq ? Lq : Lk, Lk), k = rp_shape((long long)B * heads, Lk, Lq ? Lq : Lk);
    const long long rows = Lq ? (long long)B * Lq : T, krows = T ? T : (long long)B * Lk;
    if (p.small) return cfl_align256((size_t)B * heads * 64 * 4) + rp_share_bytes(heads, 64, B, nb);
    return cfl_align256((size_t)B * heads * k.blocks * k.ns * (2 * R + 1) * 4) +
           rp_share_bytes(heads, 2 * R + 1, (long long)B * k.blocks * k.ns, nb) + rp_row_bytes(p, heads, rows) + rp_part_bytes(p, heads, rows) + 2 * rp_part_bytes(k, heads, krows);
}

int cfl_relpos_fwd(const void* q, long long ldq, const void* k, const void* v, long long ldk, const unsigned char* mask, const int* cu,
                   int B, int Lq, int Lk, int T, int heads, int head_dim, float scale, const void* table, int table_bf16, int nb,
                   const int* bucket, int R, void* o, long long ldo, float* lse, void* ws, void* stream_) {
    RpArgs a{};
    a.q = (const u16*)q; a.k = (const u16*)k; a.v = (const u16*)v; a.ldq = ldq; a.ldk = ldk; a.ldo = ldo; a.out = (u16*)o;
    a.mask = mask; a.cu = cu; a.B = B; a.Lq = Lq; a.Lk = Lk; a.T = T; a.heads = heads; a.scale = scale; a.scale2 = scale * LOG2E;
    a.table = table; a.table_bf16 = table_bf16; a.nb = nb; a.R = R; a.bucket = bucket; a.lse = lse;
    a.rows = Lq ? (long long)B * Lq : T;
    const int rc = rp_check(a, head_dim);
    if (rc) return rc;
    const Shape p = rp_shape((long long)B * heads, Lq ? Lq : Lk, Lk);
    if (!o || (p.ns > 1 && !ws)) return CFL_EINVAL;
    if ((uintptr_t)o & 15) return CFL_EALIGN;
    hipStream_t stream = (hipStream_t)stream_;
    a.nqb = p.blocks; a.ns = p.ns;
    a.po = (float*)ws;
    a.pm = p.ns > 1 ? (float*)((char*)ws + rp_part_bytes(p, heads, a.rows)) : nullptr;
    const size_t lds = (size_t)rp_nd(R) * 4;
#define RP_LDS(NW) lds
    if (p.small)
        CFL_LAUNCH(K_RELPOS_FWD, (cfl_relpos_fwd_kernel<1, 32, 1>), dim3((unsigned)(B * heads)), dim3(64), lds, stream, a);
    else
        RP_LAUNCH(K_RELPOS_FWD, cfl_relpos_fwd_kernel, p, RP_LDS, a);
#undef RP_LDS
    if (p.ns > 1)
        CFL_LAUNCH(K_RELPOS_JOIN, cfl_relpos_join_kernel, dim3((unsigned)((a.rows * heads + 3) / 4)), dim3(256), 0, stream, a.po, a.pm, p.ns, heads,
                   a.rows, a.rows, cu && !Lq ? cu + B : (const int*)nullptr, (u16*)o, ldo, lse);
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
    a.krows = cu ? T : (long long)B * Lk;
    const int rc = rp_check(a, head_dim);
    if (rc) return rc;
    if (!o || !dout || !lse || !dsum || !dq || !dk || !dv || !dtable || !ws) return CFL_EINVAL;
    if (lddq % 8 || lddk % 8 || (((uintptr_t)o | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15)) return CFL_EALIGN;
    hipStream_t stream = (hipStream_t)stream_;
    const int L = Lq ? Lq : Lk;
    const Shape p = rp_shape((long long)B * heads, L, Lk), kp = rp_shape((long long)B * heads, Lk, L);
    const size_t bl = (size_t)rp_nd(R) * 4;
    char* at = (char*)ws;
    a.diag = (float*)at;
    const int nd = p.small ? 64 : 2 * R + 1;
    const long long slots = p.small ? B : (long long)B * kp.blocks * kp.ns;
    const dim3 tg(heads, cfl_cdiv(nd, 64), (unsigned)cfl_cdiv(slots, rp_per(slots)));
    at += cfl_align256((size_t)heads * slots * nd * 4);
    float* share = tg.y * tg.z > 1 ? (float*)at : nullptr;
    at += rp_share_bytes(heads, nd, slots, nb);
#define RP_TABLE()                                                                                                                             \
    CFL_LAUNCH(K_RELPOS_DTABLE, cfl_relpos_dtable_kernel, tg, dim3(1024), 0, stream, a.diag, nd, p.small ? 32 : R, slots, rp_per(slots),       \
               bucket, R, nb, heads, share, dtable, table_bf16);                                                                               \
    if (share)                                                                                                                                 \
        CFL_LAUNCH(K_RELPOS_DTABLE_JOIN, cfl_relpos_dtable_join_kernel, dim3(heads), dim3(1024), 0, stream, share, (int)(tg.y * tg.z), nb,     \
                   heads, dtable, table_bf16)
    if (p.small) {
        a.ns = 1;
        CFL_LAUNCH(K_RELPOS_BWD32, cfl_relpos_bwd32_kernel, dim3((unsigned)(B * heads)), dim3(64), 0, stream, a);
        RP_TABLE();
        return 0;
    }
    a.pr = (float*)at;
    at += rp_row_bytes(p, heads, a.rows);
    a.po = (float*)at;
    at += rp_part_bytes(p, heads, a.rows);
    a.nqb = p.blocks; a.ns = p.ns;
#define RP_LDS(NW) bl
    RP_LAUNCH(K_RELPOS_DQ, cfl_relpos_dq_kernel, p, RP_LDS, a);
#undef RP_LDS
    const int* qend = cu && !Lq ? cu + B : nullptr;
    if (p.ns > 1)
        CFL_LAUNCH(K_RELPOS_JOIN, cfl_relpos_join_sum_kernel, dim3((unsigned)((a.rows * heads + 3) / 4)), dim3(256), 0, stream, a.po, p.ns, heads,
                   a.rows, a.rows, qend, scale, (u16*)dq, lddq, a.pr, dsum);
    a.po = (float*)at;
    a.pv = (float*)(at + rp_part_bytes(kp, heads, a.krows));
    a.ns = kp.ns;
#define RP_LDS(NW) bl * (1 + (NW)) + 64 * 4
    RP_LAUNCH(K_RELPOS_DKV, cfl_relpos_dkv_kernel, kp, RP_LDS, a, kp.blocks);
#undef RP_LDS
    RP_TABLE();
#undef RP_TABLE
    if (kp.ns > 1) {
        const dim3 g((unsigned)((a.krows * heads + 3) / 4));
        const int* kend = cu ? cu + B : nullptr;
        CFL_LAUNCH(K_RELPOS_JOIN, cfl_relpos_join_sum_kernel, g, dim3(256), 0, stream, a.po, kp.ns, heads, a.krows, a.krows, kend, scale, (u16*)dk,
                   lddk, (const float*)nullptr, (float*)nullptr);
        CFL_LAUNCH(K_RELPOS_JOIN, cfl_relpos_join_sum_kernel, g, dim3(256), 0, stream, a.pv, kp.ns, heads, a.krows, a.krows, kend, 1.f, (u16*)dv,
                   lddk, (const float*)nullptr, (float*)nullptr);
    }
    return 0;
}

}  // extern "C"
