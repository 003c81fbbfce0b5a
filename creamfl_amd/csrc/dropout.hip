// dropout.hip -- element-wise dropout of an activation from the counter-based generator of rng.h; the mask is never stored.
//
//   y_e = keep(e) ? x_e / (1 - p') : 0,    keep(e) = (16 random bits of (seed, e)) >= thr,   thr = round(65536 p),  p' = thr / 65536
//
// Where it sits: the embeddings' dropout of the BertModel at src/networks/models/pcme.py:36-38 (BertEmbeddings of the third-party
// `transformers`, restated from its published definition).  The backward is the same map on the gradient, with the seed the forward
// used: a launch may draw its seed from the device (the captured steps' tick, cfl_set_dropout_tick), so the forward leaves the
// effective seed in a word of memory and the backward reads it from there -- also when the tick has moved on in between.
// HBM-bound: one read and one write per element; 131072 x 768 bf16 in 72 us (5.6 TB/s; 5.75 at two to eight times the size, where a library copy
// reaches 5.0 to 5.4), 24 x 256 in 4 us of launch.
#include "common.h"
#include "colmap.h"
#include "rng.h"
#include <math.h>

const unsigned* cfl_dropout_tick_ptr();                // bertfuse.hip

namespace {

// 16 bytes per access and U accesses in flight per thread; the flags are formed while the loads travel (one mix32 per two elements: at
// 131072 x 768 bf16 the hashes alone are a quarter of the memory's time).  Elements behind the last whole access: the last workgroup.
template <class T, int U>
__global__ __launch_bounds__(256) void cfl_dropout_kernel(const T* __restrict__ x, long long n, u32 thr, float scale, u32 seed,
                                                          const u32* __restrict__ tick, const u32* __restrict__ seed_dev,
                                                          T* __restrict__ y, u32* __restrict__ seed_used) {
    constexpr int VE = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(VE)));
    const long long nv = n / VE, v0 = (long long)blockIdx.x * 256 * U + threadIdx.x;
    vec in[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (v0 + u * 256 < nv) in[u] = reinterpret_cast<const vec*>(x)[v0 + u * 256];
    seed = seed_dev ? *seed_dev : tick_seed(seed, tick);
    if (seed_used && v0 == 0) *seed_used = seed;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long v = v0 + u * 256;
        if (v < nv) {
            vec out;
#pragma unroll
            for (int j = 0; j < VE / 2; ++j) {
                const long long i = v * (VE / 2) + j;
                const u32 h = mix32(seed + (u32)(i >> 32) * 0x632BE5ABu, (u32)i);
                out[2 * j] = (h & 0xffffu) >= thr ? (T)((float)in[u][2 * j] * scale) : (T)0.f;
                out[2 * j + 1] = (h >> 16) >= thr ? (T)((float)in[u][2 * j + 1] * scale) : (T)0.f;
            }
            reinterpret_cast<vec*>(y)[v] = out;
        }
    }
    const long long e = nv * VE + threadIdx.x;
    if (blockIdx.x == gridDim.x - 1 && e < n) {
        const long long i = e >> 1;
        const u32 h = mix32(seed + (u32)(i >> 32) * 0x632BE5ABu, (u32)i);
        y[e] = ((e & 1) ? h >> 16 : h & 0xffffu) >= thr ? (T)((float)x[e] * scale) : (T)0.f;
    }
}
// Any alignment: a pair of elements per thread and step.
template <class T>
__global__ __launch_bounds__(256) void cfl_dropout_pairs_kernel(const T* __restrict__ x, long long n, u32 thr, float scale, u32 seed,
                                                                const u32* __restrict__ tick, const u32* __restrict__ seed_dev,
                                                                T* __restrict__ y, u32* __restrict__ seed_used) {
    seed = seed_dev ? *seed_dev : tick_seed(seed, tick);
    const long long t0 = (long long)blockIdx.x * 256 + threadIdx.x;
    if (seed_used && t0 == 0) *seed_used = seed;
    const long long step = (long long)gridDim.x * 256;
    for (long long i = t0; 2 * i < n; i += step) {
        const u32 h = mix32(seed + (u32)(i >> 32) * 0x632BE5ABu, (u32)i);
        const long long e = 2 * i;
        y[e] = (h & 0xffffu) >= thr ? (T)((float)x[e] * scale) : (T)0.f;
        if (e + 1 < n) y[e + 1] = (h >> 16) >= thr ? (T)((float)x[e + 1] * scale) : (T)0.f;
    }
}

template <class T>
int drop_launch(const void* x, long long n, u32 thr, float scale, u32 seed, const u32* seed_dev, void* y, u32* seed_used, hipStream_t stream) {
    const u32* tick = cfl_dropout_tick_ptr();
    constexpr int U = 4, per = 256 * U * (16 / (int)sizeof(T));
    if ((((uintptr_t)x | (uintptr_t)y) & 15) == 0) {
        CFL_LAUNCH(K_DROPOUT, (cfl_dropout_kernel<T, U>), dim3((unsigned)((n + per - 1) / per)), dim3(256), 0, stream, (const T*)x, n, thr, scale,
                   seed, tick, seed_dev, (T*)y, seed_used);
    } else {
        const long long blocks = ((n + 1) / 2 + 255) / 256;
        CFL_LAUNCH(K_DROPOUT, cfl_dropout_pairs_kernel<T>, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, stream, (const T*)x, n,
                   thr, scale, seed, tick, seed_dev, (T*)y, seed_used);
    }
    return 0;
}

}  // namespace

extern "C" {

int cfl_dropout(const void* x, int dtype, long long n, double p, unsigned seed, const unsigned* seed_dev, void* y,
                unsigned* seed_used, void* stream_) {
    if (!x || !y || n < 1 || dtype < 0 || dtype > 2 || !(p >= 0. && p <= 1.)) return CFL_EINVAL;
    const int size = dtype == 0 ? 4 : 2;
    if (((uintptr_t)x | (uintptr_t)y) % size) return CFL_EALIGN;
    if (n >= (1ll << 40)) return CFL_ELIMIT;
    hipStream_t stream = (hipStream_t)stream_;
    const u32 thr = (u32)rint(p * 65536.);
    const float scale = thr < 65536u ? 65536.f / (float)(65536u - thr) : 0.f;
    if (dtype == 0) return drop_launch<float>(x, n, thr, scale, seed, seed_dev, y, seed_used, stream);
    if (dtype == 1) return drop_launch<__bf16>(x, n, thr, scale, seed, seed_dev, y, seed_used, stream);
    return drop_launch<_Float16>(x, n, thr, scale, seed, seed_dev, y, seed_used, stream);
}

}  // extern "C"
