// dropout.hip -- element-wise dropout of an activation from the counter-based generator of rng.h; the mask is never stored.
//
//   y_e = keep(e) ? x_e / (1 - p') : 0,    keep(e) = (16 random bits of (seed, e)) >= thr,   thr = round(65536 p),  p' = thr / 65536
//
// Where it sits: the embeddings' dropout of the BertModel at src/networks/models/pcme.py:36-38 (BertEmbeddings of the third-party
// `transformers`, restated from its published definition).  The backward is the same map on the gradient, with the seed the forward
// used: a launch may draw its seed from the device (the captured steps' tick, cfl_set_dropout_tick), so the forward leaves the
// effective seed in a word of memory and the backward reads it from there -- also when the tick has moved on in between.
// HBM-bound: one read and one write per element.
#include "common.h"
#include "colmap.h"
#include "rng.h"
#include <math.h>

const unsigned* cfl_dropout_tick_ptr();                // bertfuse.hip

namespace {

typedef unsigned short u16;

template <class T> __device__ __forceinline__ float drop_load(T v);
template <> __device__ __forceinline__ float drop_load<float>(float v) { return v; }
template <> __device__ __forceinline__ float drop_load<_Float16>(_Float16 v) { return (float)v; }
template <> __device__ __forceinline__ float drop_load<__bf16>(__bf16 v) { return (float)v; }

// One pair of elements per thread and step (a pair shares one hash); any alignment.
template <class T>
__global__ __launch_bounds__(256) void cfl_dropout_kernel(const T* __restrict__ x, long long n, u32 thr, float scale, u32 seed,
                                                          const u32* __restrict__ tick, const u32* __restrict__ seed_dev,
                                                          T* __restrict__ y, u32* __restrict__ seed_used) {
    seed = seed_dev ? *seed_dev : tick_seed(seed, tick);
    const long long t0 = (long long)blockIdx.x * 256 + threadIdx.x;
    if (seed_used && t0 == 0) *seed_used = seed;
    const long long step = (long long)gridDim.x * 256;
    for (long long i = t0; 2 * i < n; i += step) {
        const u32 h = mix32(seed + (u32)(i >> 32) * 0x632BE5ABu, (u32)i);
        const long long e = 2 * i;
        y[e] = (h & 0xffffu) >= thr ? (T)(drop_load(x[e]) * scale) : (T)0.f;
        if (e + 1 < n) y[e + 1] = (h >> 16) >= thr ? (T)(drop_load(x[e + 1]) * scale) : (T)0.f;
    }
}

}  // namespace

extern "C" {

int cfl_dropout(const void* x, int dtype, long long n, double p, unsigned seed, const unsigned* seed_dev, void* y,
                unsigned* seed_used, void* stream_) {
    if (!x || !y || n < 1 || dtype < 0 || dtype > 2 || !(p >= 0. && p <= 1.)) return CFL_EINVAL;
    const int size = dtype == 0 ? 4 : 2;
    if (((uintptr_t)x | (uintptr_t)y) % size) return CFL_EALIGN;
    if (n >= (1ll << 48)) return CFL_ELIMIT;
    hipStream_t stream = (hipStream_t)stream_;
    const u32 thr = (u32)rint(p * 65536.);
    const float scale = thr < 65536u ? 65536.f / (float)(65536u - thr) : 0.f;
    long long blocks = ((n + 1) / 2 + 255) / 256;
    if (blocks > 256 * 32) blocks = 256 * 32;
    const u32* tick = cfl_dropout_tick_ptr();
#define CFL_DROP(T)                                                                                                              \
    CFL_LAUNCH(K_DROPOUT, cfl_dropout_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)x, n, thr, scale, seed, \
               tick, seed_dev, (T*)y, seed_used)
    if (dtype == 0) { CFL_DROP(float); }
    else if (dtype == 1) { CFL_DROP(__bf16); }
    else { CFL_DROP(_Float16); }
#undef CFL_DROP
    return 0;
}

}  // extern "C"
