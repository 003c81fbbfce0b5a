// rng.h -- the counter-based keep flags of the dropout kernels (csrc/bertfuse.hip, csrc/dropout.hip): a flag is a hash of (seed,
// element index), recomputed wherever it is needed and never stored.
#pragma once
#include "common.h"
#include "colmap.h"

namespace {

__device__ __forceinline__ u32 mix32(u32 seed, u32 i) {
    u32 h = (i * 0x9E3779B1u) ^ seed;
    h ^= h >> 16; h *= 0x85EBCA6Bu; h ^= h >> 13; h *= 0xC2B2AE35u; h ^= h >> 16;
    return h;
}
// Steps replayed from a HIP graph: the host's per-call seed is a constant of the graph, so the masks would repeat every step.  With a
// step tick on the device (cfl_set_dropout_tick; the caller increments it on the stream once per step) the effective seed of a launch is
// seed + tick * odd constant: forward and backward of one step read the same tick, successive replays different ones.
__device__ __forceinline__ u32 tick_seed(u32 seed, const u32* __restrict__ tick) {
    return tick ? seed + *tick * 0x85EBCA6Bu : seed;
}
// keep flags of the 4 consecutive elements starting at element index e (e % 4 == 0): 16 random bits per element
__device__ __forceinline__ void keep4(u32 seed, long long e, u32 thr16, bool (&k)[4]) {
    const u32 i = (u32)(e >> 1);
    const u32 s2 = seed + (u32)(e >> 33) * 0x632BE5ABu;
    const u32 h0 = mix32(s2, i), h1 = mix32(s2, i + 1);
    k[0] = (h0 & 0xffffu) >= thr16; k[1] = (h0 >> 16) >= thr16;
    k[2] = (h1 & 0xffffu) >= thr16; k[3] = (h1 >> 16) >= thr16;
}

}  // namespace
