// What the kernels that choose a token share (sampling.cu, logit_rules.cu): the noise of a sampled row and the rule for ties.
#pragma once
#include "common.cuh"

__device__ __forceinline__ uint64_t mix64(uint64_t x) {
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    return x ^ (x >> 31);
}

// The noise of a sampled row is keyed by (seed, request id, output position); vocabulary entry i adds i to the key.
__device__ __forceinline__ uint64_t noise_key(uint64_t seed, int64_t request, int position) {
    const uint64_t key = mix64(seed * 0x9E3779B97F4A7C15ull + (uint64_t)request);
    return mix64(key ^ ((uint64_t)position * 0xD1B54A32D192ED03ull));
}
// logit v of entry i at temperature t > 0 with its Gumbel noise -log(-log(u))
__device__ __forceinline__ float noisy_score(float v, float t, uint64_t key, int i) {
    const uint64_t h = mix64(key + (uint64_t)i);
    const float u = ((float)(h >> 41) + 0.5f) * (1.0f / 8388608.0f);   // 23 bits + 0.5: never 0 or 1
    return v / t - logf(-logf(u));
}

// the larger value wins, the lower index at a tie
__device__ __forceinline__ void take(float& bv, int& bi, float v, int i) {
    if (v > bv || (v == bv && i < bi)) { bv = v; bi = i; }
}
