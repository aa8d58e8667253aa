// rng.h — the counter RNG of the per-step kernels (splitmix64), on the device and on the host.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace siren {

// splitmix64 finaliser over (seed, step, i): a stateless counter RNG (the oracle restates it bit for bit)
__host__ __device__ inline uint64_t mix64(uint64_t z) {
    z += 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
__host__ __device__ inline uint64_t rng_key(uint64_t seed, uint64_t step) { return mix64(seed ^ mix64(step)); }
__host__ __device__ inline uint64_t rng64(uint64_t seed, uint64_t step, uint64_t i) {
    return mix64(rng_key(seed, step) + i);
}

}  // namespace siren
