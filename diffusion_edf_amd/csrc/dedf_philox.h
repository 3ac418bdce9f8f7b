// Philox4x32-10 (Salmon et al., 2011) as the dropout masks use it: key = seed, counter = (c0, c1, offset).  The sampler's noise draws from the same
// generator (dedf_langevin.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dedf {

struct Words { uint32_t w[4]; };

__device__ inline Words dropout_words(uint32_t c0, uint32_t c1, uint64_t offset, uint64_t seed) {
    uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32), k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0; c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1; c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    return Words{{c0, c1, c2, c3}};
}

}  // namespace dedf
