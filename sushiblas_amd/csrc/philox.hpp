// philox.hpp -- Philox4x32-10, the counter-based generator of Salmon et al.
// (SC'11), shared by the fills and the dropout.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sbx {

// The four words of counter (c0, c1, c2, c3) under the key `seed`.
__device__ inline void philox4x32(uint64_t seed, uint32_t c0, uint32_t c1, uint32_t c2,
                                  uint32_t c3, uint32_t (&w)[4])
{
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

}  // namespace sbx
