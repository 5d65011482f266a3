// philox.h -- the counter-based generator behind every draw of the HIP kernels (replay indices, exploration and smoothing noise, dropout masks).
#ifndef PLEN_PHILOX_H
#define PLEN_PHILOX_H
#include <stdint.h>

// ---- counter-based random numbers (Philox4x32-10, Salmon et al. 2011) so that the captured graphs need no library RNG call (each costs a
//      draw kernel plus a fill of the generator's offset tensor per graph replay).  rng = device uint64[2] {seed, calls so far}; a kernel reads
//      the call counter at its start and a LATER kernel of the same stream bumps it, so every launch sees one consistent value.
//      PHILOX_XOR3: a file may bring its own three-way exclusive or.
//      Element i of draw `tag` of call c gets the 4 words philox(counter = (i, c_lo, c_hi, tag), key = seed).
#ifndef PHILOX_XOR3
#define PHILOX_XOR3(a, b, c) ((a) ^ (b) ^ (c))
#endif
struct u4 { uint32_t x, y, z, w; };
static __device__ __forceinline__ u4 philox4x32(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        const uint32_t n0 = PHILOX_XOR3((uint32_t)(p1 >> 32), c1, k0), n2 = PHILOX_XOR3((uint32_t)(p0 >> 32), c3, k1);
        c1 = (uint32_t)p1; c3 = (uint32_t)p0; c0 = n0; c2 = n2;
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    return u4{c0, c1, c2, c3};
}

#endif
