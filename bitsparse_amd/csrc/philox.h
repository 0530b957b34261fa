// Random bits of dropout: Philox 4x32 with 10 rounds (J. K. Salmon, M. A.
// Moraes, R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as 1, 2,
// 3", SC 2011), a function of key and counter alone, so that a backward pass
// forms the forward's mask again and none is stored.
//
// Eight consecutive elements of a row, one chunk, take the 128 bits of one
// counter: element i has half i % 2 of word i / 2.  The mask depends on row and
// column only, not on a row's length, stride or type.
#pragma once

#include "bs_device.h"

namespace bs {

struct DropRule {
    uint32_t key0, key1;        // the seed's words
    uint32_t offset0, offset1;  // the offset's
    const int64_t* at;          // or both of these in memory, [seed, offset]
    uint32_t bound;             // the number that a half below it drops its element, times 65536
    uint32_t mask;              // of the words: all of them, or 0 where everything is dropped, which no bound says
    float keep_scale;           // of those that stay
};

struct DropKey {
    uint32_t k0, k1, c2, c3;
};
__device__ __forceinline__ DropKey drop_key(const DropRule& r)
{
    if (r.at == nullptr) return {r.key0, r.key1, r.offset0, r.offset1};
    const uint64_t s = (uint64_t)r.at[0], o = (uint64_t)r.at[1];
    return {uniform_u32((uint32_t)s), uniform_u32((uint32_t)(s >> 32)), uniform_u32((uint32_t)o), uniform_u32((uint32_t)(o >> 32))};
}

// the eight halves of a chunk
__device__ __forceinline__ uint4 drop_bits(const DropKey& key, uint32_t chunk, uint32_t row)
{
    uint32_t c0 = chunk, c1 = row, c2 = key.c2, c3 = key.c3, k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return uint4{c0, c1, c2, c3};
}

// A chunk's mask.  A half is compared where it lies, in the upper half of a word (the lower ones moved there).
struct DropMask {
    uint32_t w[4];
    __device__ __forceinline__ DropMask(const DropRule& r, const DropKey& key, uint32_t chunk, uint32_t row)
    {
        const uint4 u = drop_bits(key, chunk, row);
        w[0] = u.x & r.mask, w[1] = u.y & r.mask, w[2] = u.z & r.mask, w[3] = u.w & r.mask;
    }
    __device__ __forceinline__ bool kept(const DropRule& r, int e) const { return (e & 1 ? w[e >> 1] : w[e >> 1] << 16) >= r.bound; }
    // v as the dropout leaves it: 0 where it is dropped, whatever it was
    __device__ __forceinline__ float of(const DropRule& r, int e, float v) const { return kept(r, e) ? v * r.keep_scale : 0.f; }
};

// the same of a step without dropout
struct DropNothing {
    __device__ __forceinline__ DropNothing(const DropRule&, const DropKey&, uint32_t, uint32_t) {}
    __device__ __forceinline__ bool kept(const DropRule&, int) const { return true; }
    __device__ __forceinline__ float of(const DropRule&, int, float v) const { return v; }
};

}  // namespace bs
