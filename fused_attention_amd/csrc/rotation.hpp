// Rotating 16 values by rows of the rotary tables: what the rotation of queries and keys and the appending of rotary keys share.
//
// Every product and every sum is rounded to float32 by itself, as where keys are rotated on their way into the 8-bit cache, so that the
// same tables give the same 16-bit values by either way.
#pragma once

#include "cache_kernels.hpp"

namespace fa {
namespace rotary {

using cache::Elem;
using cache::Pairs;

// Eight pairs of a row of the tables.
struct Turn {
    float cos[8], sin[8];
};

__device__ __forceinline__ Turn load_turn(const float* cos, const float* sin, bool inverse) {
    const floatx4 c0 = reinterpret_cast<const floatx4*>(cos)[0], c1 = reinterpret_cast<const floatx4*>(cos)[1];
    const floatx4 s0 = reinterpret_cast<const floatx4*>(sin)[0], s1 = reinterpret_cast<const floatx4*>(sin)[1];
    Turn t;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        t.cos[j] = c0[j], t.cos[4 + j] = c1[j];
        t.sin[j] = inverse ? -s0[j] : s0[j], t.sin[4 + j] = inverse ? -s1[j] : s1[j];
    }
    return t;
}

// Sixteen values that are eight pairs, from two loads of 16 bytes and back into two stores: the first values and, further on, the second
// ones; or pairs as neighbours.
template <bool BF, bool IL>
__device__ __forceinline__ void turn_pairs(u32x4& lo, u32x4& hi, const Turn& t) {
    Pairs x;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t w = IL ? (j < 4 ? lo[j & 3] : hi[j & 3]) : lo[j / 2], v = IL ? w : hi[j / 2];
        x.a[j] = Elem<BF>::to_float((uint16_t)(IL ? w : w >> (16 * (j & 1))));
        x.b[j] = Elem<BF>::to_float((uint16_t)(IL ? v >> 16 : v >> (16 * (j & 1))));
    }
    cache::rotate(x, t.cos, t.sin);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        lo[j] = IL ? Elem<BF>::pack(x.a[j], x.b[j]) : Elem<BF>::pack(x.a[2 * j], x.a[2 * j + 1]);
        hi[j] = IL ? Elem<BF>::pack(x.a[4 + j], x.b[4 + j]) : Elem<BF>::pack(x.b[2 * j], x.b[2 * j + 1]);
    }
}

}  // namespace rotary
}  // namespace fa
