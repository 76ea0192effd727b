// Kernels of the paged key/value cache for gfx950 (MI355X, CDNA4): appending tokens to it, attention over it, and the
// selection of pages by a cheap score.  No counterpart in the reference, whose keys and values are the call's own
// (reference src/fused_attn_extention.cu:15-22).
//
// The cache holds keys and values in 8 bits (e4m3) as [pages, heads, P tokens, H], with one power of two for each page and
// head: value = code * 2^exponent.  A power of two, because codes then move to a larger exponent without rounding as long as
// they stay normal numbers, and because it costs nothing to apply: the keys' goes into the factor of the scores, the values'
// is an operand of the conversion to 16 bits.  A page of one head is contiguous, P * H bytes, and a group of 16 tokens (a
// "sub-tile", the edge of the matrix instruction's tile) never crosses a page, because P is a multiple of 16.
#pragma once

#include "fused_attn_kernel.hpp"

namespace fa {
namespace cache {

constexpr int kSub = 16;                 // tokens of a sub-tile
constexpr int kLeastExponent = -80;      // of a page of zeros; 448 * 2^-80 is below any 16-bit value that matters

// The cache and the call's sequences, as the kernels see them.  Numbers that come from device memory (pages, starts,
// lengths) are checked where they are read: a page outside [0, pages) is no page.
struct View {
    uint8_t* k;
    uint8_t* v;
    int8_t* k_exponents;
    int8_t* v_exponents;
    int8_t* bounds;            // [pages, heads, 2, H]: largest and smallest key of each channel, or nullptr
    const int32_t* table;      // [B, W]
    int64_t table_stride;
    const int32_t* starts;     // [B]
    const int32_t* new_lens;   // [B] or nullptr
    int B, L, R, Rkv, W, pages;
    int log2_p;
    int group;                 // query heads of a key head

    __device__ __forceinline__ int page_size() const { return 1 << log2_p; }
    __device__ __forceinline__ int tokens(int b) const {
        if (new_lens == nullptr) return L;
        const int n = new_lens[b];
        return n < 0 ? 0 : n > L ? L : n;
    }
    // the page of the b-th sequence's tokens w P .. w P + P - 1, or -1
    __device__ __forceinline__ int page_of(int b, int w) const {
        const int page = table[b * table_stride + w];
        return (uint32_t)page < (uint32_t)pages ? page : -1;
    }
};

struct Strides3 {
    int64_t b, h, l;
};

template <bool BF>
struct Elem;
template <>
struct Elem<false> {
    static __device__ __forceinline__ float to_float(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ __forceinline__ uint16_t from_float(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {   // v_cvt_pk_f16_f32: to nearest, unlike pack_rtz
        const half2v p = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, p);
    }
    template <bool HI>
    static __device__ __forceinline__ uint32_t codes(uint32_t x, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, HI));
    }
    static __device__ __forceinline__ floatx4 mfma(u32x4 a, u32x4 b, floatx4 c) {
        return fa::mfma16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c);
    }
};
template <>
struct Elem<true> {
    static __device__ __forceinline__ float to_float(uint16_t x) { return __builtin_bit_cast(float, (uint32_t)x << 16); }
    static __device__ __forceinline__ uint16_t from_float(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return fa::bf16::pack_pair(a, b); }
    template <bool HI>
    static __device__ __forceinline__ uint32_t codes(uint32_t x, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, HI));
    }
    static __device__ __forceinline__ floatx4 mfma(u32x4 a, u32x4 b, floatx4 c) {
        return fa::bf16::mfma16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c);
    }
};

__device__ __forceinline__ float quad_sum(float x) {
    const uint32_t xb = __builtin_bit_cast(uint32_t, x);
    const u32x2 r = __builtin_amdgcn_permlane16_swap(xb, xb, false, false);
    const uint32_t r0 = r[0], r1 = r[1];
    return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}

// Of a wave's lanes: up to and with this one, and all.  Within rows of 16 lanes by 1, 2, 4 and 8, then the last lane of the first and third
// row to the next, and of the second to the upper half; by way of LDS, six exchanges one after the other took 0.3 us.
__device__ __forceinline__ int wave_sums(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_sums(x), 63); }

// Between LDS accesses of the lanes of one wave to each other's places.  LDS serves a wave in order, so that nothing has to wait: this
// keeps the compiler from exchanging them, and is no instruction.
__device__ __forceinline__ void lanes_in_order() {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }   // e in [-126, 127]

__device__ __forceinline__ bool is_finite(float x) { return (__builtin_bit_cast(uint32_t, x) & 0x7f800000u) != 0x7f800000u; }

// The smallest e with amax <= 448 * 2^e, not below kLeastExponent (448 = 0.875 * 2^9; amax = m * 2^ex, m in [0.5, 1)).
__device__ __forceinline__ int exponent_of(float amax) {
    if (!(amax > 0.f)) return kLeastExponent;
    const int ex = __builtin_amdgcn_frexp_expf(amax);
    const int e = __builtin_amdgcn_frexp_mantf(amax) <= 0.875f ? ex - 9 : ex - 8;
    return e < kLeastExponent ? kLeastExponent : e;
}

#include "cache_append.inc"
#include "cache_attend.inc"
#include "cache_select.inc"

}  // namespace cache
}  // namespace fa
