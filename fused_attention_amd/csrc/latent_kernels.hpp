// Latent attention for gfx950 (MI355X, CDNA4): a paged cache of one latent vector and one rotary key for each token, in 16 bits, and
// attention in the absorbed form, where every query head reads the same latent as key and as value, and in the expanded form, where
// each head has keys and values of its own beside the shared rotary key.  No counterpart in the reference, whose keys and values
// are the call's own, for each head (reference src/fused_attn_extention.cu:15-22).
//
// The products are those of the other attention kernels:
//   S^T = K Q^T         v_mfma_f32_16x16x32_{f16,bf16}: 16 tokens of a sub-tile by 16 query rows, 32 channels a step
//   online softmax      f32
//   O^T += V^T P^T      the same instruction over the 32 tokens of two sub-tiles
// with lane (c, g), c = lane % 16, g = lane / 16, holding of A row c, k = 8 g + j, of B column c, k = 8 g + j, of C column c, rows
// 4 g + i.
//
// LDS holds keys and values as blocks of 16 tokens by 32 channels, 1 KiB, written by one direct-to-LDS load of a wave: lane l brings 16
// bytes of token l / 4, so that four lanes read 64 bytes in a row and the lane's offset is the same for every block.  Which of the four
// quarters lane l brings is (l % 4) ^ quarter_of(l / 16), so that the lanes that LDS serves at once, lanes 0..3, 12..15, 20..23 and 24..27
// of a 16-byte read and so on, and 32 lanes in a row of a transposing one, meet in no bank.  (With l / 16 in its place, as 16 lanes in a
// row would have it, LDS lost half as many cycles again to conflicts as it worked.)
#pragma once

#include "rotation.hpp"

namespace fa {
namespace latent {

using cache::Elem;
using cache::Strides3;
using cache::exp2_fast;
using cache::kNoReference;
using cache::quad_sum;

constexpr int kSub = 16, kBlock = 1024, kKeys = 64;
constexpr int kNowhere = 0x7fffff00;

// The cache and the call's sequences.  Numbers from device memory are checked where they are read.
struct View {
    uint16_t* latents;         // [pages, P, C + DR]
    const int32_t* table;      // [B, W]
    int64_t table_stride;
    const int32_t* starts;     // [B]
    const int32_t* new_lens;   // [B] or nullptr
    int B, L, R, W, pages, log2_p;

    __device__ __forceinline__ int tokens(int b) const {
        if (new_lens == nullptr) return L;
        const int n = new_lens[b];
        return n < 0 ? 0 : n > L ? L : n;
    }
    __device__ __forceinline__ int page_of(int b, int w) const {
        const int page = table[b * table_stride + w];
        return (uint32_t)page < (uint32_t)pages ? page : -1;
    }
};

struct AppendParams : View {
    const uint16_t* c;         // [B, L, C]
    const uint16_t* k;         // [B, L, DR]
    int64_t c_stride_b, c_stride_l, k_stride_b, k_stride_l;
    const uint16_t* q;         // [B, L, R, DR], or nullptr
    uint16_t* q_out;
    Strides3 qs, qo;
    const float* cos;          // [rope_rows, DR / 2], or nullptr
    const float* sin;
    int64_t rope_rows;
    int C, DR;
    int64_t cache_units, q_units;
    Divisor by_units, by_q_units, by_heads, by_tokens;   // division by (C + DR) / 16, DR / 16, R and L
};

// Sixteen values to a thread: of a token's latent, of its rotary key, or of a query head.  Bound by the bytes: 16384 tokens of 512 + 64 with
// 16 query heads of 64, 105 MB, in 18 us, 5.8 TB/s.
template <bool BF, bool IL>
__global__ __launch_bounds__(256) void latent_append_kernel(const AppendParams p) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const bool query = id >= p.cache_units;
    if (query && id - p.cache_units >= p.q_units) return;
    int token, unit, head = 0;
    if (query) {
        const int at = (int)(id - p.cache_units), row = p.by_q_units.of(at);
        unit = at - row * (p.DR / 16);
        token = p.by_heads.of(row);
        head = row - token * p.R;
    } else {
        token = p.by_units.of((int)id);
        unit = (int)id - token * ((p.C + p.DR) / 16);
    }
    const int b = p.by_tokens.of(token), i = token - b * p.L;
    const int64_t pos = (int64_t)p.starts[b] + i;
    const bool exists = i < p.tokens(b) && (p.cos == nullptr || (pos >= 0 && pos < p.rope_rows));
    const bool turned = query || unit >= p.C / 16;
    const uint16_t* from;
    uint16_t* to;
    if (query) {
        from = p.q + b * p.qs.b + head * p.qs.h + i * p.qs.l;
        to = p.q_out + b * p.qo.b + head * p.qo.h + i * p.qo.l;
    } else {
        if (!exists || pos < 0 || pos >= (int64_t)p.W << p.log2_p) return;
        const int page = p.page_of(b, (int)(pos >> p.log2_p));
        if (page < 0) return;
        to = p.latents + (((int64_t)page << p.log2_p) + (pos & ((1 << p.log2_p) - 1))) * (p.C + p.DR);
        from = p.c + b * p.c_stride_b + i * p.c_stride_l;
        if (turned) {
            unit -= p.C / 16;
            to += p.C;
            from = p.k + b * p.k_stride_b + i * p.k_stride_l;
        }
    }
    const bool half = turned && !IL;
    const int c0 = (half ? 8 : 16) * unit, c1 = c0 + (half ? p.DR / 2 : 8);
    u32x4 lo = {}, hi = {};
    if (exists) {
        lo = *reinterpret_cast<const u32x4*>(from + c0);
        hi = *reinterpret_cast<const u32x4*>(from + c1);
        if (turned && p.cos != nullptr) {
            const int64_t entry = pos * (p.DR / 2) + 8 * unit;
            rotary::turn_pairs<BF, IL>(lo, hi, rotary::load_turn(p.cos + entry, p.sin + entry, false));
        }
    }
    *reinterpret_cast<u32x4*>(to + c0) = lo;
    *reinterpret_cast<u32x4*>(to + c1) = hi;
}

// ---- what both attention kernels use ----

// How far a row's largest score may be above the reference of its exponentials before they get a new one, and what they are scaled by,
// in log2 units.  fp16: weights up to 2^15, and full 11 bits down to 2^-22 of the reference's, so that 2^17 keys below that lose 2^-16
// of a row.  bf16 has the exponents of float32.
// Weights are rounded to the cache's type, because the second product's instruction takes 16 bits; their sums are of what they were before.  The output is
// then off by 1.2 to 1.4 times what its own rounding makes of it (relative to 64 bits, bf16: 4096 tokens behind 12288, expanded, 0.0023 where a
// computation in float32 rounded once has 0.0017; 16 x 160 rows over 2000, absorbed, 0.0021 and 0.0017; fp16, 8 x 1001 tokens 0.00026 and 0.00020).
template <bool BF>
constexpr float kLeash = BF ? 16.f : 7.f;
template <bool BF>
constexpr float kBias = BF ? 0.f : 8.f;

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// A value that the compiler does not know to be the one it was: what follows from it is not worked out ahead of a loop and kept through it.
__device__ __forceinline__ int afresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ uint32_t afresh_uniform(uint32_t x) {
    x = __builtin_amdgcn_readfirstlane(x);
    asm volatile("" : "+s"(x));
    return x;
}
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Of the tokens 4 k .. 4 k + 3 of a block: what their quarters' numbers are changed by.
__device__ __forceinline__ int quarter_of(int k) { return (2 * k & 3) ^ (k & 2 ? 3 : 0); }     // 0, 2, 3, 1

// Lane's bytes within a block: as loaded from rows `row_bytes` apart, as an operand of the first product, and as a transposed one of
// the second (channel tiles with an even and an odd number).
__device__ __forceinline__ uint32_t from_row(int lane, uint32_t row_bytes) {
    return (uint32_t)(lane >> 2) * row_bytes + (uint32_t)((lane & 3) ^ quarter_of(lane >> 4)) * 16u;
}
__device__ __forceinline__ int key_at(int lane) {
    const int c = lane & 15, g = lane >> 4;
    return (4 * c + (g ^ quarter_of(c >> 2))) * 16;
}
__device__ __forceinline__ int value_at(int lane, int odd) {
    const int s = lane & 15, g = lane >> 4;
    return ((4 * g + (s >> 2)) * 4 + ((2 * odd + ((s & 3) >> 1)) ^ quarter_of(g))) * 16 + (s & 1) * 8;
}

__device__ __forceinline__ u32x2 read_transposed(const uint8_t* at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((FA_LDS short4v*)(at)));
}

// Whether any of eight 16-bit values is infinite or no number.
template <bool BF>
__device__ __forceinline__ bool not_finite(u32x4 x) {
    constexpr uint32_t kExponent = BF ? 0x7f807f80u : 0x7c007c00u, kOne = BF ? 0x00800080u : 0x04000400u;
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) any |= (x[j] & kExponent) + kOne;
    return (any & 0x80008000u) != 0;
}

// Joins the parts that a row's keys were cut into: WAVES waves a row, of each C / 8 lanes with eight channels, the parts dealt out to
// waves and lane groups and summed in a fixed order.  A part without any key has nothing but its log-sum-exp, -inf.  `part_lse` and
// `part_o`: the first part, the others `stride` rows further on each.
template <int C, bool BF, int WAVES>
__device__ __forceinline__ void join_row(const float* part_lse, const float* part_o, int parts, int64_t stride, uint16_t* out, float* lse) {
    constexpr int kLanes = C / 8, kAtOnce = 64 / kLanes * WAVES;
    __shared__ float exchange[WAVES > 1 ? WAVES : 1][C];
    const int lane = threadIdx.x & 63, wave = WAVES > 1 ? threadIdx.x >> 6 : 0, d = lane % kLanes * 8;
    float top = -__builtin_inff();
    for (int s = lane; s < parts; s += 64) top = fmax2(top, part_lse[s * stride]);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) top = fmax2(top, __shfl_xor(top, s));
    const float less = top == -__builtin_inff() ? 0.f : top;
    float total = 0.f;
    for (int s = lane; s < parts; s += 64) total += exp2_fast(part_lse[s * stride] - less);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) total += __shfl_xor(total, s);
    float y[8] = {};
#pragma unroll 4
    for (int s = wave * (64 / kLanes) + lane / kLanes; s < parts; s += kAtOnce) {
        const float part = part_lse[s * stride], w = exp2_fast(part - less);
        const floatx4* from = reinterpret_cast<const floatx4*>(part_o + s * stride * C + d);
        const floatx4 a = from[0], b = from[1];
        const bool empty = part == -__builtin_inff();    // nothing was written there
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] += empty ? 0.f : w * a[j], y[4 + j] += empty ? 0.f : w * b[j];
    }
#pragma unroll
    for (int s = kLanes; s < 64; s <<= 1)
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] += __shfl_xor(y[j], s);
    if constexpr (WAVES > 1) {
        if (lane < kLanes) {
#pragma unroll
            for (int j = 0; j < 8; ++j) exchange[wave][d + j] = y[j];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] += exchange[w][d + j];
    }
    if (lane >= kLanes) return;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    u32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = Elem<BF>::pack(y[2 * j] * inv, y[2 * j + 1] * inv);
    *reinterpret_cast<u32x4*>(out + d) = r;
    if (d == 0 && lse != nullptr) *lse = total == 0.f ? -__builtin_inff() : (less + __log2f(total)) * 0.6931471805599453f;
}
// Rows of a workgroup of the joining kernels.
constexpr int rows_of_join(int waves) { return waves > 1 ? 1 : 4; }

// A direct-to-LDS load from an address of each lane's own.
__device__ __forceinline__ void lds_load16(uint32_t lds_addr, const uint16_t* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_addr), "v"(from) : "memory", "m0");
}

// ... from addresses next to each other, by all lanes (lanes = ~0) or none (0).  Not said to change memory, so that reads of other rooms may pass it: those of
// its own room stand behind a barrier, which does say so.
__device__ __forceinline__ void masked_dma16(uint32_t lds_addr, const uint16_t* base, uint32_t voff, uint32_t lanes) {
    asm volatile("s_mov_b32 m0, %0\n\ts_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, -1" ::"s"(lds_addr), "v"(voff),
                 "s"(base), "s"(lanes) : "m0");
}

#include "latent_attend.inc"
#include "latent_expanded.inc"

}  // namespace latent
}  // namespace fa
