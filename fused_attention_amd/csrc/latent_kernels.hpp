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
// quarters lane l brings is (l % 4) ^ (l / 16): the 16 lanes that read one quarter of 16 tokens as an operand, and the 16 that read
// four tokens by 16 channels for a transpose, then touch all banks alike.
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

// Sixteen values to a thread: of a token's latent, of its rotary key, or of a query head.  Bound by the bytes.
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
template <bool BF>
constexpr float kLeash = BF ? 16.f : 7.f;
template <bool BF>
constexpr float kBias = BF ? 0.f : 8.f;

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Lane's bytes within a block: as loaded from rows `row_bytes` apart, as an operand of the first product, and as a transposed one of
// the second (channel tiles with an even and an odd number).
__device__ __forceinline__ uint32_t from_row(int lane, uint32_t row_bytes) {
    return (uint32_t)(lane >> 2) * row_bytes + (uint32_t)((lane & 3) ^ (lane >> 4)) * 16u;
}
__device__ __forceinline__ int key_at(int lane) {
    const int c = lane & 15, g = lane >> 4;
    return (4 * c + (g ^ (c >> 2))) * 16;
}
__device__ __forceinline__ int value_at(int lane, int odd) {
    const int s = lane & 15, g = lane >> 4;
    return ((4 * g + (s >> 2)) * 4 + ((2 * odd + ((s & 3) >> 1)) ^ g)) * 16 + (s & 1) * 8;
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

// Joins the parts that a row's keys were cut into: a wave a row, C / 8 lanes with eight channels each, the parts dealt out to the
// others and summed in a fixed order.  A part without any key has nothing but its log-sum-exp, -inf.
struct JoinParams {
    const float* part_o;       // [rows, splits, C]
    const float* part_lse;     // [rows, splits], log2 units
    uint16_t* out;
    Strides3 os;
    float* lse;                // [B, R, L] or nullptr
    int64_t rows;
    int L, R, splits;
    Divisor by_heads, by_tokens;
};
template <int C, bool BF>
__global__ __launch_bounds__(256) void latent_join_kernel(const JoinParams p) {
    constexpr int kLanes = C / 8, kAtOnce = 64 / kLanes;
    const int lane = threadIdx.x & 63, d = lane % kLanes * 8;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.rows) return;
    const float* parts = p.part_lse + row * p.splits;
    float top = -__builtin_inff();
    for (int s = lane; s < p.splits; s += 64) top = fmax2(top, parts[s]);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) top = fmax2(top, __shfl_xor(top, s));
    const float less = top == -__builtin_inff() ? 0.f : top;
    float total = 0.f;
    for (int s = lane; s < p.splits; s += 64) total += exp2_fast(parts[s] - less);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) total += __shfl_xor(total, s);
    float y[8] = {};
    for (int s = lane / kLanes; s < p.splits; s += kAtOnce) {
        const float part = parts[s];
        if (part == -__builtin_inff()) continue;
        const float w = exp2_fast(part - less);
        const floatx4* from = reinterpret_cast<const floatx4*>(p.part_o + (row * p.splits + s) * C + d);
        const floatx4 a = from[0], b = from[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] += w * a[j], y[4 + j] += w * b[j];
    }
#pragma unroll
    for (int s = kLanes; s < 64; s <<= 1)
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] += __shfl_xor(y[j], s);
    if (lane >= kLanes) return;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    u32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = Elem<BF>::pack(y[2 * j] * inv, y[2 * j + 1] * inv);
    const int token = p.by_heads.of((int)row), head = (int)row - token * p.R, b = p.by_tokens.of(token), i = token - b * p.L;
    *reinterpret_cast<u32x4*>(p.out + b * p.os.b + head * p.os.h + i * p.os.l + d) = r;
    if (d == 0 && p.lse != nullptr)
        p.lse[((int64_t)b * p.R + head) * p.L + i] = total == 0.f ? -__builtin_inff() : (less + __log2f(total)) * 0.6931471805599453f;
}

#include "latent_attend.inc"
#include "latent_expanded.inc"

}  // namespace latent
}  // namespace fa
