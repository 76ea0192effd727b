// Rotary positions for gfx950 (MI355X, CDNA4): tables of cosines and sines, scaled for long contexts, and the rotation of queries and
// keys by them in either pairing, of a part of each head, forwards and back.  No counterpart in the reference, whose queries and keys
// come as they are (reference src/fused_attn_extention.cu:15-22).
//
//   half          channels first + j and first + dims / 2 + j are a pair, j < dims / 2
//   interleaved   channels first + 2 j and first + 2 j + 1
//   (a, b) -> (a cos - b sin, b cos + a sin), with -sin for sin on the way back, which is the gradient's way
#pragma once

#include "rotation.hpp"

namespace fa {
namespace rotary {

using cache::Strides3;

constexpr int kMostDims = 256;

struct TablesParams {
    float* cos;                // [rows, half]
    float* sin;
    int64_t rows;
    int half;
    Divisor by_groups;         // division by half / 4
    double amplitude;
    double turns[kMostDims / 2];   // what a column turns by for each position, in whole turns
};

// Four columns of a row to a thread.  Angles are kept in turns: the whole ones fall away without an error, the quarters decide which of
// the two series is the cosine and with what sign, and both run over at most an eighth of a turn, y in [-pi / 4, pi / 4], where
// Taylor's series to y^11 and y^12 are within 7e-12.  All of it in 64 bits, one rounding at the end: at position 131071 the product of
// position and frequency in float32 would be off by a thousandth of a turn.  131072 rows of 2 x 64: 17 us, 67 MB at 3.9 TB/s, where a fill
// of that size reaches 6.0; 8192 rows of 2 x 32 4 us, a launch.
__global__ __launch_bounds__(256) void rotary_tables_kernel(const TablesParams p) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int groups = p.half / 4;
    if (at >= p.rows * groups) return;
    const int64_t row = at < 0x7fffffff ? p.by_groups.of((int)at) : at / groups;
    const int j0 = (int)(at - row * groups) * 4;
    floatx4 cos, sin;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double t = (double)row * p.turns[j0 + j], r = t - __builtin_rint(t), quarter = __builtin_rint(4.0 * r);
        const double y = (r - 0.25 * quarter) * 6.283185307179586476925, z = y * y;
        double s = -1.0 / 39916800.0, c = 1.0 / 479001600.0;
        s = __builtin_fma(s, z, 1.0 / 362880.0), c = __builtin_fma(c, z, -1.0 / 3628800.0);
        s = __builtin_fma(s, z, -1.0 / 5040.0), c = __builtin_fma(c, z, 1.0 / 40320.0);
        s = __builtin_fma(s, z, 1.0 / 120.0), c = __builtin_fma(c, z, -1.0 / 720.0);
        s = __builtin_fma(s, z, -1.0 / 6.0), c = __builtin_fma(c, z, 1.0 / 24.0);
        s = __builtin_fma(s * z, y, y), c = __builtin_fma(__builtin_fma(c, z, -0.5), z, 1.0);
        const int q = (int)quarter;                       // -2 .. 2
        const double cq = q & 1 ? s : c, sq = q & 1 ? c : s;
        // cos(y + q pi / 2): c, -s, -c, s; the sine: s, c, -s, -c
        cos[j] = (float)((q == 1 || q == 2 || q == -2 ? -cq : cq) * p.amplitude);
        sin[j] = (float)((q == -1 || q == 2 || q == -2 ? -sq : sq) * p.amplitude);
    }
    *reinterpret_cast<floatx4*>(p.cos + row * p.half + j0) = cos;
    *reinterpret_cast<floatx4*>(p.sin + row * p.half + j0) = sin;
}

struct Rotated {
    const uint16_t* x;
    uint16_t* out;
    Strides3 xs, os;
    int heads, chunks;         // chunks of heads that a thread takes, 0: nothing to rotate
};

struct RotateParams {
    Rotated of[2];             // queries and keys
    int B, L, H, first, dims;
    const float* cos;          // [rope_rows, dims / 2]
    const float* sin;
    int64_t rope_rows;
    const int32_t* positions;  // [B, L], or nullptr: starts[b] + i
    const int32_t* starts;     // [B], or nullptr: zeros
    const int32_t* new_lens;   // [B], or nullptr: L
    int inverse;
    int64_t total;             // threads with work
    Divisor by_units, by_chunks, by_tokens;      // division by H / 16, the chunks of both and L
};

// A thread takes 16 values, eight pairs or what is copied beside them, of HEADS heads of a token: the tables' row, 64 bytes, is
// read once for all of them.  Four heads where there is work for the whole chip then too, otherwise one.  Bound by the bytes: up to 8192
// tokens of 40 + 8 heads of 128, 185 MB, in 31 us, 6.0 TB/s (a copy of 64 MB 6.9, of 2 GB 5.0); a token of 4 + 4 heads 2 us.
template <bool BF, bool IL, int HEADS>
__global__ __launch_bounds__(256) void rotate_kernel(const RotateParams p) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= p.total) return;
    const int at = (int)id, row = p.by_units.of(at), unit = at - row * (p.H / 16);
    const int token = p.by_chunks.of(row), chunk = row - token * (p.of[0].chunks + p.of[1].chunks);
    const int b = p.by_tokens.of(token), i = token - b * p.L;
    const bool keys = chunk >= p.of[0].chunks;
    const Rotated& of = p.of[keys];
    const int head0 = (keys ? chunk - p.of[0].chunks : chunk) * HEADS, heads = of.heads - head0 < HEADS ? of.heads - head0 : HEADS;
    const int64_t pos = p.positions != nullptr ? p.positions[token] : (p.starts != nullptr ? (int64_t)p.starts[b] : 0) + i;
    int tokens = p.L;
    if (p.new_lens != nullptr) tokens = p.new_lens[b];
    const bool exists = i < tokens && pos >= 0 && pos < p.rope_rows, turned = unit < p.dims / 16;
    int c0, c1;                                          // the channels of the two halves of the unit
    if (turned) {
        c0 = p.first + (IL ? 16 : 8) * unit;
        c1 = c0 + (IL ? 8 : p.dims / 2);
    } else {
        c0 = 16 * unit - p.dims, c1 = c0 + 8;            // among what is copied
        c0 += c0 < p.first ? 0 : p.dims;
        c1 += c1 < p.first ? 0 : p.dims;
    }
    const uint16_t* x = of.x + b * of.xs.b + head0 * of.xs.h + i * of.xs.l;
    uint16_t* out = of.out + b * of.os.b + head0 * of.os.h + i * of.os.l;
    if (exists && !turned && x == out) return;           // in place: they are there
    u32x4 lo[HEADS] = {}, hi[HEADS] = {};
    if (exists) {
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
            if (h < heads) {
                lo[h] = *reinterpret_cast<const u32x4*>(x + h * of.xs.h + c0);
                hi[h] = *reinterpret_cast<const u32x4*>(x + h * of.xs.h + c1);
            }
        if (turned) {
            const int64_t entry = pos * (p.dims / 2) + 8 * unit;
            const Turn t = load_turn(p.cos + entry, p.sin + entry, p.inverse != 0);
#pragma unroll
            for (int h = 0; h < HEADS; ++h) turn_pairs<BF, IL>(lo[h], hi[h], t);
        }
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
        if (h < heads) {
            *reinterpret_cast<u32x4*>(out + h * of.os.h + c0) = lo[h];
            *reinterpret_cast<u32x4*>(out + h * of.os.h + c1) = hi[h];
        }
}

}  // namespace rotary
}  // namespace fa
