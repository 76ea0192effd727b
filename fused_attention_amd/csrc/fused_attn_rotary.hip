// C ABI of the rotary positions (include/fused_attn.h): argument validation and the launches.
#include "host_checks.hpp"
#include "rotary_kernels.hpp"

namespace {

using fa::rotary::RotateParams;
using fa::rotary::TablesParams;

// What every column turns by for each position, in turns.  False where the numbers make none.
bool turns_of(const fa_rotary* r, int64_t dims, double* turns) {
    const double two_pi = 6.283185307179586476925;
    double base = r->base;
    if (r->scaling == FA_ROTARY_BASE) base *= std::pow(r->factor, (double)dims / (double)(dims - 2));
    if (!std::isfinite(base)) return false;
    double low = 0, high = 0;
    if (r->scaling == FA_ROTARY_INDEX) {
        auto index = [&](double t) { return (double)dims * std::log(r->original_rows / (two_pi * t)) / (2 * std::log(base)); };
        low = std::floor(index(r->high)), high = std::ceil(index(r->low));
        low = low > 0 ? low : 0, high = high < (double)(dims - 1) ? high : (double)(dims - 1);
    }
    for (int64_t j = 0; j < dims / 2; ++j) {
        const double f = std::pow(base, -2.0 * (double)j / (double)dims);
        double kept = 1;                                 // the share of the frequency that stays as it is
        if (r->scaling == FA_ROTARY_LINEAR) kept = 0;
        if (r->scaling == FA_ROTARY_TURNS) kept = (r->original_rows * f / two_pi - r->low) / (r->high - r->low);
        if (r->scaling == FA_ROTARY_INDEX) kept = 1 - ((double)j - low) / (high - low > 0.001 ? high - low : 0.001);
        kept = kept < 0 ? 0 : kept > 1 ? 1 : kept;
        turns[j] = f * (kept + (1 - kept) / (r->scaling == FA_ROTARY_BASE ? 1 : r->factor)) / two_pi;
        if (!std::isfinite(turns[j])) return false;
    }
    return true;
}

bool is_positive(double x) { return x > 0 && std::isfinite(x); }

// Rows of H values by their first address, strides and numbers.
struct Rows {
    const void* at;
    Strides3 s;
    int64_t B, heads, L;
    bool same_places(const Rows& o) const {
        return at == o.at && (B == 1 || s.b == o.s.b) && (heads == 1 || s.h == o.s.h) && (L == 1 || s.l == o.s.l);
    }
    uintptr_t begin() const { return reinterpret_cast<uintptr_t>(at); }
    uintptr_t end(int64_t H) const { return begin() + 2 * (uintptr_t)((B - 1) * s.b + (heads - 1) * s.h + (L - 1) * s.l + H); }
};
struct Steps {
    int64_t stride, least, most;
};

// Whether `d` is less than a row from a sum of so many of each stride.  A stride steps over all that those behind it reach, so that no more than two
// numbers of steps come into question.
bool reaches(int64_t d, const Steps* s, int n, int64_t H) {
    if (n == 0) return -H < d && d < H;
    const int64_t down = d / s->stride - (d % s->stride < 0 ? 1 : 0);
    for (int64_t i : {down, down + 1}) {
        i = std::min(std::max(i, s->least), s->most);
        if (reaches(d - i * s->stride, s + 1, n - 1, H)) return true;
    }
    return false;
}

// Whether a row of `a` and one of `b` share a place.  Exact where both have the same strides, as views of one tensor have; otherwise it is looked whether the
// first row of either is among the other's.
bool meet(const Rows& a, const Rows& b, int64_t H) {
    if (a.end(H) <= b.begin() || b.end(H) <= a.begin()) return false;        // new outputs
    const int64_t strides[2][3] = {{a.s.b, a.s.h, a.s.l}, {b.s.b, b.s.h, b.s.l}}, counts[2][3] = {{a.B, a.heads, a.L}, {b.B, b.heads, b.L}};
    const int64_t d = ((int64_t)reinterpret_cast<uintptr_t>(b.at) - (int64_t)reinterpret_cast<uintptr_t>(a.at)) / 2;
    bool alike = true;
    for (int i = 0; i < 3; ++i) alike = alike && (counts[0][i] == 1 || counts[1][i] == 1 || strides[0][i] == strides[1][i]);
    auto within = [&](bool of_a, bool of_b) {
        Steps steps[3];
        int n = 0;
        for (int i = 0; i < 3; ++i) {
            const int64_t na = of_a ? counts[0][i] : 1, nb = of_b ? counts[1][i] : 1, stride = strides[na > 1 ? 0 : 1][i];
            if ((na > 1 || nb > 1) && stride > 0) steps[n++] = {stride, 1 - nb, na - 1};
        }
        std::sort(steps, steps + n, [](const Steps& x, const Steps& y) { return x.stride > y.stride; });
        return reaches(d, steps, n, H);
    };
    return alike ? within(true, true) : within(true, false) || within(false, true);
}

}  // namespace

extern "C" {

int fa_rotary_tables(float* cos, float* sin, int64_t rows, int64_t dims, const fa_rotary* how, void* stream) {
    if (cos == nullptr || sin == nullptr || how == nullptr) return FA_ERR_NULL_POINTER;
    if (rows < 1 || dims < 16 || dims % 16 != 0) return FA_ERR_BAD_SHAPE;
    if (dims > fa::rotary::kMostDims || rows > kMaxInt) return FA_ERR_TOO_LARGE;
    if (!aligned(cos, 16) || !aligned(sin, 16)) return FA_ERR_MISALIGNED;
    const int s = how->scaling;
    if (s < FA_ROTARY_NONE || s > FA_ROTARY_INDEX) return FA_ERR_BAD_FLAGS;
    if (!(how->base > 1) || !std::isfinite(how->base) || !is_positive(how->amplitude)) return FA_ERR_BAD_SCALE;
    if (s != FA_ROTARY_NONE && !is_positive(how->factor)) return FA_ERR_BAD_SCALE;
    if ((s == FA_ROTARY_TURNS || s == FA_ROTARY_INDEX) &&
        (!is_positive(how->original_rows) || !is_positive(how->low) || !is_positive(how->high) || !(how->low < how->high)))
        return FA_ERR_BAD_SCALE;
    TablesParams p;
    fa_rotary r = *how;
    if (s == FA_ROTARY_NONE) r.factor = 1;
    if (!turns_of(&r, dims, p.turns)) return FA_ERR_BAD_SCALE;
    p.cos = cos;
    p.sin = sin;
    p.rows = rows;
    p.half = (int)(dims / 2);
    p.by_groups = fa::divisor(p.half / 4);
    p.amplitude = how->amplitude;
    const int64_t wgs = ceil_div(rows * (p.half / 4), 256);
    if (wgs > kMostThreads / 256) return FA_ERR_TOO_LARGE;
    return static_cast<int>(launch(fa::rotary::rotary_tables_kernel, wgs, 256, p, 0, static_cast<hipStream_t>(stream)));
}

int fa_rotate(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, void* q_out, int64_t q_out_stride_b,
              int64_t q_out_stride_h, int64_t q_out_stride_l, const void* k, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_l,
              void* k_out, int64_t k_out_stride_b, int64_t k_out_stride_h, int64_t k_out_stride_l, int64_t B, int64_t L, int64_t R,
              int64_t Rkv, int64_t H, int64_t first, int64_t dims, const float* cos, const float* sin, int64_t rope_rows,
              const int32_t* positions, const int32_t* starts, const int32_t* new_lens, int flags, void* stream) {
    if ((flags & ~(FA_FLAG_BF16 | FA_FLAG_INTERLEAVED | FA_FLAG_INVERSE)) != 0) return FA_ERR_BAD_FLAGS;
    if (H < 16 || H > 1024 || H % 16 != 0) return FA_ERR_BAD_HEAD_DIM;
    if ((k == nullptr) != (k_out == nullptr)) return FA_ERR_NULL_POINTER;
    if (k == nullptr) Rkv = 0;
    if (B < 1 || L < 1 || R < 1 || (k != nullptr && Rkv < 1) || rope_rows < 1) return FA_ERR_BAD_SHAPE;
    if (dims < 16 || dims % 16 != 0 || first < 0 || first % 8 != 0 || first > H || dims > H - first) return FA_ERR_BAD_SHAPE;
    if (cos == nullptr || sin == nullptr) return FA_ERR_NULL_POINTER;
    if (positions != nullptr && starts != nullptr) return FA_ERR_BAD_SHAPE;
    if (!aligned(cos, 16) || !aligned(sin, 16) || !aligned(positions, 4) || !aligned(starts, 4) || !aligned(new_lens, 4)) return FA_ERR_MISALIGNED;
    if (B > kMaxInt || L > kMaxInt || R > kMaxInt || Rkv > kMaxInt || !below(B, L, kMaxInt) || !below(B * L, R + Rkv, kMaxInt) ||
        !below(B * L * (R + Rkv), H / 16, kMaxInt))
        return FA_ERR_TOO_LARGE;
    RotateParams p;
    p.of[0] = {static_cast<const uint16_t*>(q), static_cast<uint16_t*>(q_out), {q_stride_b, q_stride_h, q_stride_l},
               {q_out_stride_b, q_out_stride_h, q_out_stride_l}, (int)R, 0};
    p.of[1] = {static_cast<const uint16_t*>(k), static_cast<uint16_t*>(k_out), {k_stride_b, k_stride_h, k_stride_l},
               {k_out_stride_b, k_out_stride_h, k_out_stride_l}, (int)Rkv, 0};
    // A head a thread where that is what it takes to fill the chip: a single token waits for nothing but its chain of loads.
    const int64_t units = B * L * (R + Rkv) * (H / 16);
    const int heads = units >= (int64_t)4 * 2048 * kNumCu ? 4 : 1;
    for (int n = 0; n < (k != nullptr ? 2 : 1); ++n) {
        fa::rotary::Rotated& t = p.of[n];
        int rc = check_strided(t.x, t.xs, B, t.heads, L, H);
        if (rc == FA_OK) rc = check_written(t.out, t.os, B, t.heads, L, H);
        if (rc != FA_OK) return rc;
        t.chunks = (int)ceil_div(t.heads, heads);
    }
    auto rows = [&](const void* t, const Strides3& strides, int64_t heads) { return Rows{t, strides, B, heads, L}; };
    const Rows in[2] = {rows(q, p.of[0].xs, R), rows(k, p.of[1].xs, Rkv)}, written[2] = {rows(q_out, p.of[0].os, R), rows(k_out, p.of[1].os, Rkv)};
    for (int n = 0; n < (k != nullptr ? 2 : 1); ++n)
        if (!in[n].same_places(written[n]) && meet(in[n], written[n], H)) return FA_ERR_BAD_STRIDE;
    if (k != nullptr && (meet(written[0], written[1], H) || meet(written[0], in[1], H) || meet(written[1], in[0], H))) return FA_ERR_BAD_STRIDE;
    p.B = (int)B;
    p.L = (int)L;
    p.H = (int)H;
    p.first = (int)first;
    p.dims = (int)dims;
    p.cos = cos;
    p.sin = sin;
    p.rope_rows = rope_rows;
    p.positions = positions;
    p.starts = starts;
    p.new_lens = new_lens;
    p.inverse = (flags & FA_FLAG_INVERSE) != 0;
    const int64_t chunks = p.of[0].chunks + p.of[1].chunks;
    p.total = B * L * chunks * (H / 16);
    p.by_units = fa::divisor(H / 16);
    p.by_chunks = fa::divisor(chunks);
    p.by_tokens = fa::divisor(L);
    const bool bf = (flags & FA_FLAG_BF16) != 0, il = (flags & FA_FLAG_INTERLEAVED) != 0;
    using namespace fa::rotary;
    auto kernel = heads == 4 ? (bf ? (il ? rotate_kernel<true, true, 4> : rotate_kernel<true, false, 4>)
                                   : (il ? rotate_kernel<false, true, 4> : rotate_kernel<false, false, 4>))
                             : (bf ? (il ? rotate_kernel<true, true, 1> : rotate_kernel<true, false, 1>)
                                   : (il ? rotate_kernel<false, true, 1> : rotate_kernel<false, false, 1>));
    return static_cast<int>(launch(kernel, ceil_div(p.total, 256), 256, p, 0, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
