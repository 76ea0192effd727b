// C ABI of the paged key/value cache (include/fused_attn.h): argument validation, the choice of launch and the launches.
// A translation unit of its own, so that the attention and projection kernels are compiled as they were.
#include "cache_kernels.hpp"

#include "../../include/fused_attn.h"

#include <algorithm>
#include <array>
#include <cmath>
#include <mutex>
#include <utility>
#include <vector>

namespace {

using fa::cache::AppendParams;
using fa::cache::AttendParams;
using fa::cache::SelectParams;
using fa::cache::Strides3;
using fa::cache::View;

constexpr int kNumCu = 256;
constexpr int64_t kMaxInt = 0x7fffffff - 0x10000;
constexpr int64_t kMaxElems = (int64_t)1 << 62;
constexpr int64_t kMostThreads = 0xffffffffll;       // of a grid: the dispatch packet holds no more

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool below(int64_t a, int64_t b, int64_t most) { return a <= most / b; }     // a * b <= most, for positive b

// The sizes of the cache and the call, without any pointer.
int check_sizes(const fa_cache* c, int64_t L, int64_t R, View* p) {
    if (c == nullptr) return FA_ERR_NULL_POINTER;
    if (!fa_fwd_query(c->head_dim)) return FA_ERR_BAD_HEAD_DIM;
    int log2_p = 4;
    while (log2_p < 7 && ((int64_t)1 << log2_p) < c->page_size) ++log2_p;
    if (c->page_size != (int64_t)1 << log2_p) return FA_ERR_BAD_PAGE;
    if (c->pages < 1 || c->heads < 1 || c->sequences < 1 || c->table_width < 1 || L < 1 || R < 1 || R % c->heads != 0) return FA_ERR_BAD_SHAPE;
    if (c->table_stride < c->table_width && c->sequences > 1) return FA_ERR_BAD_STRIDE;
    if (c->table_stride < 0) return FA_ERR_BAD_STRIDE;
    if (c->pages > kMaxInt || c->heads > kMaxInt || R > kMaxInt || L > kMaxInt || c->sequences > kMaxInt || c->table_width > kMaxInt)
        return FA_ERR_TOO_LARGE;
    if (!below(c->pages * c->heads, c->page_size / 16, kMaxInt) || !below(c->table_width, c->page_size, kMaxInt) ||
        !below(L, R, kMaxInt) || !below(L * R, c->sequences, kMaxInt) || !below(c->table_stride, c->sequences, kMaxElems))
        return FA_ERR_TOO_LARGE;
    p->k = static_cast<uint8_t*>(c->keys);
    p->v = static_cast<uint8_t*>(c->values);
    p->k_exponents = static_cast<int8_t*>(c->key_exponents);
    p->v_exponents = static_cast<int8_t*>(c->value_exponents);
    p->bounds = static_cast<int8_t*>(c->key_bounds);
    p->table = c->page_table;
    p->table_stride = c->table_stride;
    p->B = (int)c->sequences;
    p->L = (int)L;
    p->R = (int)R;
    p->Rkv = (int)c->heads;
    p->W = (int)c->table_width;
    p->pages = (int)c->pages;
    p->log2_p = log2_p;
    p->group = (int)(R / c->heads);
    return FA_OK;
}

int check_tensors(const fa_cache* c, const int32_t* starts, const int32_t* new_lens, bool values, View* p) {
    if (starts == nullptr || c->page_table == nullptr || c->key_exponents == nullptr) return FA_ERR_NULL_POINTER;
    if (values && (c->keys == nullptr || c->values == nullptr || c->value_exponents == nullptr)) return FA_ERR_NULL_POINTER;
    if (!aligned(starts, 4) || !aligned(new_lens, 4) || !aligned(c->page_table, 4)) return FA_ERR_MISALIGNED;
    if (!aligned(c->key_bounds, 16) || (values && (!aligned(c->keys, 16) || !aligned(c->values, 16)))) return FA_ERR_MISALIGNED;
    p->starts = starts;
    p->new_lens = new_lens;
    return FA_OK;
}

// A tensor under the addressing rule: its strides, alignment and extent.
int check_strided(const void* t, const Strides3& s, int64_t B, int64_t heads, int64_t L, int64_t H) {
    if (t == nullptr) return FA_ERR_NULL_POINTER;
    if (s.b < 0 || s.h < 0 || s.l < H || s.b % 8 != 0 || s.h % 8 != 0 || s.l % 8 != 0) return FA_ERR_BAD_STRIDE;
    if (!aligned(t, 16)) return FA_ERR_MISALIGNED;
    if (!below(L, s.l, kMaxElems) || (s.h > 0 && !below(heads, s.h, kMaxElems)) || (s.b > 0 && !below(B, s.b, kMaxElems))) return FA_ERR_TOO_LARGE;
    return FA_OK;
}

// What is written: the same, with a place of its own for every row.  Of the dimensions with more than one element, by their strides,
// each has to step over all the rows that those before it place.
int check_written(const void* t, const Strides3& s, int64_t B, int64_t heads, int64_t L, int64_t H) {
    const int rc = check_strided(t, s, B, heads, L, H);
    if (rc != FA_OK) return rc;
    std::array<std::pair<int64_t, int64_t>, 3> dims = {{{s.b, B}, {s.h, heads}, {s.l, L}}};
    std::sort(dims.begin(), dims.end());
    uint64_t taken = (uint64_t)H;                        // three products below kMaxElems fit
    for (const auto& [stride, n] : dims) {
        if (n == 1) continue;
        if ((uint64_t)stride < taken) return FA_ERR_BAD_STRIDE;
        taken += (uint64_t)stride * (uint64_t)(n - 1);
    }
    return FA_OK;
}

// Dynamic LDS above 64 KiB has to be opted into per kernel function and per device.
hipError_t allow_large_lds(const void* kernel, int bytes) {
    static std::mutex lock;
    static std::vector<std::pair<const void*, int>> done;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    try {
        std::lock_guard<std::mutex> guard(lock);
        for (const auto& d : done)
            if (d.first == kernel && d.second == dev) return hipSuccess;
        e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == hipSuccess) done.emplace_back(kernel, dev);
        return e;
    } catch (...) {          // nothing is thrown through a C entry; not remembered, it is asked for again the next time
        return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    }
}

template <class Params>
hipError_t launch(void (*kernel)(const Params), int64_t wgs, int threads, const Params& p, int lds, hipStream_t stream) {
    Params params = p;
    void* args[] = {&params};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3((uint32_t)wgs), dim3(threads), args, lds, stream);
}

// f(std::integral_constant<int, H>, std::bool_constant<BF>) for a run-time head_dim and type
template <class F>
hipError_t for_type(int64_t H, bool bf, F f) {
    auto with = [&](auto h) { return bf ? f(h, std::true_type{}) : f(h, std::false_type{}); };
    switch (H) {
        case 16: return with(std::integral_constant<int, 16>{});
        case 32: return with(std::integral_constant<int, 32>{});
        case 64: return with(std::integral_constant<int, 64>{});
        default: return with(std::integral_constant<int, 128>{});
    }
}

// How cached_attention is launched.
struct AttendPlan {
    bool wide;             // the kernel for many rows
    bool shared;           // the lists of several tokens joined
    int nq, waves;         // the other one: blocks of 16 query rows and waves of a workgroup
    int64_t tiles, splits, wgs;
};

constexpr int64_t kMostSplits = 64;    // the join gives each a lane

// In how many parts a launch cuts its keys and what it takes, in microseconds as measured, for a causal call (what the caller asks for
// is not known where the workspace is sized, and the longest rows take the same).  The lengths are in device memory: every
// estimate takes the page table to be as wide as the longest sequence, and is off where it is wider.
struct Estimate {
    int64_t splits;
    float us;
};

// The second kernel, beside its launch: every split's sums written and read.
float join_us(const View& p, int64_t splits, int64_t H) {
    return splits > 1 ? 3.f + (float)p.B * (float)p.L * (float)p.R * (float)splits * (float)H * 8.f / 2.5e6f : 0.f;
}

// In how many parts the keys of `base` row tiles are cut, few rows.  On 14 shapes (up to 64 sequences, 256 to 131072 tokens)
// against every other count of parts, the best one is chosen or one within 5 % of it: a wave takes 1 + H / 110 for a step of
// 64 tokens, or what the bytes of all heads take at 4.8 TB/s where that is more, or the products of a compute unit's
// workgroups, those beyond one per compute unit in whole rounds; and the second kernel 3.  (B16 Rkv12 H64, 1000 tokens: 9.9 us
// in one part, 12.8 in two; Rkv8 H128, 2000 tokens: 18.5 in one part, 12.4 in four, 11.4 in eight; 131072 tokens: 75.7 in 16,
// 58.5 in 32, 66.1 in 48, 60.7 in 64.)
Estimate narrow_splits(const View& p, int64_t base, int64_t steps, int64_t H) {
    const float alone = 1.f + 0.009f * (float)H;
    const float bytes = 0.0273f * (float)H;              // a step of a workgroup's waves, by a 256th of the memory
    const float products = H > 64 ? 1.4f : 0.8f;
    const int64_t heads = (int64_t)p.B * p.Rkv;
    Estimate best{1, 3.0e38f};
    for (int64_t s = 1; s <= kMostSplits && (s == 1 || (base * s <= 4 * kNumCu && (s - 1) * fa::cache::kAttendWaves < steps)); ++s) {
        auto rounds = [](int64_t wgs) { return wgs <= kNumCu ? (float)wgs / kNumCu : (float)ceil_div(wgs, kNumCu); };
        float step = bytes * rounds(heads * s);
        if (step < products * rounds(base * s)) step = products * rounds(base * s);
        if (step < alone) step = alone;
        const float us = step * (float)ceil_div(steps, s * fa::cache::kAttendWaves) + join_us(p, s, H);
        if (us < best.us) best = {s, us};
    }
    return best;
}

// Many rows, the narrow kernel in one part: rounds of the workgroups that a chip holds, and what the products and exponentials
// take in all; or the longest workgroup; or the codes, which every row tile reads, where they are more than the second-level caches
// hold.  (Causal, estimated and measured: 8 sequences of 1000 tokens of 12 heads of 64: 46, 51 us; 2000 rows of each of 8
// heads of 128 over 8000 tokens: 94, 99; 4096 tokens of 32 heads of 128: 251, 247; by the codes, 8 tokens of 64 sequences of 1000, 40
// heads on 8 of 128: 58, 55.)
float narrow_us(const View& p, int64_t base, float keys, int64_t steps, int64_t H) {
    const int64_t resident = H > 64 ? 2 * kNumCu : 3 * kNumCu;
    const float rate = H > 64 ? 1.5e6f : H > 32 ? 2.4e6f : 3.e6f;       // rows times keys; the rows of whole tiles
    const float whole = (H > 64 ? 9.f : 6.5f) * (float)ceil_div(base, resident) + (float)base * 32.f * keys / rate;
    const float longest = 6.f + (1.f + 0.009f * (float)H) * (float)ceil_div(steps, fa::cache::kAttendWaves);
    const float us = whole > longest ? whole : longest;
    const float heads = (float)p.B * (float)p.Rkv, bytes = heads * keys * 2.f * (float)H;
    const float read = 6.f + (float)base / heads * bytes / 5.e6f;
    return bytes > 3.2e7f && read > us ? read : us;
}

// The wide kernel: the longest workgroup's tiles of 64 keys, or what the chip's workgroups take in all, of which a compute
// unit holds one at head_dim 128 and two below; with one block of 16 rows a wave instead of two, two and three.  Then a tile
// takes 0.6 of the time and there are twice as many workgroups: for calls that the longest workgroup bounds.  (The same three,
// measured with two blocks and with one: 38, 33 us; 90, 91, each in four parts; 178, 199.  32 heads on 8 of 128: 1500 tokens 57,
// 43, by the other kernel 59; 2048 behind 14336 515, 528.  8 tokens of 64 sequences of 1000, 40 heads on 8 of 128: 66, 33, by the
// other 55.)
Estimate wide_us(const View& p, int64_t nq, int64_t most_keys, float keys, int64_t H) {
    Estimate best{1, 3.0e38f};
    const int64_t base = (int64_t)p.B * p.Rkv * ceil_div((int64_t)p.L * p.group, fa::cache::kWideWaves * 16 * nq);
    for (int64_t s = 1; s <= kMostSplits && (s == 1 || (base * s <= 4 * kNumCu && s * fa::cache::kWideKeys < most_keys)); ++s) {
        const float per_cu = (float)(base * s) / kNumCu;
        const float two = H > 64 ? 2.02f : (per_cu > 1.f ? 2.3f : 1.6f) - (H > 32 ? 0.f : 0.3f);
        const float one = H > 64   ? 1.36f + (per_cu > 1.f ? 0.4f * ((per_cu < 2.f ? per_cu : 2.f) - 1.f) : 0.f)
                          : H > 32 ? (per_cu > 1.f ? 1.65f : 1.17f)
                                   : (per_cu > 1.f ? 1.2f : 0.95f);
        const float tile = nq == 2 ? two : one;
        const float all = nq == 1 ? (H > 64 ? 1.12f : 0.75f) * per_cu : H > 64 ? tile * (float)ceil_div(base * s, kNumCu) : 1.3f * per_cu;
        const float longest = tile * (float)ceil_div(most_keys, s * fa::cache::kWideKeys), whole = all * keys / (float)(s * fa::cache::kWideKeys);
        const float us = 6.f + (longest > whole ? longest : whole) + join_us(p, s, H);
        if (us < best.us) best = {s, us};
    }
    return best;
}

// How often a page that one of `tokens` lists names is in them all, were they drawn by chance from the whole table: lists of
// neighbours have more in common, so that joining them gains more than this says.  (4 query heads to each of 8 key heads of 128,
// 500 tokens, 48 of 250 pages each: 1.34 by chance, 90 us instead of 110; lists that are half alike 59, equal ones 34.  2000 tokens,
// 32 pages: 1.21 by chance, 454 instead of 439, half alike 299.  With 256 tiles of four waves: 1.9 by chance, 37 instead
// of 38, half alike 25.  With 192 tiles 27 instead of 20, with 544 and 1.14 by chance 52 instead of 43.)
double overlap(const View& p, int64_t tokens, int64_t count) {
    const double listed = count < p.W ? (double)count / p.W : 1.0;
    return tokens * listed / (1.0 - std::pow(1.0 - listed, (double)tokens));
}

AttendPlan plan_attend(const View& p, int64_t count, int64_t H) {
    AttendPlan a;
    const int64_t rows = (int64_t)p.L * p.group, heads = (int64_t)p.B * p.Rkv;
    const int64_t most_keys = (count > 0 ? count : (int64_t)p.W) << p.log2_p, steps = ceil_div(most_keys, 64);
    a.wide = false;
    a.shared = false;
    a.nq = count > 0 || rows <= 16 ? 1 : 2;
    a.tiles = count > 0 ? p.L * ceil_div(p.group, 16) : ceil_div(rows, 16 * a.nq);
    a.waves = fa::cache::kAttendWaves;
    a.splits = 1;
    if (count > 0 && p.group <= 8 && p.W <= fa::cache::kMostShared) {
        const int64_t together = fa::cache::shared_tokens(p.group) < p.L ? fa::cache::shared_tokens(p.group) : p.L, tiles = ceil_div(p.L, together);
        const bool many = heads * tiles >= 3 * kNumCu;   // that fill the chip with two waves each
        if (heads * tiles >= kNumCu && overlap(p, together, count) >= (many ? 1.1 : 1.5)) {
            a.shared = true;
            a.tiles = tiles;
            a.waves = many ? 2 : fa::cache::kAttendWaves;
            a.wgs = heads * a.tiles;
            return a;
        }
    }
    const Estimate parts = narrow_splits(p, heads * a.tiles, steps, H);
    if (count > 0 && heads * a.tiles > 4 * kNumCu)
        a.waves = 1;                                     // a wave a tile, nothing to merge: 143 us where four take 152
    else
        a.splits = parts.splits;
    // (16 tokens of 8 key heads, 32 pages of 64: 19 us, in two parts of four waves 17 and 4 to join them)
    if (count > 0 && heads * a.tiles <= kNumCu && a.splits <= 2) a.waves = 8, a.splits = 1;
    if (count == 0 && rows > 32) {
        const float keys = most_keys > p.L ? (float)most_keys - 0.5f * (float)p.L : 0.5f * (float)most_keys;
        const Estimate two = wide_us(p, 2, most_keys, keys, H), one = wide_us(p, 1, most_keys, keys, H), wide = one.us < two.us ? one : two;
        const int nq = one.us < two.us ? 1 : 2;
        const float narrow = a.splits > 1 ? parts.us + 6.f : narrow_us(p, heads * a.tiles, keys, steps, H);
        if (wide.us < narrow) {
            a.nq = nq;
            a.wide = true;
            a.waves = fa::cache::kWideWaves;
            a.tiles = ceil_div(rows, fa::cache::kWideWaves * 16 * nq);
            a.splits = wide.splits;
        }
    }
    a.wgs = heads * a.tiles * a.splits;
    return a;
}

int64_t attend_workspace(const View& p, const AttendPlan& a, int64_t H) {
    return a.splits > 1 ? (int64_t)p.B * p.L * p.R * a.splits * (H + 1) * 4 : 0;
}

int check_count(int64_t count) { return count > fa::cache::kMostSelected ? FA_ERR_TOO_LARGE : FA_OK; }

constexpr int kMostTable = 32768;        // pages of a table, for a selection: their scores are held in LDS
constexpr int kMostRowKeys = 8192;       // ... of several tokens: 32 KiB, four workgroups to a compute unit

// How select_pages is launched: tokens and waves of a workgroup.
struct SelectPlan {
    int64_t tokens;
    int waves;
    int64_t wgs;
};

// Several tokens to a workgroup where they share a tile of the product (see the kernel) and there are enough of them to fill the
// chip all the same (500 tokens of 8 key heads, 250 pages: 18.6 us against 46); otherwise one, with sixteen waves, four where
// there are more than the chip holds (16 tokens of 8 key heads, 512 pages: 11.9 us against 20 with four).
SelectPlan plan_select(const View& p) {
    SelectPlan a;
    const int64_t heads = (int64_t)p.B * p.Rkv;
    a.tokens = p.group == 1 || p.group == 2 || p.group == 4 || p.group == 8 ? 16 / p.group : 1;
    if (a.tokens * p.W > kMostRowKeys || heads * ceil_div(p.L, a.tokens) < kNumCu) a.tokens = 1;
    a.wgs = heads * ceil_div(p.L, a.tokens);
    a.waves = a.tokens > 1 || a.wgs > 4 * kNumCu ? 4 : 16;
    return a;
}

}  // namespace

extern "C" {

int fa_cache_append(const fa_cache* cache, const void* k, const void* v, int64_t kv_stride_b, int64_t kv_stride_h, int64_t kv_stride_l,
                    const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, void* q_out, int64_t out_stride_b,
                    int64_t out_stride_h, int64_t out_stride_l, const int32_t* starts, const int32_t* new_lens, int64_t L, int64_t R,
                    const float* rope_cos, const float* rope_sin, int64_t rope_rows, int flags, void* stream) {
    if ((flags & ~FA_FLAG_BF16) != 0) return FA_ERR_BAD_FLAGS;
    AppendParams p;
    int rc = check_sizes(cache, L, q != nullptr || cache == nullptr ? R : cache->heads, &p);
    if (rc == FA_OK) rc = check_tensors(cache, starts, new_lens, true, &p);
    if (rc != FA_OK) return rc;
    const int64_t B = cache->sequences, H = cache->head_dim;
    p.kv = {kv_stride_b, kv_stride_h, kv_stride_l};
    p.qs = {q_stride_b, q_stride_h, q_stride_l};
    p.qo = {out_stride_b, out_stride_h, out_stride_l};
    for (const void* t : {k, v})
        if ((rc = check_strided(t, p.kv, B, cache->heads, L, H)) != FA_OK) return rc;
    if ((q == nullptr) != (q_out == nullptr)) return FA_ERR_NULL_POINTER;
    if (q != nullptr && (rc = check_strided(q, p.qs, B, R, L, H)) != FA_OK) return rc;
    if (q != nullptr && (rc = check_written(q_out, p.qo, B, R, L, H)) != FA_OK) return rc;
    if ((rope_cos == nullptr) != (rope_sin == nullptr)) return FA_ERR_NULL_POINTER;
    if (rope_cos != nullptr && rope_rows < 1) return FA_ERR_BAD_SHAPE;
    if (!aligned(rope_cos, 16) || !aligned(rope_sin, 16)) return FA_ERR_MISALIGNED;
    p.key = static_cast<const uint16_t*>(k);
    p.value = static_cast<const uint16_t*>(v);
    p.q = static_cast<const uint16_t*>(q);
    p.q_out = static_cast<uint16_t*>(q_out);
    p.rope_cos = rope_cos;
    p.rope_sin = rope_sin;
    p.rope_rows = rope_rows;
    const int64_t P = cache->page_size;
    // the page of the first token, and those of the others
    const int64_t reach = (L + P - 2) / P + 1;
    p.reach = (int)(reach < p.W ? reach : p.W);
    p.cache_items = B * p.reach * cache->heads * 2;
    p.q_units = q != nullptr ? B * L * R * (H / 16) : 0;
    p.by_query_heads = fa::divisor(p.R);
    p.by_tokens = fa::divisor(L);
    p.by_heads = fa::divisor(p.Rkv);
    p.by_reach = fa::divisor(p.reach);
    const bool bf = (flags & FA_FLAG_BF16) != 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t units = (L < P ? L : P) * (H / 16);    // of a page's new tokens
    const int threads = units <= 64 ? 64 : 256;
    const int64_t wgs = p.cache_items + ceil_div(p.q_units, threads);
    if (wgs > kMostThreads / threads || p.cache_items > 0x7fffffff) return FA_ERR_TOO_LARGE;
    return static_cast<int>(for_type(H, bf, [&](auto h, auto b) {
        using namespace fa::cache;
        if (units <= 64) return launch(cache_append_kernel<h(), b(), 64, 1>, wgs, 64, p, 0, s);
        if constexpr (h() >= 128)
            if (units > 512) return launch(cache_append_kernel<h(), b(), 256, 4>, wgs, 256, p, 0, s);
        if constexpr (h() >= 64)
            if (units > 256) return launch(cache_append_kernel<h(), b(), 256, 2>, wgs, 256, p, 0, s);
        return launch(cache_append_kernel<h(), b(), 256, 1>, wgs, 256, p, 0, s);
    }));
}

int64_t fa_cached_attention_workspace(const fa_cache* cache, int64_t L, int64_t R, int64_t count) {
    View p;
    int rc = check_sizes(cache, L, R, &p);
    if (rc == FA_OK) rc = check_count(count);
    if (rc == FA_OK && count < 0) rc = FA_ERR_BAD_SHAPE;
    if (rc != FA_OK) return rc;
    return attend_workspace(p, plan_attend(p, count, cache->head_dim), cache->head_dim);
}

int fa_cached_attention(const fa_cache* cache, const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, void* out,
                        int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_l, void* lse, const int32_t* selected,
                        int64_t count, const int32_t* starts, const int32_t* new_lens, int64_t L, int64_t R, float scale, int flags,
                        void* workspace, int64_t workspace_bytes, void* stream) {
    if ((flags & ~(FA_FLAG_BF16 | FA_FLAG_CAUSAL)) != 0) return FA_ERR_BAD_FLAGS;
    AttendParams p;
    int rc = check_sizes(cache, L, R, &p);
    if (rc == FA_OK) rc = check_tensors(cache, starts, new_lens, true, &p);
    if (rc != FA_OK) return rc;
    if (selected != nullptr && count < 1) return FA_ERR_BAD_SHAPE;
    if (selected == nullptr) count = 0;
    if ((rc = check_count(count)) != FA_OK) return rc;
    p.scale_log2e = scale * 1.4426950408889634f;
    if (!(scale > 0.f) || !std::isfinite(p.scale_log2e)) return FA_ERR_BAD_SCALE;
    const int64_t B = cache->sequences, H = cache->head_dim;
    p.qs = {q_stride_b, q_stride_h, q_stride_l};
    p.os = {out_stride_b, out_stride_h, out_stride_l};
    if ((rc = check_strided(q, p.qs, B, R, L, H)) != FA_OK) return rc;
    if ((rc = check_written(out, p.os, B, R, L, H)) != FA_OK) return rc;
    if (!aligned(lse, 4) || !aligned(selected, 4)) return FA_ERR_MISALIGNED;
    const AttendPlan a = plan_attend(p, count, H);
    if (a.wgs > kMaxInt || a.wgs > kMostThreads / (64 * fa::cache::kWideWaves)) return FA_ERR_TOO_LARGE;
    const int64_t need = attend_workspace(p, a, H);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return FA_ERR_WORKSPACE;
    if (need > 0 && !aligned(workspace, 16)) return FA_ERR_MISALIGNED;
    p.q = static_cast<const uint16_t*>(q);
    p.out = static_cast<uint16_t*>(out);
    p.lse = static_cast<float*>(lse);
    p.selected = selected;
    p.count = (int)count;
    p.causal = (flags & FA_FLAG_CAUSAL) != 0;
    p.tiles = (int)a.tiles;
    p.splits = (int)a.splits;
    p.by_parts = fa::divisor(a.wgs / a.tiles);
    p.by_splits = fa::divisor(a.splits);
    p.by_heads = fa::divisor(cache->heads);
    p.by_group = fa::divisor(p.group);
    int power;                                           // scale_log2e is at least 2^(power - 1)
    std::frexp(p.scale_log2e, &power);
    p.least_exponent = -125 - power;
    const int64_t rows = B * L * R;
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = p.part_o + rows * a.splits * H;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return static_cast<int>(for_type(H, (flags & FA_FLAG_BF16) != 0, [&](auto h, auto b) {
        using namespace fa::cache;
        constexpr int threads = 64 * kAttendWaves;
        hipError_t e;
        if (a.wide) {
            auto kernel = a.nq == 1 ? cached_attention_wide_kernel<h(), b(), 1> : cached_attention_wide_kernel<h(), b(), 2>;
            const int lds = a.nq == 1 ? wide_lds_bytes<h(), 1>() : wide_lds_bytes<h(), 2>();
            e = allow_large_lds(reinterpret_cast<const void*>(kernel), lds);
            if (e == hipSuccess) e = launch(kernel, a.wgs, 64 * kWideWaves, p, lds, s);
        } else if (count > 0) {
            auto kernel = a.shared       ? (a.waves == 2 ? cached_attention_kernel<h(), b(), 1, 2, kShared> : cached_attention_kernel<h(), b(), 1, kAttendWaves, kShared>)
                          : a.waves == 8 ? cached_attention_kernel<h(), b(), 1, 8, kListed>
                          : a.waves == 1 ? cached_attention_kernel<h(), b(), 1, 1, kListed>
                                         : cached_attention_kernel<h(), b(), 1, kAttendWaves, kListed>;
            // a list; joined: two bytes a page of the table, and the pages that are listed (beside up to 64 KiB of the kernel's own)
            const int64_t joined = shared_tokens(p.group) * count;
            const int lds = 4 * (int)(a.shared ? (p.W + 1) / 2 + (joined < p.W ? joined : p.W) : count);
            e = allow_large_lds(reinterpret_cast<const void*>(kernel), a.shared ? 6 * kMostShared : 4 * kMostSelected);
            if (e == hipSuccess) e = launch(kernel, a.wgs, 64 * a.waves, p, lds, s);
        } else if (a.nq == 1) {
            e = launch(cached_attention_kernel<h(), b(), 1, kAttendWaves, kEvery>, a.wgs, threads, p, 0, s);
        } else {
            e = launch(cached_attention_kernel<h(), b(), 2, kAttendWaves, kEvery>, a.wgs, threads, p, 0, s);
        }
        if (e != hipSuccess || a.splits == 1) return e;
        return launch(cached_attention_join_kernel<h(), b()>, ceil_div(rows, 4), 256, p, 0, s);
    }));
}

int fa_cached_attention_plan(const fa_cache* cache, int64_t L, int64_t R, int64_t count, int* plan) {
    View p;
    if (plan == nullptr) return FA_ERR_NULL_POINTER;
    int rc = check_sizes(cache, L, R, &p);
    if (rc == FA_OK) rc = check_count(count);
    if (rc == FA_OK && count < 0) rc = FA_ERR_BAD_SHAPE;
    if (rc != FA_OK) return rc;
    const AttendPlan a = plan_attend(p, count, cache->head_dim);
    if (a.wgs > kMaxInt) return FA_ERR_TOO_LARGE;
    plan[0] = a.wide ? 1 : a.shared ? 2 : 0;
    plan[1] = a.waves;
    plan[2] = 16 * a.nq * (a.wide ? fa::cache::kWideWaves : 1);
    plan[3] = (int)a.splits;
    plan[4] = (int)a.wgs;
    return FA_OK;
}

int fa_select_pages_plan(const fa_cache* cache, int64_t L, int64_t R, int* plan) {
    View p;
    if (plan == nullptr) return FA_ERR_NULL_POINTER;
    const int rc = check_sizes(cache, L, R, &p);
    if (rc != FA_OK) return rc;
    if (p.W > kMostTable) return FA_ERR_TOO_LARGE;
    const SelectPlan a = plan_select(p);
    if (a.wgs > kMaxInt) return FA_ERR_TOO_LARGE;
    plan[0] = (int)a.tokens;
    plan[1] = a.waves;
    plan[2] = (int)a.wgs;
    return FA_OK;
}

int fa_select_pages(const fa_cache* cache, const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, int32_t* selected,
                    int64_t count, const int32_t* starts, const int32_t* new_lens, int64_t L, int64_t R, int flags, void* stream) {
    if ((flags & ~FA_FLAG_BF16) != 0) return FA_ERR_BAD_FLAGS;
    SelectParams p;
    int rc = check_sizes(cache, L, R, &p);
    if (rc == FA_OK) rc = check_tensors(cache, starts, new_lens, false, &p);
    if (rc != FA_OK) return rc;
    if (selected == nullptr || cache->key_bounds == nullptr) return FA_ERR_NULL_POINTER;
    if (count < 1) return FA_ERR_BAD_SHAPE;
    if (p.W > kMostTable || (rc = check_count(count)) != FA_OK) return FA_ERR_TOO_LARGE;
    p.qs = {q_stride_b, q_stride_h, q_stride_l};
    if ((rc = check_strided(q, p.qs, p.B, R, L, cache->head_dim)) != FA_OK) return rc;
    if (!aligned(selected, 4)) return FA_ERR_MISALIGNED;
    p.q = static_cast<const uint16_t*>(q);
    p.selected = selected;
    p.count = (int)count;
    const SelectPlan a = plan_select(p);
    if (a.wgs > kMaxInt || a.wgs > kMostThreads / (64 * a.waves)) return FA_ERR_TOO_LARGE;
    p.by_heads = fa::divisor(p.Rkv);
    p.tiles = (int)ceil_div(L, a.tokens);
    p.by_tokens = fa::divisor(p.tiles);
    return static_cast<int>(for_type(cache->head_dim, (flags & FA_FLAG_BF16) != 0, [&](auto h, auto b) {
        using namespace fa::cache;
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (a.tokens > 1) return launch(select_pages_rows_kernel<h(), b()>, a.wgs, 64 * a.waves, p, (int)a.tokens * p.W * 4, s);
        auto kernel = a.waves == 4 ? select_pages_kernel<h(), b(), 256> : select_pages_kernel<h(), b(), 1024>;
        const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kernel), kMostTable * 4);
        if (e != hipSuccess) return e;
        return launch(kernel, a.wgs, 64 * a.waves, p, p.W * 4, s);
    }));
}

}  // extern "C"
