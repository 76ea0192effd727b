// C ABI of the latent attention (include/fused_attn.h): argument validation, the choice of launch and the launches.
#include "host_checks.hpp"
#include "latent_kernels.hpp"

namespace {

using namespace fa::latent;

// f(std::integral_constant<int, C>, std::integral_constant<int, DR>, std::bool_constant<BF>)
template <class F>
hipError_t for_latent(int64_t C, int64_t DR, bool bf, F f) {
    auto with = [&](auto c, auto d) { return bf ? f(c, d, std::true_type{}) : f(c, d, std::false_type{}); };
    auto wide = [&](auto c) { return DR == 32 ? with(c, std::integral_constant<int, 32>{}) : with(c, std::integral_constant<int, 64>{}); };
    return C == 128 ? wide(std::integral_constant<int, 128>{}) : C == 256 ? wide(std::integral_constant<int, 256>{}) : wide(std::integral_constant<int, 512>{});
}

int check_sizes(const fa_latent_cache* c, int64_t L, int64_t R, View* p) {
    if (c == nullptr) return FA_ERR_NULL_POINTER;
    if ((c->latent_dim != 128 && c->latent_dim != 256 && c->latent_dim != 512) || (c->rope_dim != 32 && c->rope_dim != 64)) return FA_ERR_BAD_HEAD_DIM;
    int log2_p = 4;
    while (log2_p < 7 && ((int64_t)1 << log2_p) < c->page_size) ++log2_p;
    if (c->page_size != (int64_t)1 << log2_p) return FA_ERR_BAD_PAGE;
    if (c->pages < 1 || c->sequences < 1 || c->table_width < 1 || L < 1 || R < 1) return FA_ERR_BAD_SHAPE;
    if (c->table_stride < 0 || (c->table_stride < c->table_width && c->sequences > 1)) return FA_ERR_BAD_STRIDE;
    if (c->pages > kMaxInt || R > kMaxInt || L > kMaxInt || c->sequences > kMaxInt || !below(c->table_width, c->page_size, kMaxInt) ||
        !below(L, R, kMaxInt) || !below(L * R, c->sequences, kMaxInt) || !below(c->table_stride, c->sequences, kMaxElems))
        return FA_ERR_TOO_LARGE;
    p->latents = static_cast<uint16_t*>(c->latents);
    p->table = c->page_table;
    p->table_stride = c->table_stride;
    p->B = (int)c->sequences;
    p->L = (int)L;
    p->R = (int)R;
    p->W = (int)c->table_width;
    p->pages = (int)c->pages;
    p->log2_p = log2_p;
    return FA_OK;
}

int check_tensors(const fa_latent_cache* c, const int32_t* starts, const int32_t* new_lens, View* p) {
    if (starts == nullptr || c->page_table == nullptr || c->latents == nullptr) return FA_ERR_NULL_POINTER;
    if (!aligned(starts, 4) || !aligned(new_lens, 4) || !aligned(c->page_table, 4) || !aligned(c->latents, 16)) return FA_ERR_MISALIGNED;
    p->starts = starts;
    p->new_lens = new_lens;
    return FA_OK;
}

// A tensor of one row a token.
int check_rows(const void* t, int64_t stride_b, int64_t stride_l, int64_t B, int64_t L, int64_t n) {
    return check_strided(t, {stride_b, 0, stride_l}, B, 1, L, n);
}

// [B, L, heads, n] by strides of its own, where a head may stand next to the next one's token: stride_l need not reach over a row.
int check_heads(const void* t, const Strides3& s, int64_t B, int64_t heads, int64_t L, int64_t n) {
    if (t == nullptr) return FA_ERR_NULL_POINTER;
    if (s.b < 0 || s.h < 0 || s.l < 0 || s.b % 8 != 0 || s.h % 8 != 0 || s.l % 8 != 0) return FA_ERR_BAD_STRIDE;
    if (!aligned(t, 16)) return FA_ERR_MISALIGNED;
    if ((s.l > 0 && !below(L, s.l, kMaxElems)) || (s.h > 0 && !below(heads, s.h, kMaxElems)) || (s.b > 0 && !below(B, s.b, kMaxElems)))
        return FA_ERR_TOO_LARGE;
    (void)n;
    return FA_OK;
}

bool scale_of(float scale, float* scale_log2e) {
    *scale_log2e = scale * 1.4426950408889634f;
    return scale > 0.f && std::isfinite(*scale_log2e);
}

// How latent_attention is launched.
struct LatentPlan {
    int nq;
    int64_t tiles, units, groups, wgs;       // groups: 0, a workgroup a unit
    int least_share;
};

// Rows of a workgroup by what a launch is estimated to take: tiles of 64 rows take less for each row, of 32 less to begin and to join.
// (C = 512, us, 32 and 64 rows, with the joining: 16 sequences of 2000 tokens, 160 rows each 36, 38; 2 of them 22, 25; one of 32000
// 35, 38; 128 rows of one of 131072 73, 65.)  Both are for the table's width, the lengths being in device memory, and used for 128 and 256 channels too,
// whose tiles take less than the estimate says.
LatentPlan plan_latent(const View& p, int64_t C) {
    LatentPlan a;
    const int64_t rows = (int64_t)p.L * p.R, steps = ceil_div((int64_t)p.W << p.log2_p, kKeys), resident = (C == 128 ? 2 : 1) * kNumCu;
    a.least_share = 2;                       // key tiles
    auto estimate = [&](int nq) {            // us / 0.4
        const double units = (double)p.B * (double)ceil_div(rows, 16 * nq), shares = units * (double)ceil_div(steps, a.least_share);
        return (nq == 2 ? 20. : 27.) + (nq == 2 ? 3.3 : 4.6) * units * (double)steps / (shares < (double)resident ? shares : (double)resident);
    };
    a.nq = rows <= 16 ? 1 : rows <= 32 || estimate(2) < estimate(4) ? 2 : 4;
    a.tiles = ceil_div(rows, 16 * a.nq);
    a.units = p.B * a.tiles;
    // None shared out where one workgroup is through with its unit before a second kernel would be (C = 128, 4 tiles: 5 us, shared out 10), nor from two
    // units for each place on: they even each other out where lengths are alike, but one long sequence is as slow as its own tiles are one after the
    // other (512 of 1000 tokens, 16 rows, one of them of 131072: 3960 us; 511 of them, shared out, 158).
    a.groups = 0;
    if (a.units <= kMostUnits && a.units < 2 * resident && steps > 2 + 768 / C && below(steps, a.units, 0x3fffffff)) {
        const int64_t shares = a.units * ceil_div(steps, a.least_share);         // more have nothing to do
        a.groups = shares < resident ? shares : resident;
    }
    a.wgs = a.groups > 0 ? ceil_div(a.groups, 8) * 8 : a.units;
    return a;
}

// The parts' sums, their log-sum-exps and the plan.
int64_t latent_workspace(const LatentPlan& a, int64_t C) {
    return a.groups > 0 ? ((a.groups + a.units) * 16 * a.nq * (C + 1) + 2 * a.units + 1) * 4 : 0;
}

// How expanded_attention is launched.
struct Plan {
    int nq;
    int64_t tiles, splits, wgs;
};

// Waves that join the parts of a row, about so many of them.
int join_waves(int64_t parts) { return parts >= 32 ? 16 : parts >= 8 ? 4 : 1; }

constexpr int64_t kMostParts = 128;          // of a row's keys

// Rooms of LDS for tiles: two where that lets a third workgroup onto a compute unit that has one to take.
int rooms_of(int nq, int64_t wgs, int64_t D) { return nq == 1 && D == 64 && wgs > 2 * kNumCu ? 2 : 3; }

// Rows of a workgroup and parts of the keys by what a launch is estimated to take, causal (what the caller asks for is not known where the
// workspace is sized): the longest workgroup's tiles, each `alone` us, or all tiles by what a compute unit takes for one, and the second
// kernel's.  (Measured, with 128 and with 256 rows, us: 8 sequences of 1001 tokens of 12 heads of 64: 32, 38; 4 of them 23, 33; 16 of 500 of
// 16 heads 29, 27; 4 of 2048 of 16 heads 71, 78; 2048 tokens of 16 heads of 128, 4 sequences 142, 111; one of 4096 118, 152; 4096 behind 12288, 32 heads 1357, 1067.)
Plan plan_expanded(int64_t B, int64_t L, int64_t R, int64_t K, int64_t D) {
    Plan best = {};
    float best_us = 3.0e38f;
    const float longest = (float)ceil_div(K, kKeys), halfway = K > L ? ((float)K - 0.5f * (float)L) / kKeys : 0.5f * longest;
    for (int nq = 1; nq <= 2; ++nq) {
        const float alone = D == 128 ? (nq == 2 ? 2.2f : 1.4f) : (nq == 2 ? 1.65f : 1.3f);
        const int64_t tiles = ceil_div(L, kExpandedWaves * 16 * nq), base = B * R * tiles;
        for (int64_t s = 1; s <= kMostParts && (s == 1 || (base * s <= 4 * kNumCu && 2 * s <= ceil_div(K, kKeys))); s *= 2) {
            const bool many = rooms_of(nq, base * s, D) == 2;
            const float each = D == 128 ? alone : nq == 2 ? 1.9f : many ? 0.86f : 0.9f, begin = many ? 1.55f : 0.f;
            const float mean = D == 128 ? halfway : halfway + (float)nq, steps = mean < longest ? mean : longest;
            const float chain = alone * (float)ceil_div((int64_t)longest, s), all = (each * steps + begin * (float)s) * (float)base / kNumCu;
            const float join = s > 1 ? 4.f + (float)(B * L * R) * (float)(s * D) * 8.f / 2.5e6f : 0.f;
            const float us = 6.f + (chain > all ? chain : all) + join;
            if (us < best_us) best_us = us, best = {nq, tiles, s, base * s};
        }
    }
    return best;
}

int64_t parts_bytes(int64_t rows, int64_t splits, int64_t C) { return splits > 1 ? rows * splits * (C + 1) * 4 : 0; }

int check_workspace(const void* workspace, int64_t bytes, int64_t need) {
    if (need > 0 && (workspace == nullptr || bytes < need)) return FA_ERR_WORKSPACE;
    return need > 0 && !aligned(workspace, 16) ? FA_ERR_MISALIGNED : FA_OK;
}

int check_expanded(const fa_expanded* x) {
    if (x == nullptr) return FA_ERR_NULL_POINTER;
    if ((x->key_dim != 64 && x->key_dim != 128) || x->value_dim != x->key_dim || (x->rope_dim != 32 && x->rope_dim != 64)) return FA_ERR_BAD_HEAD_DIM;
    const int64_t B = x->sequences, L = x->tokens, R = x->heads, K = x->keys;
    if (B < 1 || L < 1 || R < 1 || K < 1) return FA_ERR_BAD_SHAPE;
    if (B > kMaxInt || L > kMaxInt || R > kMaxInt || K > kMaxInt || !below(L, R, kMaxInt) || !below(L * R, B, kMaxInt)) return FA_ERR_TOO_LARGE;
    return FA_OK;
}

}  // namespace

extern "C" {

int fa_latent_append(const fa_latent_cache* cache, const void* c, int64_t c_stride_b, int64_t c_stride_l, const void* k, int64_t k_stride_b,
                     int64_t k_stride_l, const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, void* q_out,
                     int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_l, const int32_t* starts, const int32_t* new_lens, int64_t L,
                     int64_t R, const float* rope_cos, const float* rope_sin, int64_t rope_rows, int flags, void* stream) {
    if ((flags & ~(FA_FLAG_BF16 | FA_FLAG_INTERLEAVED)) != 0) return FA_ERR_BAD_FLAGS;
    AppendParams p;
    int rc = check_sizes(cache, L, q != nullptr || cache == nullptr ? R : 1, &p);
    if (rc == FA_OK) rc = check_tensors(cache, starts, new_lens, &p);
    if (rc != FA_OK) return rc;
    const int64_t B = cache->sequences, C = cache->latent_dim, DR = cache->rope_dim;
    if ((rc = check_rows(c, c_stride_b, c_stride_l, B, L, C)) != FA_OK) return rc;
    if ((rc = check_rows(k, k_stride_b, k_stride_l, B, L, DR)) != FA_OK) return rc;
    p.qs = {q_stride_b, q_stride_h, q_stride_l};
    p.qo = {out_stride_b, out_stride_h, out_stride_l};
    if ((q == nullptr) != (q_out == nullptr)) return FA_ERR_NULL_POINTER;
    if (q != nullptr && (rc = check_heads(q, p.qs, B, R, L, DR)) != FA_OK) return rc;
    if (q != nullptr && (rc = check_written(q_out, p.qo, B, R, L, DR)) != FA_OK) return rc;
    if ((rope_cos == nullptr) != (rope_sin == nullptr)) return FA_ERR_NULL_POINTER;
    if (rope_cos != nullptr && rope_rows < 1) return FA_ERR_BAD_SHAPE;
    if (!aligned(rope_cos, 16) || !aligned(rope_sin, 16)) return FA_ERR_MISALIGNED;
    if (!below(B * L, (C + DR) / 16, kMaxInt) || (q != nullptr && !below(B * L * R, DR / 16, kMaxInt))) return FA_ERR_TOO_LARGE;
    p.c = static_cast<const uint16_t*>(c);
    p.k = static_cast<const uint16_t*>(k);
    p.c_stride_b = c_stride_b, p.c_stride_l = c_stride_l, p.k_stride_b = k_stride_b, p.k_stride_l = k_stride_l;
    p.q = static_cast<const uint16_t*>(q);
    p.q_out = static_cast<uint16_t*>(q_out);
    p.cos = rope_cos;
    p.sin = rope_sin;
    p.rope_rows = rope_rows;
    p.C = (int)C;
    p.DR = (int)DR;
    p.cache_units = B * L * ((C + DR) / 16);
    p.q_units = q != nullptr ? B * L * R * (DR / 16) : 0;
    p.by_units = fa::divisor((C + DR) / 16);
    p.by_q_units = fa::divisor(DR / 16);
    p.by_heads = fa::divisor(p.R);
    p.by_tokens = fa::divisor(L);
    const bool bf = (flags & FA_FLAG_BF16) != 0, il = (flags & FA_FLAG_INTERLEAVED) != 0;
    auto kernel = bf ? (il ? latent_append_kernel<true, true> : latent_append_kernel<true, false>)
                     : (il ? latent_append_kernel<false, true> : latent_append_kernel<false, false>);
    return static_cast<int>(launch(kernel, ceil_div(p.cache_units + p.q_units, 256), 256, p, 0, static_cast<hipStream_t>(stream)));
}

int64_t fa_latent_attention_workspace(const fa_latent_cache* cache, int64_t L, int64_t R) {
    View p;
    const int rc = check_sizes(cache, L, R, &p);
    if (rc != FA_OK) return rc;
    return latent_workspace(plan_latent(p, cache->latent_dim), cache->latent_dim);
}

int fa_latent_attention(const fa_latent_cache* cache, const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, const void* r,
                        int64_t r_stride_b, int64_t r_stride_h, int64_t r_stride_l, void* out, int64_t out_stride_b, int64_t out_stride_h,
                        int64_t out_stride_l, void* lse, const int32_t* starts, const int32_t* new_lens, int64_t L, int64_t R, float scale,
                        int flags, void* workspace, int64_t workspace_bytes, void* stream) {
    if ((flags & ~(FA_FLAG_BF16 | FA_FLAG_CAUSAL)) != 0) return FA_ERR_BAD_FLAGS;
    AttendParams p;
    int rc = check_sizes(cache, L, R, &p);
    if (rc == FA_OK) rc = check_tensors(cache, starts, new_lens, &p);
    if (rc != FA_OK) return rc;
    if (!scale_of(scale, &p.scale_log2e)) return FA_ERR_BAD_SCALE;
    const int64_t B = cache->sequences, C = cache->latent_dim, DR = cache->rope_dim;
    p.qs = {q_stride_b, q_stride_h, q_stride_l};
    p.rs = {r_stride_b, r_stride_h, r_stride_l};
    p.os = {out_stride_b, out_stride_h, out_stride_l};
    if ((rc = check_heads(q, p.qs, B, R, L, C)) != FA_OK) return rc;
    if ((rc = check_heads(r, p.rs, B, R, L, DR)) != FA_OK) return rc;
    if ((rc = check_written(out, p.os, B, R, L, C)) != FA_OK) return rc;
    if (!aligned(lse, 4)) return FA_ERR_MISALIGNED;
    const LatentPlan a = plan_latent(p, C);
    if (a.wgs > kMaxInt || a.wgs > kMostThreads / 512) return FA_ERR_TOO_LARGE;
    if ((rc = check_workspace(workspace, workspace_bytes, latent_workspace(a, C))) != FA_OK) return rc;
    p.q = static_cast<const uint16_t*>(q);
    p.r = static_cast<const uint16_t*>(r);
    p.out = static_cast<uint16_t*>(out);
    p.lse = static_cast<float*>(lse);
    p.causal = (flags & FA_FLAG_CAUSAL) != 0;
    p.tiles = (int)a.tiles;
    p.units = (int)a.units;
    p.groups = (int)a.groups;
    p.least_share = a.least_share;
    p.rows_of_unit = 16 * a.nq;
    const int64_t parts = (a.groups + a.units) * 16 * a.nq;
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = p.part_o + parts * C;
    p.plan = reinterpret_cast<int32_t*>(p.part_lse + parts);
    p.by_heads = fa::divisor(R);
    p.by_tiles = fa::divisor(a.tiles);
    p.by_sequences = fa::divisor(B);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return static_cast<int>(for_latent(C, DR, (flags & FA_FLAG_BF16) != 0, [&](auto c, auto d, auto bf) {
        auto run = [&](auto nq) {
            using S = Shape<c(), d(), nq()>;
            auto kernel = latent_attention_kernel<c(), d(), bf(), nq()>;
            const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kernel), S::kLds);
            return e != hipSuccess ? e : launch(kernel, a.wgs, 64 * S::WAVES, p, S::kLds, s);
        };
        const hipError_t e = a.nq == 1   ? run(std::integral_constant<int, 1>{})
                             : a.nq == 2 ? run(std::integral_constant<int, 2>{})
                                         : run(std::integral_constant<int, 4>{});
        if (e != hipSuccess || a.groups == 0) return e;
        const int waves = join_waves(a.groups / a.units);
        auto kernel = waves == 16 ? latent_join_kernel<c(), bf(), 16> : waves == 4 ? latent_join_kernel<c(), bf(), 4> : latent_join_kernel<c(), bf(), 1>;
        return launch(kernel, ceil_div(B * L * R, rows_of_join(waves)), waves > 1 ? 64 * waves : 256, p, 0, s);
    }));
}

int fa_latent_attention_plan(const fa_latent_cache* cache, int64_t L, int64_t R, int* plan) {
    View p;
    if (plan == nullptr) return FA_ERR_NULL_POINTER;
    const int rc = check_sizes(cache, L, R, &p);
    if (rc != FA_OK) return rc;
    const LatentPlan a = plan_latent(p, cache->latent_dim);
    if (a.wgs > kMaxInt) return FA_ERR_TOO_LARGE;
    plan[0] = 16 * a.nq;
    plan[1] = a.groups > 0;
    plan[2] = (int)a.wgs;
    return FA_OK;
}

int64_t fa_expanded_attention_workspace(const fa_expanded* x) {
    const int rc = check_expanded(x);
    if (rc != FA_OK) return rc;
    return parts_bytes(x->sequences * x->tokens * x->heads, plan_expanded(x->sequences, x->tokens, x->heads, x->keys, x->key_dim).splits, x->value_dim);
}

int fa_expanded_attention(const fa_expanded* x, float scale, int flags, void* workspace, int64_t workspace_bytes, void* stream) {
    if ((flags & ~(FA_FLAG_BF16 | FA_FLAG_CAUSAL)) != 0) return FA_ERR_BAD_FLAGS;
    int rc = check_expanded(x);
    if (rc != FA_OK) return rc;
    ExpandedParams p;
    if (!scale_of(scale, &p.scale_log2e)) return FA_ERR_BAD_SCALE;
    const int64_t B = x->sequences, L = x->tokens, R = x->heads, K = x->keys, D = x->key_dim, DR = x->rope_dim;
    p.qs = {x->q_strides[0], x->q_strides[1], x->q_strides[2]};
    p.ks = {x->k_strides[0], x->k_strides[1], x->k_strides[2]};
    p.vs = {x->v_strides[0], x->v_strides[1], x->v_strides[2]};
    p.os = {x->out_strides[0], x->out_strides[1], x->out_strides[2]};
    p.kr_stride_b = x->rope_k_strides[0], p.kr_stride_l = x->rope_k_strides[1];
    if ((rc = check_heads(x->q, p.qs, B, R, L, D + DR)) != FA_OK) return rc;
    if ((rc = check_heads(x->k, p.ks, B, R, K, D)) != FA_OK) return rc;
    if ((rc = check_heads(x->v, p.vs, B, R, K, D)) != FA_OK) return rc;
    if ((rc = check_heads(x->rope_k, {p.kr_stride_b, 0, p.kr_stride_l}, B, 1, K, DR)) != FA_OK) return rc;
    if ((rc = check_written(x->out, p.os, B, R, L, D)) != FA_OK) return rc;
    if (!aligned(x->lse, 4) || !aligned(x->starts, 4) || !aligned(x->new_lens, 4)) return FA_ERR_MISALIGNED;
    constexpr int64_t kMostStride = (int64_t)1 << 24;    // the loads' offsets within 16 keys have 32 bits
    if (p.ks.l > kMostStride || p.vs.l > kMostStride || p.kr_stride_l > kMostStride) return FA_ERR_TOO_LARGE;
    const Plan a = plan_expanded(B, L, R, K, D);
    if (a.wgs > kMaxInt || a.wgs > kMostThreads / (64 * kExpandedWaves)) return FA_ERR_TOO_LARGE;
    const int64_t rows = B * L * R;
    if ((rc = check_workspace(workspace, workspace_bytes, parts_bytes(rows, a.splits, D))) != FA_OK) return rc;
    p.q = static_cast<const uint16_t*>(x->q);
    p.k = static_cast<const uint16_t*>(x->k);
    p.kr = static_cast<const uint16_t*>(x->rope_k);
    p.v = static_cast<const uint16_t*>(x->v);
    p.out = static_cast<uint16_t*>(x->out);
    p.lse = static_cast<float*>(x->lse);
    p.starts = x->starts;
    p.new_lens = x->new_lens;
    p.B = (int)B, p.L = (int)L, p.R = (int)R, p.K = (int)K;
    p.causal = (flags & FA_FLAG_CAUSAL) != 0;
    p.tiles = (int)a.tiles;
    p.splits = (int)a.splits;
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = p.part_o + rows * a.splits * D;
    p.by_parts = fa::divisor(B * R * a.splits);
    p.by_splits = fa::divisor(a.splits);
    p.by_heads = fa::divisor(R);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto with = [&](auto d, auto dr, auto bf) {
        auto run = [&](auto nq, auto rooms) {
            auto kernel = expanded_attention_kernel<d(), dr(), bf(), nq(), rooms()>;
            constexpr int lds = Expanded<d(), dr(), rooms()>::kLds;
            const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kernel), lds);
            return e != hipSuccess ? e : launch(kernel, a.wgs, 64 * kExpandedWaves, p, lds, s);
        };
        auto in_rooms = [&]() {
            constexpr std::integral_constant<int, 1> one;
            constexpr std::integral_constant<int, 3> three;
            if (a.nq == 2) return run(std::integral_constant<int, 2>{}, three);
            if constexpr (d() == 64) {
                if (rooms_of(a.nq, a.wgs, D) == 2) return run(one, std::integral_constant<int, 2>{});
            }
            return run(one, three);
        };
        const hipError_t e = in_rooms();
        if (e != hipSuccess || a.splits == 1) return e;
        const int waves = join_waves(a.splits);
        auto kernel = waves == 16 ? expanded_join_kernel<d(), bf(), 16> : waves == 4 ? expanded_join_kernel<d(), bf(), 4> : expanded_join_kernel<d(), bf(), 1>;
        return launch(kernel, ceil_div(rows, rows_of_join(waves)), waves > 1 ? 64 * waves : 256, p, 0, s);
    };
    auto typed = [&](auto d, auto dr) { return (flags & FA_FLAG_BF16) != 0 ? with(d, dr, std::true_type{}) : with(d, dr, std::false_type{}); };
    auto wide = [&](auto d) { return DR == 32 ? typed(d, std::integral_constant<int, 32>{}) : typed(d, std::integral_constant<int, 64>{}); };
    return static_cast<int>(D == 64 ? wide(std::integral_constant<int, 64>{}) : wide(std::integral_constant<int, 128>{}));
}

int fa_expanded_attention_plan(const fa_expanded* x, int* plan) {
    if (plan == nullptr) return FA_ERR_NULL_POINTER;
    const int rc = check_expanded(x);
    if (rc != FA_OK) return rc;
    const Plan a = plan_expanded(x->sequences, x->tokens, x->heads, x->keys, x->key_dim);
    if (a.wgs > kMaxInt) return FA_ERR_TOO_LARGE;
    plan[0] = 16 * a.nq * kExpandedWaves;
    plan[1] = (int)a.splits;
    plan[2] = (int)a.wgs;
    return FA_OK;
}

}  // extern "C"
