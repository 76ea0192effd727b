/*
 * C ABI of the gfx950 fused multi-head attention forward library
 * (libfused_attn_gfx950.so).  Plain pointers and sizes only: no torch types, no HIP
 * types in the signatures, so the same entry points can be bound from C++, ctypes or
 * any FFI.
 *
 * All tensors are IEEE fp16 in device memory.  q, k, v and out share one addressing
 * rule, given in ELEMENTS:
 *     element(b, h, l, d) = base + b*stride_b + h*stride_h + l*stride_l + d      (d < H)
 * The reference layout [B, L, R*H] (reference src/fused_attn_extention.cu:24-27,50-52;
 * head h = columns [h*H, (h+1)*H), reference include/fused_attn.cuh:683-690) is
 *     stride_b = L*R*H, stride_h = H, stride_l = R*H,
 * and a [B, R, L, H] tensor is stride_b = R*L*H, stride_h = L*H, stride_l = H.
 * Strides must be multiples of 8 elements and the base pointers 16-byte aligned.
 *
 * Return value of every int function: 0 = success, < 0 = invalid argument (FA_ERR_*),
 * > 0 = a hipError_t raised by the runtime.  Nothing here ever calls exit().
 */
#ifndef FUSED_ATTN_H_
#define FUSED_ATTN_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FA_OK 0
#define FA_ERR_NULL_POINTER (-1)
#define FA_ERR_BAD_HEAD_DIM (-2)
#define FA_ERR_BAD_SHAPE (-3)
#define FA_ERR_BAD_STRIDE (-4)
#define FA_ERR_MISALIGNED (-5)
#define FA_ERR_TOO_LARGE (-6)
#define FA_ERR_BAD_FLAGS (-7)
#define FA_ERR_BAD_SCALE (-8)
#define FA_ERR_BAD_PAGE (-9)
#define FA_ERR_WORKSPACE (-10)

#define FA_FLAG_CAUSAL 1
#define FA_FLAG_BF16 2
#define FA_FLAG_INTERLEAVED 4
#define FA_FLAG_INVERSE 8

/*
 * out = softmax(q k^T * scale [+ mask]) v for every (batch, head), non-causal.
 *
 * Replaces launch_attention_kernel<head_dim, chunk_size>(batch_size, seq_len,
 * num_features, queries, keys, values, mask, output, syncronize)
 * (reference include/fused_attn.cuh:860-894) together with the kernel it launches
 * (reference include/fused_attn.cuh:605-858).  Differences a caller can see:
 *   - head_dim is a run-time argument (16, 32, 64 or 128), there is no chunk_size:
 *     the key tile is an internal choice and L need not be a multiple of anything;
 *   - the launch goes to `stream` (a hipStream_t, NULL = the null stream) and the
 *     call returns without synchronising;
 *   - `mask` (nullable) is an additive fp16 [B, L, L] tensor shared by all heads and is
 *     applied to every key, not only to the first chunk.  Rows whose keys are all -inf
 *     produce zeros.
 * `scale` is finite and > 0 (FA_ERR_BAD_SCALE otherwise); the reference fixes it at
 * 1/sqrt(head_dim) (reference include/fused_attn.cuh:727).
 * B, R, L >= 1.  L*stride_l, R*stride_h and B*stride_b must stay below 2^62 elements and
 * stride_l must not exceed 2^24 elements (FA_ERR_TOO_LARGE otherwise).
 * Accuracy: scores, softmax state and both products are accumulated in float32; the softmax
 * weights are rounded to fp16 before they multiply the values, scaled by a power of two chosen
 * from L so that a row of L keys loses at most 2^-13 (1.2e-4) of its weight to the bottom of the
 * fp16 range: a key more than 13 + ceil(log2 L) log2 units below the largest score of its row
 * contributes nothing (25 units, 17 natural-log units, at L = 4096).  The reference accumulates
 * everything in fp16 (reference include/fused_attn.cuh:174,257,650-653).
 */
int fa_fwd(const void* q, const void* k, const void* v, const void* mask, void* out,
           int64_t B, int64_t R, int64_t L, int64_t H,
           int64_t stride_b, int64_t stride_h, int64_t stride_l,
           float scale, void* stream);

/*
 * fa_fwd with two extensions the reference lists as not done yet (reference README.md:135-142,
 * "backward pass", and its GPT/LLaMA use case, README.md:8):
 *   flags & FA_FLAG_CAUSAL : query i attends to keys j <= i only; key tiles above the diagonal
 *                            are skipped.  Not combinable with `mask`.
 *   flags & FA_FLAG_BF16   : q, k, v, out (and mask) hold bfloat16 instead of fp16 (reference
 *                            README.md:137 lists other input types as not done).  Same kernels,
 *                            bf16 matrix instructions, probabilities rounded to bf16 (with the exponents
 *                            of float32: no key of a row is too small to contribute).
 *   lse (nullable)         : float32 [B, R, L] in device memory, receives
 *                            log(sum_j exp(score_ij)) per query row (-inf for a row whose keys
 *                            are all masked): what a backward pass needs to recompute the
 *                            probabilities.
 * Everything else as fa_fwd, which is fa_fwd_ex with lse = NULL and flags = 0.  There is no
 * counterpart in the reference (its kernel is non-causal and keeps no row statistics).
 */
int fa_fwd_ex(const void* q, const void* k, const void* v, const void* mask, void* out, void* lse,
              int64_t B, int64_t R, int64_t L, int64_t H,
              int64_t stride_b, int64_t stride_h, int64_t stride_l,
              float scale, int flags, void* stream);

/*
 * fa_fwd_ex with strides of its own for `out`: q, k and v share (stride_b, stride_h, stride_l),
 * out is addressed with (out_stride_b, out_stride_h, out_stride_l), under the same rules
 * (multiples of 8 elements, last dimension contiguous; the 2^24 limit applies to stride_l only).
 * This is what lets q, k and v be three views into one packed projection output (say
 * [B, L, 3, R, H], the layout a fused QKV projection writes: reference README.md:137 lists that
 * front end as not done) while out is an ordinary contiguous tensor, with no copy on either side.
 * The reference has no counterpart: its launcher takes contiguous [B, L, R*H] tensors only
 * (reference src/fused_attn_extention.cu:34-44).
 */
int fa_fwd_strided(const void* q, const void* k, const void* v, const void* mask, void* out, void* lse,
                   int64_t B, int64_t R, int64_t L, int64_t H,
                   int64_t stride_b, int64_t stride_h, int64_t stride_l,
                   int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_l,
                   float scale, int flags, void* stream);

/*
 * The launch the library would make for a problem, without making it (no GPU is touched): for
 * tests of the launcher and for tuning.  has_mask != 0 stands for an additive mask.  Fills plan[0..6]
 * with: wave64s per workgroup; query rows per wave (waves may share them, see fa_fwd_variant);
 * workgroups launched; workgroups that do work (the rest exit at once); workgroups per (batch, head),
 * or pairs of query tiles per head for a causal launch of a tile kernel and for those masked
 * launches of one that pairs cost no round of the chip; 0, or, when the query tiles of a causal launch
 * are dealt out to a resident grid, the heads per XCD; the edge of the matrix instruction's tile: 16,
 * or, in a tile kernel, 32 except at head_dim 64 and 128 for plain launches whose workgroups fill whole
 * rounds of the chip (the last round at least seven eighths full) and for causal launches from seven
 * eighths of a round on.
 * (A problem whose grid would have 2^32 threads or more is launched in parts, halves of its batch or heads.)
 * The reference has no counterpart (its grid is fixed at (B, L / chunk_size, R),
 * reference include/fused_attn.cuh:872-883).
 */
int fa_fwd_plan(int64_t B, int64_t R, int64_t L, int64_t H, int flags, int has_mask, int* plan);

/*
 * Which kernel fa_fwd runs a problem on, without running it (no GPU is touched), has_mask as in fa_fwd_plan.
 * Fills variant[0..6] with: 0 = a tile kernel, 1 = the key-split kernel, 2 = the group kernel; waves per workgroup; query rows per workgroup; waves that share a row's keys between
 * them; workgroups launched; workgroups that do work; workgroups per (batch, head) (pairs of query
 * tiles where fa_fwd_plan says so).  No counterpart in the reference (see fa_fwd_plan).
 */
int fa_fwd_variant(int64_t B, int64_t R, int64_t L, int64_t H, int flags, int has_mask, int* variant);

/*
 * 1 if fa_fwd accepts this head_dim, else 0.  Counterpart of the compile-time
 * (head_dim, chunk_size) dispatch table (reference src/fused_attn_extention.cu:72-111).
 */
int fa_fwd_query(int64_t H);

/*
 * The power of two (as a base-2 exponent) the softmax weights of a row of L keys are divided by
 * before they are rounded to fp16 for the second product (bf16 weights: 2^14 at every length): a key at the running maximum of its
 * row gets the weight 2^-bias.  11 - ceil(log2 L), kept inside [-8, 6]: see "Accuracy" under fa_fwd.
 * Exported so that callers and tests can state the accuracy limit of a launch; no counterpart in the
 * reference, which keeps every intermediate in fp16 (reference include/fused_attn.cuh:174,257,650-653).
 */
float fa_fwd_reference_bias(int64_t L);

/*
 * Human-readable text for a status returned by fa_fwd.  Replaces the print-and-exit
 * macros CHECK_CUDA_ERROR / CHECK_LAST_CUDA_ERROR (reference include/fused_attn.cuh:17-42).
 * The returned pointer is static storage.
 */
const char* fa_strerror(int status);

/*
 * Timed replay for benchmarks: launches fa_fwd `iters` times back to back on `stream`,
 * bracketed by HIP events recorded on that same stream, waits, and writes the average
 * milliseconds per launch to *ms_per_launch.  Counterpart of the timing loop in
 * reference tests/benchmark_fused_attn.py:36-42 (wall clock around 128 launches).
 */
int fa_fwd_timed(const void* q, const void* k, const void* v, const void* mask, void* out,
                 int64_t B, int64_t R, int64_t L, int64_t H,
                 int64_t stride_b, int64_t stride_h, int64_t stride_l,
                 float scale, void* stream, int iters, float* ms_per_launch);

/*
 * fa_fwd_timed for every form of the launch: the arguments of fa_fwd_strided (flags, lse, strides
 * of `out`) followed by those of the timing loop.  The same counterpart in the reference
 * (tests/benchmark_fused_attn.py:36-42); fa_fwd_timed is this with lse = NULL, flags = 0 and the
 * strides of q for out.
 */
int fa_fwd_timed_ex(const void* q, const void* k, const void* v, const void* mask, void* out, void* lse,
                    int64_t B, int64_t R, int64_t L, int64_t H,
                    int64_t stride_b, int64_t stride_h, int64_t stride_l,
                    int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_l,
                    float scale, int flags, void* stream, int iters, float* ms_per_launch);

/*
 * Fused QKV projection, the front end the reference lists as not done (reference README.md:137;
 * its kernel takes queries, keys and values as three separate tensors, reference
 * src/fused_attn_extention.cu:15-22):
 *     qkv[b, l, s, :] = x[b, l, :] w[:, s F : (s + 1) F] (+ bias[s F : (s + 1) F]),   s = 0, 1, 2,  F = R H
 * x is [B, L, F_in], w is [F_in, 3 F] (input features along the rows), bias (nullable) is [3 F], qkv
 * is the packed [B, L, 3, F] tensor, all contiguous, fp16 (bfloat16 with FA_FLAG_BF16), f32
 * accumulation, one rounding.  The three slices qkv[:, :, s, :] are what fa_fwd_strided takes as q,
 * k and v (stride_b = 3 L F, stride_h = H, stride_l = 3 F) without a copy.
 * rope_cos / rope_sin (both or neither; nullable): float32 [L, H / 2] tables of a rotary position
 * encoding in the rotate-half form, applied to every head of the q and k slices before the rounding:
 *     out[i] = y[i] cos[l, i] - y[i + H/2] sin[l, i],  out[i + H/2] = y[i + H/2] cos[l, i] + y[i] sin[l, i]
 * for i < H / 2, y the projected head vector.
 * F_in and F must be multiples of 64 (FA_ERR_BAD_SHAPE otherwise); x, w, qkv and the tables 16-byte
 * aligned, bias 8-byte aligned.  Launches on `stream` and returns without synchronising.
 */
int fa_qkv_proj(const void* x, const void* w, const void* bias, void* qkv,
                int64_t B, int64_t L, int64_t F_in, int64_t R, int64_t H,
                const float* rope_cos, const float* rope_sin, int flags, void* stream);

/*
 * The launch of the 256 x 256 tile kernel for a problem, without making it (no GPU is touched): for
 * tests of the launcher.  Fills plan[0..3] with: workgroups launched; workgroups that do work (a
 * resident grid: workgroup w of them takes the tiles w, w + working, ...); output tiles of 256 x 256
 * (row tiles times feature tiles); feature tiles.  No counterpart in the reference (see fa_qkv_proj).
 */
int fa_qkv_proj_plan(int64_t B, int64_t L, int64_t F_in, int64_t R, int64_t H, int* plan);

/*
 * The kernel fa_qkv_proj picks for a problem (rope != 0: with tables), without launching it.  Fills variant[0..5] with: rows and
 * features of a workgroup's tile (256 x 256: the launch fa_qkv_proj_plan describes; smaller ones: one tile
 * per workgroup); workgroups launched; workgroups that do work; output tiles; feature tiles.
 */
int fa_qkv_proj_variant(int64_t B, int64_t L, int64_t F_in, int64_t R, int64_t H, int rope, int* variant);

/*
 * A paged cache of keys and values in 8 bits, and the sequences of a call.  No counterpart in the reference, whose keys and
 * values are the call's own (reference src/fused_attn_extention.cu:15-22): what a program needs that answers token by token.
 *
 *   keys, values     [pages, heads, page_size, head_dim], one e4m3 code (OCP FP8: torch.float8_e4m3fn) per value
 *   key_exponents, value_exponents
 *                    int8 [pages, heads]: a code c of the page and head stands for c * 2^exponent
 *   key_bounds       (nullable) int8 [pages, heads, 2, head_dim]: the largest and the smallest key of each channel of the page, as
 *                    appended (rotated, before the rounding to e4m3), in steps of 2^(key exponent + 2), rounded upwards and
 *                    downwards; what fa_select_pages reads
 *   page_table       int32 [sequences, table_width], rows table_stride elements apart: the page of the tokens
 *                    w * page_size .. (w + 1) * page_size - 1 of a sequence; a number outside [0, pages) is no page
 *
 * page_size is 16, 32, 64 or 128 (FA_ERR_BAD_PAGE otherwise), head_dim 16, 32, 64 or 128.  All tensors but the table are
 * contiguous; keys, values and key_bounds 16-byte aligned.  pages * heads * page_size / 16 and
 * table_width * page_size must stay below 2^31 - 2^16.
 *
 * A call brings L tokens for each sequence, of which the first new_lens[b] exist (new_lens NULL: all; numbers outside
 * [0, L] count as the nearer end); token i of sequence b has the position starts[b] + i, starts[b] being the number of tokens
 * in the cache before it.  Positions are below table_width * page_size: what lies behind is not written and not read.  starts
 * and new_lens are int32 [sequences] in device memory.  The library cannot look at numbers in device memory before it
 * launches; its kernels check every page and every position against the sizes given here, so that wrong ones cost
 * results, never an access out of bounds.
 */
typedef struct fa_cache {
    void* keys;
    void* values;
    void* key_exponents;
    void* value_exponents;
    void* key_bounds;
    const int32_t* page_table;
    int64_t pages, heads, page_size, head_dim;
    int64_t sequences, table_width, table_stride;
} fa_cache;

/*
 * Appends L new tokens per sequence.  k and v (fp16, or bfloat16 with FA_FLAG_BF16) share (kv_stride_b, kv_stride_h,
 * kv_stride_l) under the addressing rule above, with cache->heads heads.
 *   y = k rotated by its position (rotate-half as in fa_qkv_proj, in float32, each product and each sum rounded by itself), where
 *       rope_cos / rope_sin (both or neither) are float32 [rope_rows, head_dim / 2] tables, indexed by position; v is kept
 *   e = the smallest exponent, not below -80, with |y| <= 448 * 2^e for all new tokens of the page and head; where the page
 *       holds earlier tokens of the sequence (its first new token is not in its first place), not below their exponent
 *   code = e4m3(y * 2^-e), to nearest even; codes of earlier tokens move to e in the same way (without rounding unless they
 *       become subnormal)
 * and key_bounds, where the cache has them, follow; they do not depend on the parts in which tokens were appended.  Values that
 * are not finite become NaN codes and count as zero in the exponent and the bounds.  Tokens at positions from
 * rope_rows on are not appended; places of a page behind the last token keep their codes, pages that get no token everything.
 * A page that a call writes must belong to one sequence and stand once in its table.
 * q (nullable, strides q_stride_*, R heads) is rotated likewise into q_out (strides out_stride_*, not overlapping q),
 * rounded once; rows of tokens that do not exist, or from rope_rows on, become zeros.  R is not looked at without q.
 * What is written (q_out here, out below) has a place of its own for every row: of its dimensions with more than one element, in
 * the order of their strides, each steps over all the rows that those before it place (FA_ERR_BAD_STRIDE otherwise; strides of 0 and
 * rows that overlap are for k, v and q only).
 */
int fa_cache_append(const fa_cache* cache, const void* k, const void* v, int64_t kv_stride_b, int64_t kv_stride_h, int64_t kv_stride_l,
                    const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l,
                    void* q_out, int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_l,
                    const int32_t* starts, const int32_t* new_lens, int64_t L, int64_t R,
                    const float* rope_cos, const float* rope_sin, int64_t rope_rows, int flags, void* stream);

/*
 * out = softmax(q k^T * scale) v over the cached tokens of each sequence, for L tokens of R query heads; R is a multiple of
 * cache->heads, query head h reads key head h / (R / heads).  Token i of sequence b sees the first starts[b] + i + 1 tokens
 * with FA_FLAG_CAUSAL (the new ones are in the cache already: fa_cache_append goes first), all starts[b] + new_lens[b]
 * without, of those on a page; and, where `selected` (nullable) is given, int32 [sequences, L, heads, count], only those on
 * the pages of its sequence that its list names by their places in the page table, each once however often it is named;
 * numbers outside [0, table_width) name nothing.  count is at most 4096 (FA_ERR_TOO_LARGE), and not looked at without a list.
 * Rows that see nothing, and those of tokens that do not exist, are zeros with an lse of -inf.  lse (nullable) as in fa_fwd_ex.
 * q and out as in fa_fwd_strided, fp16 or bfloat16 (FA_FLAG_BF16), whatever type the cache was filled from.
 * Accuracy: codes enter both products as they are; scores, sums and outputs are float32; softmax weights are rounded to the
 * type of q.  fp16 weights keep 11 bits down to 2^-21 of the row's largest, and values 4 bits down to 2^-15 of the largest
 * power of two among the pages that a wave reads: pages without weight in the row are among them, and those that only
 * rows beside it see.  With bfloat16 such a page costs no more than 2^-117 of its power of two.  scale * log2(e) has to be finite in
 * float32 (FA_ERR_BAD_SCALE), and times the power of two of a page's keys as well: scores of pages beyond that may become NaN.
 * A value that is not a number reaches the rows that see it only.
 * workspace: fa_cached_attention_workspace bytes of device memory, 16-byte aligned (FA_ERR_WORKSPACE if it is too small;
 * nullable where that is 0), not used by another call at the same time; nothing in it is kept between calls.
 * The launch is chosen from the sizes: for sequences about as long as table_width allows.  Much wider tables cost time, not results.
 */
int fa_cached_attention(const fa_cache* cache, const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l,
                        void* out, int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_l, void* lse,
                        const int32_t* selected, int64_t count, const int32_t* starts, const int32_t* new_lens,
                        int64_t L, int64_t R, float scale, int flags, void* workspace, int64_t workspace_bytes, void* stream);

/* Bytes of workspace that fa_cached_attention needs for these sizes (count = 0: no list), or a negative status.  Only the sizes
 * in `cache` are looked at; no GPU is touched. */
int64_t fa_cached_attention_workspace(const fa_cache* cache, int64_t L, int64_t R, int64_t count);

/*
 * The pages that each new token's query heads attend to: for every token and key head `count` places of the page table in
 * ascending order into `selected`, int32 [sequences, L, heads, count], -1 behind the last where there are fewer.  Candidates are
 * the pages up to the one of the token itself, which is always taken; of the others those with the largest
 *   2^(key exponent) * max over the key head's query heads of  sum_d max(q8_d, 0) * largest_d + min(q8_d, 0) * smallest_d
 * where q8 = round(q * 2^-e) with the smallest e that keeps the group's queries within 127 (not finite: 0), and largest and
 * smallest are the cache's key_bounds: 2^-(e + 2) times an upper bound of what the page's keys score with q8 * 2^e as they were
 * appended.  What the cache holds of them may score more by the rounding to e4m3: in each channel a code may lie outside its bounds by a
 * sixteenth of the key (of small keys, 2^-9 of the page's power of two).  Whole numbers throughout; equal scores go to the lowest place.  Tokens that do not exist get -1 only.
 * q as above, rotated already.  cache->keys, values and value_exponents are not looked at.  table_width is at most 32768 and
 * count at most 4096 (FA_ERR_TOO_LARGE).  Needs no workspace.
 */
int fa_select_pages(const fa_cache* cache, const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l,
                    int32_t* selected, int64_t count, const int32_t* starts, const int32_t* new_lens,
                    int64_t L, int64_t R, int flags, void* stream);

/*
 * The launches that fa_cached_attention and fa_select_pages would make for these sizes, without making them (no GPU is touched; only
 * the sizes in `cache` are looked at): for tests of the launcher and for tuning.  fa_cached_attention_plan fills
 * plan[0..4] with: 0 = the kernel for few rows, 1 = the one for many, 2 = that for few with the lists of several tokens joined;
 * waves per workgroup; query rows per workgroup; parts that a row's keys are cut into; workgroups.  fa_select_pages_plan fills plan[0..2] with: tokens per workgroup; waves per
 * workgroup; workgroups.
 */
int fa_cached_attention_plan(const fa_cache* cache, int64_t L, int64_t R, int64_t count, int* plan);
int fa_select_pages_plan(const fa_cache* cache, int64_t L, int64_t R, int* plan);

/*
 * Tables of a rotary position encoding, scaled for contexts longer than a model was made for: float32 [rows, dims / 2],
 *     cos[p, j] = amplitude * cos(p f'_j),   sin[p, j] = amplitude * sin(p f'_j),   f_j = base^(-2 j / dims)
 * in 64 bits, rounded once.  No counterpart in the reference, whose queries and keys come as they are
 * (reference src/fused_attn_extention.cu:15-22).  scaling:
 *   FA_ROTARY_NONE    f' = f
 *   FA_ROTARY_LINEAR  f' = f / factor
 *   FA_ROTARY_BASE    f' = (base * factor^(dims / (dims - 2)))^(-2 j / dims)
 *   FA_ROTARY_TURNS   f' = f * (g + (1 - g) / factor) with t = original_rows * f / (2 pi), the turns of the column over the original
 *                     context, and g = (t - low) / (high - low) within [0, 1]
 *   FA_ROTARY_INDEX   the same with g = 1 - (j - a) / max(b - a, 0.001) within [0, 1], where
 *                     i(t) = dims * ln(original_rows / (2 pi t)) / (2 ln base), a = max(floor(i(high)), 0), b = min(ceil(i(low)), dims - 1)
 * base > 1; factor, original_rows, low < high and amplitude positive, where they are looked at, all finite (FA_ERR_BAD_SCALE).  dims is a
 * multiple of 16 (FA_ERR_BAD_SHAPE) of at most 256 (FA_ERR_TOO_LARGE).  cos and sin 16-byte aligned.
 */
#define FA_ROTARY_NONE 0
#define FA_ROTARY_LINEAR 1
#define FA_ROTARY_BASE 2
#define FA_ROTARY_TURNS 3
#define FA_ROTARY_INDEX 4
typedef struct fa_rotary {
    int scaling;
    double base, factor, original_rows, low, high, amplitude;
} fa_rotary;

int fa_rotary_tables(float* cos, float* sin, int64_t rows, int64_t dims, const fa_rotary* how, void* stream);

/*
 * Rotates queries, and keys (nullable, with k_out) beside them, by the positions of their tokens.  q has R heads and k has Rkv, of H
 * channels (a multiple of 16 up to 1024), each with strides of its own under the addressing rule above, as have q_out and k_out.  The
 * channels first .. first + dims of a head are rotated, the others copied; dims a multiple of 16, first of 8.  Pairs are the channels
 * first + j and first + dims / 2 + j, or first + 2 j and first + 2 j + 1 with FA_FLAG_INTERLEAVED (j < dims / 2):
 *     (a, b) -> (a cos - b sin, b cos + a sin)     with -sin for sin under FA_FLAG_INVERSE, which is also what a gradient needs
 * each product and each sum rounded to float32, the result to 16 bits.  cos / sin: float32 [rope_rows, dims / 2], 16-byte aligned.
 * Token i of sequence b has the position positions[b, i] (int32 [B, L], nullable) or starts[b] + i (int32 [B], nullable: zeros; not both:
 * FA_ERR_BAD_SHAPE).  Rows of tokens behind new_lens[b] (int32 [B], nullable), or whose position is outside [0, rope_rows), become
 * zeros.  out may be its input with the same strides; otherwise the two must not overlap, nor may q_out and k_out, or one's output and the
 * other's input (FA_ERR_BAD_STRIDE where both have the same strides, as views of one tensor, or the first row of either meets the other).
 */
int fa_rotate(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, void* q_out, int64_t q_out_stride_b,
              int64_t q_out_stride_h, int64_t q_out_stride_l, const void* k, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_l,
              void* k_out, int64_t k_out_stride_b, int64_t k_out_stride_h, int64_t k_out_stride_l, int64_t B, int64_t L, int64_t R,
              int64_t Rkv, int64_t H, int64_t first, int64_t dims, const float* cos, const float* sin, int64_t rope_rows,
              const int32_t* positions, const int32_t* starts, const int32_t* new_lens, int flags, void* stream);

/*
 * Keeping the pages of a cache, the 8-bit one above or the one of latents below: all in device memory, so that a step never waits for
 * the host.  No counterpart in the reference, which has no cache.
 *
 *   page_table  int32 [sequences, table_width], rows table_stride elements apart; a number outside [0, pages) is no page
 *   starts      int32 [sequences]: tokens in the cache (not looked at by fa_copy_pages and fa_compact_pages)
 *   uses        int32 [pages]: how many entries of the table name the page; a page without uses is free
 *   data        `tensors` (up to 8) tensors of `pages` pages of page_bytes each, one behind the other: what a page holds
 *               (looked at by fa_copy_pages, fa_fork_pages and fa_compact_pages)
 * Where one table keeps more tensors than a call takes, those of a model's other layers, fa_fork_pages and fa_compact_pages are called once all the
 * same, for each of them changes the table and the uses: the other tensors' pages are then copied by fa_copy_pages, from every page to where `moved`
 * says, and from the page that a forked parent's tokens end in, where they do not fill it, to the one at the same place of its child's row.
 *
 * Lists are int32 in device memory; numbers in them that are no sequence, or no page, are passed over.  A count of 0 does nothing.
 * Of a page's bytes 16 are moved at a time where the tensor is aligned to 16 and page_bytes is a multiple of it; otherwise 4, or 1.
 */
typedef struct fa_pages {
    int32_t* page_table;
    int32_t* starts;
    int32_t* uses;
    int64_t pages, page_size, sequences, table_width, table_stride;
    int64_t tensors;
    void* data[8];
    int64_t page_bytes[8];
} fa_pages;

/* Page sources[n] into page targets[n] in all tensors, n < count.  A target is named once and is no source of another pair: what it
 * holds otherwise is any mixture of the sources. */
int fa_copy_pages(const fa_pages* pages, const int32_t* sources, const int32_t* targets, int64_t count, void* stream);

/* The listed sequences end: every page of their rows loses a use, the rows become -1 and their starts 0.  Up to 65536 of them; one that
 * is named twice ends once. */
int fa_free_pages(const fa_pages* pages, const int32_t* sequences, int64_t count, void* stream);

/*
 * Pages for new tokens: sequence b brings new_lens[b] of them (nullable: L; within [0, L]), behind starts[b].  The places
 * ceil(starts[b] / page_size) .. ceil((starts[b] + new_lens[b]) / page_size) of its row that name no page get the lowest free ones, in the
 * order of the rows and places, and a use each.  missing, int32 [sequences], receives how many places found no page or lie behind
 * the table; starts are left to the caller.  The table has fewer than 2^31 - 2^16 places, sequences * table_width (FA_ERR_TOO_LARGE).
 * workspace: fa_take_pages_workspace bytes, 16-byte aligned, of no other call at the same time.
 */
int fa_take_pages(const fa_pages* pages, const int32_t* new_lens, int64_t L, int32_t* missing, void* workspace, int64_t workspace_bytes,
                  void* stream);
int64_t fa_take_pages_workspace(const fa_pages* pages);

/*
 * Sequence children[n] continues sequence parents[n]: its row names the parent's full pages, which gain a use each, and where the
 * parent's last page is not full the child gets a copy of it in the lowest free page (those of smaller n first).  Its starts
 * become the parent's.  forked, int32 [count], receives 1; 0, and nothing else happens, where one of the two is no sequence, both are the same,
 * the child has tokens, smaller n name the child as well, or no page is free for the copy.  All parents are as before the call.  Pages that
 * an empty child's row names lose a use, also where the parent has no tokens and the row becomes -1.  count is at most 4096
 * (FA_ERR_TOO_LARGE).  workspace as above.
 */
int fa_fork_pages(const fa_pages* pages, const int32_t* parents, const int32_t* children, int64_t count, int32_t* forked, void* workspace,
                  int64_t workspace_bytes, void* stream);
int64_t fa_fork_pages_workspace(int64_t count);

/*
 * Moves the used pages together: of U used pages, those at U and above move, in ascending order, to the free places below U in
 * ascending order, with their uses, and the table follows (entries that name a free page become -1).  moved, int32 [pages], receives
 * where each used page is now, and -1 for the others.  workspace as above.
 */
int fa_compact_pages(const fa_pages* pages, int32_t* moved, void* workspace, int64_t workspace_bytes, void* stream);
int64_t fa_compact_pages_workspace(const fa_pages* pages);

/*
 * A paged cache of latents: for each token one vector of latent_dim channels that all heads share as key and as value, and one rotary
 * key of rope_dim channels, latents [pages, page_size, latent_dim + rope_dim], contiguous, 16-byte aligned, fp16 or bfloat16
 * (FA_FLAG_BF16).  page_table as in fa_cache.  latent_dim 128, 256 or 512, rope_dim 32 or 64 (FA_ERR_BAD_HEAD_DIM); page_size 16, 32, 64 or
 * 128.  L, starts and new_lens as with fa_cache; positions are below table_width * page_size.  No counterpart in the reference.
 */
typedef struct fa_latent_cache {
    void* latents;
    const int32_t* page_table;
    int64_t pages, page_size, latent_dim, rope_dim;
    int64_t sequences, table_width, table_stride;
} fa_latent_cache;

/*
 * Appends L new tokens per sequence: latents c [sequences, L, latent_dim] as they are, rotary keys k [sequences, L, rope_dim] rotated by
 * their positions as fa_rotate does (tables [rope_rows, rope_dim / 2], both or neither; FA_FLAG_INTERLEAVED).  q (nullable: the rotary
 * channels of R query heads, [sequences, L, R, rope_dim] by q_stride_b, _h, _l) is rotated likewise into q_out; rows of tokens that do not
 * exist, or from rope_rows on, become zeros.  Nothing else of the cache is written.  A page that a call writes must belong to one sequence and
 * stand once in its table.  c, k, q and q_out have 16-byte aligned addresses and strides that are multiples of 8 elements.
 */
int fa_latent_append(const fa_latent_cache* cache, const void* c, int64_t c_stride_b, int64_t c_stride_l, const void* k, int64_t k_stride_b,
                     int64_t k_stride_l, const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, void* q_out,
                     int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_l, const int32_t* starts, const int32_t* new_lens, int64_t L,
                     int64_t R, const float* rope_cos, const float* rope_sin, int64_t rope_rows, int flags, void* stream);

/*
 * Attention in the absorbed form: for each token and query head, with its queries q (latent_dim, the head's map of latents to keys
 * multiplied in) and r (rope_dim, rotated),
 *     s_j = scale * (q . c_j + r . k_j),   out = sum_j softmax(s)_j c_j   (latent_dim; the head's map to values is the caller's)
 * over the cached tokens that fa_cached_attention would see: starts[b] + i + 1 with FA_FLAG_CAUSAL, otherwise starts[b] + new_lens[b], of
 * those on a page.  q, r and out [sequences, L, R, .] by strides of their own.  Rows that see nothing, and those of tokens that do not
 * exist, are zeros with an lse of -inf.  lse (nullable): float32 [sequences, R, L].  Scores and sums are float32; weights,
 * and the outputs, are rounded to the cache's type once.
 * fp16 weights keep 11 bits down to 2^-22 of the row's largest and lose what is below 2^-32.  A latent or rotary key that is not finite makes rows
 * that see it NaN where the formula does, or wholly; others never meet it.
 * workspace: fa_latent_attention_workspace bytes, 16-byte aligned, of no other call at the same time (nullable where that is 0).  The launch is
 * chosen from the sizes: for sequences about as long as table_width allows.
 */
int fa_latent_attention(const fa_latent_cache* cache, const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_l, const void* r,
                        int64_t r_stride_b, int64_t r_stride_h, int64_t r_stride_l, void* out, int64_t out_stride_b, int64_t out_stride_h,
                        int64_t out_stride_l, void* lse, const int32_t* starts, const int32_t* new_lens, int64_t L, int64_t R, float scale,
                        int flags, void* workspace, int64_t workspace_bytes, void* stream);
int64_t fa_latent_attention_workspace(const fa_latent_cache* cache, int64_t L, int64_t R);

/*
 * Attention in the expanded form, for prompts: every head h has keys k and values v of its own, and all heads share the rotary keys,
 *     s_j = scale * (q[: key_dim] . k_hj + q[key_dim :] . rope_k_j),   out = sum_j softmax(s)_j v_hj
 * q [sequences, tokens, heads, key_dim + rope_dim], k [sequences, keys, heads, key_dim], rope_k [sequences, keys, rope_dim], v [sequences, keys,
 * heads, value_dim], out [sequences, tokens, heads, value_dim] by strides {b, h, l} (rope_k: {b, l}) in elements, multiples of 8, those of the
 * keys' dimension at most 2^24; fp16 or bfloat16.  key_dim = value_dim is 64 or 128, rope_dim 32 or 64 (FA_ERR_BAD_HEAD_DIM).  Token i of sequence b
 * sees the first starts[b] + i + 1 keys with FA_FLAG_CAUSAL and starts[b] + new_lens[b] otherwise, of those there are (starts, int32
 * [sequences], nullable: keys - tokens; new_lens nullable: tokens).  Rows, lse, workspace and accuracy as with fa_latent_attention; a value that is not finite
 * makes rows that see it NaN or infinite in its channel, others never meet it.
 */
typedef struct fa_expanded {
    const void* q;
    const void* k;
    const void* rope_k;
    const void* v;
    void* out;
    void* lse;
    const int32_t* starts;
    const int32_t* new_lens;
    int64_t sequences, tokens, heads, keys, key_dim, rope_dim, value_dim;
    int64_t q_strides[3], k_strides[3], rope_k_strides[2], v_strides[3], out_strides[3];
} fa_expanded;

int fa_expanded_attention(const fa_expanded* x, float scale, int flags, void* workspace, int64_t workspace_bytes, void* stream);
int64_t fa_expanded_attention_workspace(const fa_expanded* x);

/*
 * The launches of the two for these sizes, without making them (no GPU is touched, only sizes are looked at): plan[0..2] = query rows per
 * workgroup; for fa_latent_attention 1 where the workgroups share out the keys of all rows and 0 where each has rows to itself, for
 * fa_expanded_attention the parts that a row's keys are cut into; workgroups.
 */
int fa_latent_attention_plan(const fa_latent_cache* cache, int64_t L, int64_t R, int* plan);
int fa_expanded_attention_plan(const fa_expanded* x, int* plan);

#ifdef __cplusplus
}
#endif

#endif /* FUSED_ATTN_H_ */
