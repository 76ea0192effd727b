// C ABI of the page keeping (include/fused_attn.h): argument validation and the launches.
#include "host_checks.hpp"
#include "page_kernels.hpp"

namespace {

using namespace fa::pages;

// Sequences of a list: both look through what stands before each, and the plan of a fork does so in one workgroup.
constexpr int64_t kMostFreed = 65536, kMostForked = 4096;

// The page table, the lengths and the uses.
int check_keeping(const fa_pages* c, bool lengths, View* v) {
    if (c == nullptr) return FA_ERR_NULL_POINTER;
    int log2_p = 4;
    while (log2_p < 7 && ((int64_t)1 << log2_p) < c->page_size) ++log2_p;
    if (lengths && c->page_size != (int64_t)1 << log2_p) return FA_ERR_BAD_PAGE;
    if (c->pages < 1 || c->sequences < 1 || c->table_width < 1) return FA_ERR_BAD_SHAPE;
    if (c->table_stride < 0 || (c->table_stride < c->table_width && c->sequences > 1)) return FA_ERR_BAD_STRIDE;
    if (c->pages > kMaxInt || c->sequences > kMaxInt || c->table_width > kMaxInt / 128 || !below(c->table_stride, c->sequences, kMaxElems))
        return FA_ERR_TOO_LARGE;
    if (c->page_table == nullptr || c->uses == nullptr || (lengths && c->starts == nullptr)) return FA_ERR_NULL_POINTER;
    if (!aligned(c->page_table, 4) || !aligned(c->uses, 4) || !aligned(c->starts, 4)) return FA_ERR_MISALIGNED;
    v->table = c->page_table;
    v->table_stride = c->table_stride;
    v->starts = c->starts;
    v->uses = c->uses;
    v->N = (int)c->pages;
    v->S = (int)c->sequences;
    v->W = (int)c->table_width;
    v->log2_p = log2_p;
    return FA_OK;
}

// The tensors whose pages are copied.
int check_tensors(const fa_pages* c, Tensors* t) {
    if (c == nullptr) return FA_ERR_NULL_POINTER;
    if (c->pages < 1 || c->tensors < 1) return FA_ERR_BAD_SHAPE;
    if (c->tensors > kMostTensors || c->pages > kMaxInt) return FA_ERR_TOO_LARGE;
    t->count = (int)c->tensors;
    int64_t chunks = 0;
    for (int n = 0; n < t->count; ++n) {
        const int64_t bytes = c->page_bytes[n];
        if (c->data[n] == nullptr) return FA_ERR_NULL_POINTER;
        if (bytes < 1) return FA_ERR_BAD_SHAPE;
        if (!below(bytes, c->pages, kMaxElems) || bytes > (int64_t)1 << 40) return FA_ERR_TOO_LARGE;
        t->data[n] = static_cast<uint8_t*>(c->data[n]);
        t->page_bytes[n] = bytes;
        t->unit[n] = aligned(c->data[n], 16) && bytes % 16 == 0 ? 16 : aligned(c->data[n], 4) && bytes % 4 == 0 ? 4 : 1;
        t->first_chunk[n] = (int)chunks;
        chunks += ceil_div(bytes / t->unit[n], kChunk);
        if (chunks > 0x3fffffff) return FA_ERR_TOO_LARGE;
    }
    t->first_chunk[t->count] = (int)chunks;
    return FA_OK;
}

int check_list(const int32_t* list, int64_t count) {
    if (list == nullptr) return FA_ERR_NULL_POINTER;
    if (!aligned(list, 4)) return FA_ERR_MISALIGNED;
    return count < 0 ? FA_ERR_BAD_SHAPE : FA_OK;
}

// Workgroups that share out the chunks of what is copied: eight to a compute unit.
constexpr int64_t kCopyWgs = 8 * kNumCu;

}  // namespace

extern "C" {

int fa_copy_pages(const fa_pages* c, const int32_t* sources, const int32_t* targets, int64_t count, void* stream) {
    CopyParams p;
    int rc = check_tensors(c, &p.tensors);
    if (rc == FA_OK) rc = check_list(sources, count);
    if (rc == FA_OK) rc = check_list(targets, count);
    if (rc != FA_OK) return rc;
    if (count > kMaxInt) return FA_ERR_TOO_LARGE;
    if (count == 0) return FA_OK;
    p.sources = sources;
    p.targets = targets;
    p.count = (int)count;
    p.N = (int)c->pages;
    const int64_t chunks = p.tensors.first_chunk[p.tensors.count];
    p.by_chunks = fa::divisor(chunks);
    const int64_t wgs = below(chunks, count, kCopyWgs) ? chunks * count : kCopyWgs;
    return static_cast<int>(launch(copy_pages_kernel, wgs, 256, p, 0, static_cast<hipStream_t>(stream)));
}

int fa_free_pages(const fa_pages* c, const int32_t* sequences, int64_t count, void* stream) {
    FreeParams p;
    int rc = check_keeping(c, true, &p);
    if (rc == FA_OK) rc = check_list(sequences, count);
    if (rc != FA_OK) return rc;
    if (count > kMostFreed) return FA_ERR_TOO_LARGE;
    if (count == 0) return FA_OK;
    p.sequences = sequences;
    p.count = (int)count;
    return static_cast<int>(launch(free_pages_kernel, count, 256, p, 0, static_cast<hipStream_t>(stream)));
}

int64_t fa_take_pages_workspace(const fa_pages* c) {
    if (c == nullptr) return FA_ERR_NULL_POINTER;
    if (c->pages < 1) return FA_ERR_BAD_SHAPE;
    return c->pages > kMaxInt ? (int64_t)FA_ERR_TOO_LARGE : 4 * c->pages;
}

int fa_take_pages(const fa_pages* c, const int32_t* new_lens, int64_t L, int32_t* missing, void* workspace, int64_t workspace_bytes, void* stream) {
    TakeParams p;
    const int rc = check_keeping(c, true, &p);
    if (rc != FA_OK) return rc;
    if (L < 1) return FA_ERR_BAD_SHAPE;
    // the places of the whole table are counted in 32 bits: what every row wants, and the rank of each among all
    if (L > kMaxInt || !below(c->sequences, c->table_width, kMaxInt)) return FA_ERR_TOO_LARGE;
    if (missing == nullptr) return FA_ERR_NULL_POINTER;
    if (!aligned(missing, 4) || !aligned(new_lens, 4)) return FA_ERR_MISALIGNED;
    if (workspace == nullptr || workspace_bytes < fa_take_pages_workspace(c)) return FA_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return FA_ERR_MISALIGNED;
    p.new_lens = new_lens;
    p.L = (int)L;
    p.missing = missing;
    p.list = static_cast<int32_t*>(workspace);
    return static_cast<int>(launch(take_pages_kernel, 1, kPlanThreads, p, 0, static_cast<hipStream_t>(stream)));
}

int64_t fa_fork_pages_workspace(int64_t count) {
    if (count < 0) return FA_ERR_BAD_SHAPE;
    return count > kMostForked ? (int64_t)FA_ERR_TOO_LARGE : 3 * 4 * count;
}

int fa_fork_pages(const fa_pages* c, const int32_t* parents, const int32_t* children, int64_t count, int32_t* forked, void* workspace,
                  int64_t workspace_bytes, void* stream) {
    ForkParams p;
    int rc = check_keeping(c, true, &p);
    if (rc == FA_OK) rc = check_tensors(c, &p.tensors);
    if (rc == FA_OK) rc = check_list(parents, count);
    if (rc == FA_OK) rc = check_list(children, count);
    if (rc == FA_OK) rc = check_list(forked, count);
    if (rc != FA_OK) return rc;
    if (count > kMostForked) return FA_ERR_TOO_LARGE;
    if (count == 0) return FA_OK;
    if (workspace == nullptr || workspace_bytes < fa_fork_pages_workspace(count)) return FA_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return FA_ERR_MISALIGNED;
    const int64_t per = 1 + (int64_t)p.tensors.first_chunk[p.tensors.count];
    if (!below(per, count, kMostThreads / 256)) return FA_ERR_TOO_LARGE;
    p.parents = parents;
    p.children = children;
    p.count = (int)count;
    p.forked = forked;
    p.lengths = static_cast<int32_t*>(workspace);
    p.copies = p.lengths + count;
    p.list = p.copies + count;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = launch(plan_fork_kernel, 1, kPlanThreads, p, 0, s);
    if (e != hipSuccess) return static_cast<int>(e);
    return static_cast<int>(launch(fork_pages_kernel, per * count, 256, p, 0, s));
}

int64_t fa_compact_pages_workspace(const fa_pages* c) {
    const int64_t n = fa_take_pages_workspace(c);
    return n < 0 ? n : n + 16;
}

int fa_compact_pages(const fa_pages* c, int32_t* moved, void* workspace, int64_t workspace_bytes, void* stream) {
    CompactParams p;
    int rc = check_keeping(c, false, &p);
    if (rc == FA_OK) rc = check_tensors(c, &p.tensors);
    if (rc == FA_OK) rc = check_list(moved, 0);
    if (rc != FA_OK) return rc;
    if (workspace == nullptr || workspace_bytes < fa_compact_pages_workspace(c)) return FA_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return FA_ERR_MISALIGNED;
    p.moved = moved;
    p.count = static_cast<int32_t*>(workspace);
    p.holes = p.count + 4;
    p.movers = p.holes + c->pages / 2;
    const int64_t chunks = p.tensors.first_chunk[p.tensors.count];
    p.by_chunks = fa::divisor(chunks);
    p.by_width = fa::divisor(p.W);
    const int64_t most = c->pages / 2;                   // pages that can move
    p.copy_wgs = (int)(below(chunks, most > 0 ? most : 1, kCopyWgs) ? chunks * (most > 0 ? most : 1) : kCopyWgs);
    const int64_t entries = ceil_div(c->sequences * c->table_width, 256);
    p.table_wgs = (int)(entries < kNumCu ? entries : kNumCu);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = launch(plan_compact_kernel, 1, kPlanThreads, p, 0, s);
    if (e != hipSuccess) return static_cast<int>(e);
    return static_cast<int>(launch(compact_pages_kernel, p.copy_wgs + p.table_wgs, 256, p, 0, s));
}

}  // extern "C"
