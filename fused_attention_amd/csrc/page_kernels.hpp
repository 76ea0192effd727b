// Keeping the pages of a cache for gfx950 (MI355X, CDNA4): copying them, sharing them between sequences, freeing, dealing out and moving
// them together.  No counterpart in the reference, which has no cache.
//
// All that is kept is in device memory, so that no step waits for the host and every one can be captured in a graph: the page table,
// the sequences' lengths, and for every page its uses, the number of table entries that name it.  A page without uses is free.  What
// is dealt out is decided by place alone, the lowest free page to the first request, so that results do not depend on the order in which
// anything runs; counts are changed by whole-number atomics.
#pragma once

#include "cache_kernels.hpp"

namespace fa {
namespace pages {

constexpr int kMostTensors = 8;
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kFew = 2048;               // pages whose list stays in LDS
constexpr int kChunk = 256 * 4;          // units of a chunk of a page, four a thread

struct Tensors {
    uint8_t* data[kMostTensors];
    int64_t page_bytes[kMostTensors];
    int unit[kMostTensors];              // bytes of an access: 16, 4 or 1
    int first_chunk[kMostTensors + 1];   // of a page's chunks, over all tensors
    int count;
};

struct View {
    int32_t* table;                      // [S, W]
    int64_t table_stride;
    int32_t* starts;                     // [S]
    int32_t* uses;                       // [N]
    int N, S, W, log2_p;
    __device__ __forceinline__ bool is_page(int page) const { return (uint32_t)page < (uint32_t)N; }
};

template <typename T>
__device__ __forceinline__ void copy_units(uint8_t* to, const uint8_t* from, int64_t units, int64_t at) {
    T x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i * 256 < units) x[i] = reinterpret_cast<const T*>(from)[at + i * 256];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i * 256 < units) reinterpret_cast<T*>(to)[at + i * 256] = x[i];
}

// Chunk `chunk` of page `from` into page `to`, by 256 threads.
__device__ __forceinline__ void copy_chunk(const Tensors& t, int chunk, int from, int to) {
    int n = 0;
    while (n + 1 < t.count && chunk >= t.first_chunk[n + 1]) ++n;
    const int64_t bytes = t.page_bytes[n], at = (int64_t)(chunk - t.first_chunk[n]) * kChunk + threadIdx.x;
    uint8_t* const target = t.data[n] + to * bytes;
    const uint8_t* const source = t.data[n] + from * bytes;
    if (t.unit[n] == 16)
        copy_units<u32x4>(target, source, bytes / 16, at);
    else if (t.unit[n] == 4)
        copy_units<uint32_t>(target, source, bytes / 4, at);
    else
        copy_units<uint8_t>(target, source, bytes, at);
}

// How many threads before this one say yes, and how many in all, of a workgroup of kPlanThreads.
struct Ranks {
    int before, all;
};
// The sum of `n` over the threads before this one, and over all.  `room` has kPlanWaves numbers; the barrier before it is written again is
// this function's first.
__device__ __forceinline__ Ranks rank_of(int n, int* room) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sum = cache::wave_sums(n);
    __syncthreads();
    if (lane == 63) room[wave] = sum;
    __syncthreads();
    Ranks r = {sum - n, 0};
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        r.before += w < wave ? room[w] : 0;
        r.all += room[w];
    }
    return r;
}

// The lowest `wanted` free pages in ascending order into `list`, or as many as there are; their number.
__device__ __forceinline__ int find_free(const View& v, int wanted, int* list, int* room) {
    int found = 0;
    for (int base = 0; base < v.N && found < wanted; base += 4 * kPlanThreads) {
        const int at = base + 4 * threadIdx.x;
        int is[4], n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            is[i] = at + i < v.N && v.uses[at + i] <= 0;
            n += is[i];
        }
        const Ranks r = rank_of(n, room);
        int rank = found + r.before;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (is[i]) {
                if (rank < wanted) list[rank] = at + i;
                ++rank;
            }
        found += r.all;
    }
    __syncthreads();
    return found < wanted ? found : wanted;
}

struct CopyParams {
    Tensors tensors;
    const int32_t* sources;
    const int32_t* targets;
    int count, N;
    Divisor by_chunks;
};

// A workgroup a chunk of 16 KiB, or several of them.  Bound by the bytes; 32 pages of 132 KB, 8.4 MB, 6 us.
__global__ __launch_bounds__(256) void copy_pages_kernel(const CopyParams p) {
    const int chunks = p.tensors.first_chunk[p.tensors.count];
    const int64_t items = (int64_t)p.count * chunks;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int n = item < 0x7fffffff ? p.by_chunks.of((int)item) : (int)(item / chunks);
        const int from = p.sources[n], to = p.targets[n];
        if ((uint32_t)from >= (uint32_t)p.N || (uint32_t)to >= (uint32_t)p.N || from == to) continue;
        copy_chunk(p.tensors, (int)(item - (int64_t)n * chunks), from, to);
    }
}

struct FreeParams : View {
    const int32_t* sequences;
    int count;
};

// A workgroup a sequence; one that the list names again is done already.  A launch: 3 to 5 us.
__global__ __launch_bounds__(256) void free_pages_kernel(const FreeParams p) {
    const int n = blockIdx.x, row = p.sequences[n];
    if ((uint32_t)row >= (uint32_t)p.S) return;
    bool again = false;
    for (int m = threadIdx.x; m < n; m += 256) again = again || p.sequences[m] == row;
    if (__syncthreads_or(again)) return;
    int32_t* entries = p.table + row * p.table_stride;
    for (int w = threadIdx.x; w < p.W; w += 256) {
        const int page = entries[w];
        if (p.is_page(page)) atomicSub(&p.uses[page], 1);
        entries[w] = -1;
    }
    if (threadIdx.x == 0) p.starts[row] = 0;
}

struct TakeParams : View {
    const int32_t* new_lens;   // [S], or nullptr: L
    int L;
    int32_t* missing;          // [S]
    int32_t* list;             // [N]
    // places first .. end of a sequence's row get pages where they have none; beyond the table there is no place
    __device__ __forceinline__ void places(int row, int64_t* first, int64_t* end) const {
        const int64_t P = (int64_t)1 << log2_p, start = starts[row];
        int n = new_lens != nullptr ? new_lens[row] : L;
        n = n < 0 ? 0 : n > L ? L : n;
        const int64_t low = start < 0 ? 0 : start, high = start + n < 0 ? 0 : start + n;
        *first = (low + P - 1) >> log2_p;
        *end = n > 0 ? (high + P - 1) >> log2_p : *first;
    }
};

// One workgroup: the sequences' wants, the free pages in ascending order, and the pages to the places in the order of the rows.  Barriers
// and loads one after the other, not bytes: 5.1 us for 18 sequences and 350 pages, 7.7 for 50 and 4500 (with the
// sequences' places looked up row by row, and lists by way of memory, 6.4 and 12.6); 4096 pages by way of memory behind 50000 used ones 29.
__global__ __launch_bounds__(kPlanThreads) void take_pages_kernel(const TakeParams p) {
    __shared__ int room[kPlanWaves], wants[kPlanThreads];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ int from[kPlanThreads], upto[kPlanThreads], few[kFew];
    // the places first .. last of row base + s that have no page: `got(w, before)` of each lane's, and how many
    auto walk = [&](int base, int s, auto got) {
        const int32_t* const entries = p.table + (base + s) * p.table_stride;
        const int first = from[s], last = upto[s] < p.W ? upto[s] : p.W;
        int n = 0;
        for (int w0 = first; w0 < last; w0 += 4 * 64) {
            int page[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int w = w0 + 64 * i + lane;
                page[i] = w < last ? entries[w] : 0;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool lacks = !p.is_page(page[i]);
                const uint64_t all = __ballot(lacks);
                if (lacks) got(w0 + 64 * i + lane, n + __popcll(all & ((1ull << lane) - 1)));
                n += __popcll(all);
            }
        }
        return n;
    };
    // twice over the rows, kPlanThreads at a time: what all want, then (found pages in `list`) who gets which
    int total = 0;
    int* list = p.list;
    for (int pass = 0; pass < 2; ++pass) {
        int have = 0, given = 0;
        if (pass == 1) {
            if (total > p.N) total = p.N;
            if (total <= kFew) list = few;
            have = find_free(p, total, list, room);
        }
        for (int base = 0; base < p.S; base += kPlanThreads) {
            const int row = base + (int)threadIdx.x, rows = p.S - base < kPlanThreads ? p.S - base : kPlanThreads;
            __syncthreads();
            if (row < p.S) {
                int64_t first, end;
                p.places(row, &first, &end);
                from[threadIdx.x] = (int)first, upto[threadIdx.x] = (int)end;
            }
            __syncthreads();
            for (int s = wave; s < rows; s += kPlanWaves) {
                const int n = walk(base, s, [](int, int) {});
                if (lane == 0) wants[s] = n;
            }
            __syncthreads();
            const Ranks r = rank_of(row < p.S ? wants[threadIdx.x] : 0, room);
            if (pass == 0) {
                total += r.all;                          // at most the table's places, as every sum here
                continue;
            }
            if (row < p.S) wants[threadIdx.x] = given + r.before;        // the rank of its first
            __syncthreads();
            for (int s = wave; s < rows; s += kPlanWaves) {
                const int rank = wants[s], w = from[s] > p.W ? from[s] : p.W;
                const int n = walk(base, s, [&](int w, int before) {
                    const int page = rank + before < have ? list[rank + before] : -1;
                    p.table[(base + s) * p.table_stride + w] = page;
                    if (page >= 0) p.uses[page] = 1;
                });
                const int without = rank + n > have ? (rank > have ? n : rank + n - have) : 0;
                if (lane == 0) p.missing[base + s] = without + (upto[s] > w ? upto[s] - w : 0);
            }
            given += r.all;
        }
    }
}

struct ForkParams : View {
    Tensors tensors;
    const int32_t* parents;
    const int32_t* children;
    int count;
    int32_t* forked;           // [count]
    int32_t* lengths;          // [count]: of the parents, -1: not forked
    int32_t* copies;           // [count]: the page that the child's last tokens go to, -1: none
    int32_t* list;             // [count]
};

// The parent's page that its child cannot share, because the last tokens do not fill it; -1: there is none.
__device__ __forceinline__ int unshared(const ForkParams& p, int parent, int length) {
    const int w = length >> p.log2_p;
    if ((length & ((1 << p.log2_p) - 1)) == 0 || w >= p.W) return -1;
    const int page = p.table[parent * p.table_stride + w];
    return p.is_page(page) ? page : -1;
}

// One workgroup: which pairs are forked, and the pages that they take.  Changes nothing but uses, of pages that were free.  4 to 6 us for up to 16 pairs;
// each looks through all before it (both kernels, 256 pairs 42 us, 1024 156, 4096 1370).
__global__ __launch_bounds__(kPlanThreads) void plan_fork_kernel(const ForkParams p) {
    __shared__ int room[kPlanWaves];
    int total = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int have = 0, given = 0;
        if (pass == 1) have = find_free(p, total < p.N ? total : p.N, p.list, room);
        for (int base = 0; base < p.count; base += kPlanThreads) {
            const int n = base + (int)threadIdx.x;
            int length = -1, needs = 0;
            if (n < p.count) {
                const int parent = p.parents[n], child = p.children[n];
                if ((uint32_t)parent < (uint32_t)p.S && (uint32_t)child < (uint32_t)p.S && parent != child && p.starts[child] == 0) {
                    length = p.starts[parent] < 0 ? 0 : p.starts[parent];
                    for (int m = 0; m < n; ++m)
                        if (p.children[m] == child) length = -1;
                    needs = length > 0 && unshared(p, parent, length) >= 0;
                }
            }
            const Ranks r = rank_of(needs, room);
            total += pass == 0 ? r.all : 0;
            if (pass == 1 && n < p.count) {
                const int rank = given + r.before;
                int page = -1;
                if (needs) {
                    if (rank < have)
                        page = p.list[rank], p.uses[page] = 1;
                    else
                        length = -1;
                }
                p.lengths[n] = length;
                p.copies[n] = page;
                p.forked[n] = length >= 0;
            }
            given += r.all;
        }
    }
}

// Workgroups (n, 0): the child's row, its length and the uses of what it shares; (n, 1 + chunk): a chunk of the copied page.  4 to 6 us for up
// to eight pages of 132 KB.
__global__ __launch_bounds__(256) void fork_pages_kernel(const ForkParams p) {
    const int per = 1 + p.tensors.first_chunk[p.tensors.count], n = (int)(blockIdx.x / per), part = (int)(blockIdx.x % per);
    const int length = p.lengths[n], copy = p.copies[n];
    if (length < 0) return;                              // not forked; of a parent without tokens the child's row is cleared all the same
    const int parent = p.parents[n], child = p.children[n];
    if (part > 0) {
        if (copy >= 0) copy_chunk(p.tensors, part - 1, unshared(p, parent, length), copy);
        return;
    }
    const int full = length >> p.log2_p;
    for (int w = threadIdx.x; w < p.W; w += 256) {
        int32_t* const entry = p.table + child * p.table_stride + w;
        int page = -1;
        if (w < full) {
            page = p.table[parent * p.table_stride + w];
            if (p.is_page(page)) atomicAdd(&p.uses[page], 1);
        } else if (w == full) {
            page = copy;
        }
        if (const int was = *entry; p.is_page(was)) atomicSub(&p.uses[was], 1);      // taken before it had a token
        *entry = page;
    }
    if (threadIdx.x == 0) p.starts[child] = length;
}

struct CompactParams : View {
    Tensors tensors;
    int32_t* moved;            // [N]
    int32_t* holes;            // [N / 2]
    int32_t* movers;           // [N / 2]
    int32_t* count;            // [1]
    int copy_wgs, table_wgs;
    Divisor by_width, by_chunks;
};

// One workgroup: the used pages are counted, U of them; the k-th hole among the first U pages takes the k-th used page behind them.  3.3 us for
// 350 pages, 7.9 for 4500, barrier after barrier (with the second kernel 18 for 20000, 70 for 100000).
__global__ __launch_bounds__(kPlanThreads) void plan_compact_kernel(const CompactParams p) {
    __shared__ int room[kPlanWaves];
    constexpr int kEach = 4;
    int mine = 0;
    for (int base = 0; base < p.N; base += kEach * kPlanThreads) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int page = base + i * kPlanThreads + (int)threadIdx.x;
            mine += page < p.N && p.uses[page] > 0;
        }
    }
    const int U = rank_of(mine, room).all;
    int holes = 0, movers = 0;
    for (int base = 0; base < p.N; base += kEach * kPlanThreads) {
        const int at = base + kEach * (int)threadIdx.x;
        bool used[kEach];
        int n = 0;                                       // holes, and movers from bit 16 on: at most kEach * kPlanThreads of each
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            used[i] = at + i < p.N && p.uses[at + i] > 0;
            n += at + i < U ? !used[i] : used[i] << 16;
        }
        const Ranks r = rank_of(n, room);
        int hole = holes + (r.before & 0xffff), mover = movers + (r.before >> 16);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (at + i >= p.N) break;
            if (at + i < U && !used[i]) p.holes[hole++] = at + i;
            if (at + i >= U && used[i]) p.movers[mover++] = at + i;
            if (at + i < U || !used[i]) p.moved[at + i] = used[i] ? at + i : -1;
        }
        holes += r.all & 0xffff;
        movers += r.all >> 16;
    }
    __syncthreads();                                     // both lists are written
    for (int k = threadIdx.x; k < holes; k += kPlanThreads) {
        const int from = p.movers[k], to = p.holes[k];
        p.moved[from] = to;
        p.uses[to] = p.uses[from];
        p.uses[from] = 0;
    }
    if (threadIdx.x == 0) *p.count = holes;
}

// The first workgroups copy the pages that move, the others write the table's new entries.  Bound by the bytes: 1500 pages of 132 KB, 412 MB
// read and written, in 90 us, 4.6 TB/s.
__global__ __launch_bounds__(256) void compact_pages_kernel(const CompactParams p) {
    if ((int)blockIdx.x < p.copy_wgs) {
        const int chunks = p.tensors.first_chunk[p.tensors.count];
        const int64_t items = (int64_t)*p.count * chunks;
        for (int64_t item = blockIdx.x; item < items; item += p.copy_wgs) {
            const int n = item < 0x7fffffff ? p.by_chunks.of((int)item) : (int)(item / chunks);
            copy_chunk(p.tensors, (int)(item - (int64_t)n * chunks), p.movers[n], p.holes[n]);
        }
        return;
    }
    const int64_t entries = (int64_t)p.S * p.W;
    for (int64_t e = (int64_t)(blockIdx.x - p.copy_wgs) * 256 + threadIdx.x; e < entries; e += (int64_t)p.table_wgs * 256) {
        const int row = e < 0x7fffffff ? p.by_width.of((int)e) : (int)(e / p.W);
        int32_t* entry = p.table + row * p.table_stride + (e - (int64_t)row * p.W);
        const int page = *entry;
        *entry = p.is_page(page) ? p.moved[page] : -1;
    }
}

}  // namespace pages
}  // namespace fa
