// What the C entries of the cache, the rotary positions, the page keeping and the latent attention check and do on the host.
#pragma once

#include "cache_kernels.hpp"

#include "../../include/fused_attn.h"

#include <algorithm>
#include <array>
#include <cmath>
#include <mutex>
#include <utility>
#include <vector>

namespace {

using fa::cache::Strides3;

constexpr int kNumCu = 256;
constexpr int64_t kMaxInt = 0x7fffffff - 0x10000;
constexpr int64_t kMaxElems = (int64_t)1 << 62;
constexpr int64_t kMostThreads = 0xffffffffll;       // of a grid: the dispatch packet holds no more

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool below(int64_t a, int64_t b, int64_t most) { return a <= most / b; }     // a * b <= most, for positive b

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

}  // namespace
