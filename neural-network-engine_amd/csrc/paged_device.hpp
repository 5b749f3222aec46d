// Device helpers of the paged-cache kernels.
#pragma once

#include "nne_common.hpp"
#include "paged.hpp"

namespace nne {

__device__ __forceinline__ int quotient(int n, Divisor d) { return (int)(__umulhi(2u * (uint32_t)n, d.mul) >> d.shift); }

// Pool row (page through page_size) of row r of the sequence with page table
// row `table`, or -1 where its page is outside the pool.
__device__ __forceinline__ int paged_row(const PagedPool& p, const int32_t* table, int h, int r) {
    const int which = quotient(r, p.by_page);
    if (which >= p.max_pages) return -1;
    const int page = table[which];
    if ((unsigned)page >= (unsigned)p.n_pages) return -1;
    return (page * p.Hkv + h) * p.page_size + (r - which * p.page_size);
}

// A sequence's counted rows, at most what its pages hold (the host keeps that
// and a step's tokens together below 2^31).
__device__ __forceinline__ int paged_clamp(const PagedPool& p, int len) {
    const int cap = p.max_pages * p.page_size;
    return len < 0 ? 0 : len > cap ? cap : len;
}
__device__ __forceinline__ int paged_len(const PagedPool& p, int b) { return paged_clamp(p, p.lens[b]); }

__device__ __forceinline__ int paged_count(const int32_t* counts, int b, int T) {
    if (!counts) return T;
    const int c = counts[b];
    return c < 0 ? 0 : c > T ? T : c;
}

}  // namespace nne
