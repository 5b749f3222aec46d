// Launch parameters and plan of the paged-cache kernels (paged.hip,
// paged_attn.hip), in plain C++.
#pragma once

#include <stdint.h>

#include "nne_params.hpp"

namespace nne {

constexpr int kPagedSeqs = 128;       // sequences of one attention launch
constexpr int kPagedTreeNodes = 256;  // drafted tokens with parents
constexpr int kPagedMaxDim = 256;

// One layer's pools and the sequences' pages.  Rows of the pools are counted
// through: page pg, KV head h and row r of the page are row
// (pg * Hkv + h) * page_size + r, d elements each.
struct PagedPool {
    void *k, *v;
    int bf16;
    int n_pages, Hkv, page_size, d, max_pages;
    // row / page_size == (row * page_mul) >> page_shift for 0 <= row < 2^31
    uint32_t page_mul;
    int page_shift;
    const int32_t* table;
    int32_t* lens;
};

// row / page_size as a multiplication: with 2^(s-1) < page_size <= 2^s and
// mul = ceil(2^(31+s) / page_size) < 2^32, mul * page_size = 2^(31+s) + e with
// e < page_size <= 2^s, so the quotient's error row * e / (page_size * 2^(31+s))
// is below 1 / page_size and never carries it past an integer.
inline void paged_division(PagedPool& p) {
    int s = 0;
    while ((int64_t{1} << s) < p.page_size) ++s;
    p.page_mul = (uint32_t)(((uint64_t{1} << (31 + s)) + (uint64_t)p.page_size - 1) / (uint64_t)p.page_size);
    p.page_shift = 31 + s;
}

struct PagedAttnParams {
    View4 q;
    OutView4 o;
    PagedPool pool;
    const int32_t* counts;     // [B] or null: T
    const int32_t* parents;    // [B][T] or null: a chain
    int Hq, G, T;
    int R;                     // query rows of a KV head, G * T: row r is token r / G, head r % G
    int n_rb;                  // blocks of kernel-tile rows
    int rec_rows;              // rows of a record: min(R, rows of the tile)
    int vec_q;                 // q rows are 16-byte vectors
    float qscale;              // softmax scale * log2(e)
    int b0;                    // first sequence of the launch
    int B;                     // sequences of the launch
    float* ws;                 // records: (max, sum) and O of rec_rows rows each
    uint32_t* cnt;             // arrivals per (sequence, KV head, row block)
    // Sequence b's keys are cut into parts prefix[b + 1] - prefix[b], numbered
    // through the launch.
    int prefix[kPagedSeqs + 1];
};

// Rows of the tile that R query rows of d dims take, and its dims.
inline int paged_tile_rows(int R, int d) { return R <= 16 ? 16 : R <= 32 || d > 128 ? 32 : 64; }
inline int paged_tile_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// Floats of a record: (max, sum) of each row, then 16-byte aligned rows of O.
#ifdef __HIPCC__
__host__ __device__
#endif
inline int64_t paged_record_floats(int rows, int D) { return ((2 * rows + 3) & ~3) + (int64_t)rows * D; }

// Fills p.prefix for sequences of keys[b] keys (p.R, p.n_rb and p.pool set) on a
// device of `cus` CUs; returns the number of parts.
int paged_plan(PagedAttnParams& p, const int64_t* keys, int cus);

// Most records a launch over B sequences can need.
int64_t paged_max_records(int64_t B, int64_t heads_blocks, int cus);

struct PagedAppendParams {
    View4 k, v;
    PagedPool pool;
    const int32_t *counts, *depths;
    const float *cos, *sin;    // null: no rotation
    int max_seq_len;
    int B, T;
    int vec;                   // k and v rows are 16-byte vectors
};

struct PagedCommitParams {
    PagedPool pool;
    int64_t layer_stride;      // bytes
    const int32_t* counts;     // or null: `count`
    const int32_t* paths;
    int count, J, B, n_layers;
    uint32_t* cnt;             // [B]
};

struct NormRopeParams {
    View4 x[2];                // q, k
    OutView4 o[2];
    const float* w[2];         // or null: ones
    int H[2];
    int B, T, d;
    int norm;
    float eps;
    const float *cos, *sin;    // null: no rotation
    int max_seq_len;
    const int32_t *start, *depths;
    int vec;
};

}  // namespace nne
