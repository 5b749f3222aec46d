// Launch parameters and plan of the paged-cache kernels (paged.hip,
// paged_attn.hip), in plain C++.
#pragma once

#include <stdint.h>

#include "nne_params.hpp"

namespace nne {

constexpr int kPagedSeqs = 128;       // sequences of one attention launch
constexpr int kPagedTreeNodes = 256;  // drafted tokens with parents
constexpr int kPagedMaxDim = 256;

// Division by a positive d < 2^31 as a multiplication, for 0 <= n < 2^31: with
// 2^(s-1) < d <= 2^s and mul = ceil(2^(31+s) / d) < 2^32, mul * d = 2^(31+s) + e
// with e < d <= 2^s, so the quotient's error n * e / (d * 2^(31+s)) is below 1 / d
// and never carries it past an integer.  (A division takes a wave about 30
// instructions, and a launch of one block of keys is its instructions.)
struct Divisor {
    uint32_t mul;
    int shift;
};
inline Divisor divisor(int64_t d) {
    int s = 0;
    while ((int64_t{1} << s) < d) ++s;
    return Divisor{(uint32_t)(((uint64_t{1} << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d), s};
}

// One layer's pools and the sequences' pages.  Rows of the pools are counted
// through: page pg, KV head h and row r of the page are row
// (pg * Hkv + h) * page_size + r, d elements each.
struct PagedPool {
    void *k, *v;
    int bf16;
    int n_pages, Hkv, page_size, d, max_pages;
    Divisor by_page;
    const int32_t* table;
    int32_t* lens;
};

struct PagedAttnParams {
    View4 q;
    OutView4 o;
    PagedPool pool;
    const int32_t* counts;     // [B] or null: T
    const int32_t* parents;    // [B][T] or null: a chain
    int G, T;
    Divisor by_g, by_hkv, by_rb;
    int R;                     // query rows of a KV head, G * T: row r is token r / G, head r % G
    int tile_rows;             // 16 or 32
    int n_rb;                  // blocks of tile_rows rows
    int rec_rows;              // rows of a record: min(R, rows of the tile)
    int vec_q, vec_o;          // q's and o's rows are 16-byte vectors
    float qscale;              // softmax scale * log2(e)
    int b0;                    // first sequence of the launch
    int B;                     // sequences of the launch
    float* ws;                 // records: (max, sum) and O of rec_rows rows each
    uint32_t* cnt;             // arrivals per (sequence, KV head, row block)
    int combine;               // records are merged by a kernel of their own, not by the last to arrive
    // The keys of sequence b0 + order[i] are cut into prefix[i + 1] - prefix[i] equal
    // parts, numbered through the launch.
    uint16_t prefix[kPagedSeqs + 1];
    uint8_t order[kPagedSeqs];
};

// Dims of the tile.
inline int paged_tile_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// Floats of a record: (max, sum) of each row, then 16-byte aligned rows of O.
#ifdef __HIPCC__
__host__ __device__
#endif
inline int64_t paged_record_floats(int rows, int D) { return ((2 * rows + 3) & ~3) + (int64_t)rows * D; }

// Most bytes of records of a launch over B sequences of R query rows per KV head, on a
// device of `cus` CUs; 0 where it never splits (they would pass kPagedRecordBytes).
constexpr int64_t kPagedRecordBytes = int64_t{1} << 28;
int64_t paged_record_bytes(int64_t B, int64_t Hkv, int64_t R, int64_t d, int cus);

// Tiles of 16 or 32 rows: sets tile_rows, n_rb, by_rb and rec_rows of p.
void paged_set_tile(PagedAttnParams& p, int tile_rows);

// Takes the tile and fills p.prefix and p.combine for sequences of keys[b] keys (p's
// sizes set); returns the number of records (0: nothing is split).
int64_t paged_plan(PagedAttnParams& p, const int64_t* keys, int cus);

struct PagedAppendParams {
    View4 k, v;
    PagedPool pool;
    const int32_t *counts, *depths;
    const float *cos, *sin;    // null: no rotation
    int max_seq_len;
    int B, T;
    Divisor by_token, by_row, by_t;       // threads of a token and of a row, T
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
    Divisor by_heads, by_t;
    int norm;
    float eps;
    const float *cos, *sin;    // null: no rotation
    int max_seq_len;
    const int32_t *start, *depths;
    int vec;                   // rows, weights and tables are 16-byte vectors
};

}  // namespace nne
