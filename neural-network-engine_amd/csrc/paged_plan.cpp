// Rows of the tile and key split of the paged-attention kernel: how many workgroups
// share a sequence's rows and keys.
#include <algorithm>
#include <cmath>
#include <functional>

#include "paged.hpp"

namespace nne {

namespace {

constexpr int kTargetPerCu = 4;    // workgroups per CU that a split may make

// Times of the kernel, fitted to 3390 launches of 240 shapes (1-64 sequences of 5-8000
// keys, 1-512 rows, both types, parts of 128-8448 keys; rms error of the fit 7 %; the
// tile and part length it picks take 1.1 % more than the best of those timed).
// [tiles of 16, of 32 rows][f32, bf16 pools][dims up to 64, 128, 256]
constexpr float kStart[2][2][3] = {{{3.1f, 3.7f, 5.3f}, {3.7f, 3.6f, 5.1f}},       // us of a workgroup
                                   {{4.2f, 5.8f, 9.3f}, {5.1f, 6.1f, 8.8f}}};
constexpr float kKey[2][2][3] = {{{.0133f, .0199f, .0286f}, {.0074f, .0101f, .0153f}},   // us of a key
                                 {{.0200f, .0314f, .0539f}, {.0083f, .0130f, .0177f}}};
constexpr float kAtOnce[2][2][3] = {{{1.52f, 1.07f, .73f}, {1.91f, 1.25f, .82f}},  // gain of several on a CU
                                    {{1.23f, 1.03f, .83f}, {1.72f, 1.39f, .83f}}};
constexpr float kLaunch = 2.0f, kBytesPerUs = 6.41e6f;
constexpr float kAgain = 1.38f;         // of bytes that several row blocks read
constexpr float kUneven = .78f, kTail = .13f;   // of the memory's time: of what the longest workgroup has
                                                // over the mean one, and of the last to end
constexpr float kMerge = 1.76f, kMergePart = .078f, kMergeFloat = 7.6e-5f;   // by the last to arrive
constexpr float kCombine = 4.3f, kCombinePart = .034f;                       // by a launch of its own

// Sum of the fourth powers' root: the largest of the three, with the overlap of
// those that come near it.
float joined(float a, float b, float c) {
    a *= a, b *= b, c *= c;
    return std::sqrt(std::sqrt(a * a + b * b + c * c));
}

// Upwards to a whole number (conversions, which vectorise where ceil is a call).
float up(float x) { return (float)(int)(std::min(x, 1e9f) + .9999f); }

// Fills p.order and p.prefix, sequence i in n_parts[i] parts.  Workgroups start in
// this order: those with the longest parts first, so that the last to end are short
// (32 sequences of 512-4096 keys, f32: 107.5 us, 109.9 as they come).  Where all run
// at once, two on a CU, the second ones from the shortest on, so that each CU has a
// long and a short one (256 rows of 8 sequences of 1024-4160 keys: 80 us, 86).
void order_parts(PagedAttnParams& p, const int64_t* keys, const int64_t* n_parts, int64_t units, int cus) {
    uint64_t by_length[kPagedSeqs];
    int64_t total = 0, first = 0;
    for (int i = 0; i < p.B; ++i) {
        by_length[i] = (uint64_t)((keys[i] + n_parts[i] - 1) / n_parts[i]) << 8 | (uint64_t)(kPagedSeqs - 1 - i);
        total += n_parts[i] * units;
    }
    std::sort(by_length, by_length + p.B, std::greater<uint64_t>());
    for (int i = 0; i < p.B; ++i) p.order[i] = (uint8_t)(kPagedSeqs - 1 - (int)(by_length[i] & 255));
    if (total > cus && total <= 2 * (int64_t)cus) {
        int i = 0;
        while (i < p.B && first < cus) first += n_parts[p.order[i++]] * units;
        std::reverse(p.order + i, p.order + p.B);
    }
    p.prefix[0] = 0;
    for (int i = 0; i < p.B; ++i) p.prefix[i + 1] = (uint16_t)(p.prefix[i] + n_parts[p.order[i]]);
}

}  // namespace

int64_t paged_record_bytes(int64_t B, int64_t Hkv, int64_t R, int64_t d, int cus) {
    const int64_t n = (int64_t)kTargetPerCu * cus + B * Hkv * ((R + 31) / 32);
    const int64_t record = 4 * paged_record_floats((int)std::min<int64_t>(R, 32), paged_tile_dim((int)d));
    return n <= kPagedRecordBytes / record ? n * record : 0;
}

void paged_set_tile(PagedAttnParams& p, int tile_rows) {
    p.tile_rows = tile_rows;
    p.n_rb = (p.R + tile_rows - 1) / tile_rows;
    p.by_rb = divisor(p.n_rb);
    p.rec_rows = std::min(p.R, tile_rows);
}

int64_t paged_plan(PagedAttnParams& p, const int64_t* keys, int cus) {
    const int D = paged_tile_dim(p.pool.d), type = p.pool.bf16 ? 1 : 0;
    const int64_t step = p.pool.bf16 ? 128 : 64;           // keys of a round of the waves
    const int64_t most_bytes = paged_record_bytes(p.B, p.pool.Hkv, p.R, p.pool.d, cus);
    float rounds[kPagedSeqs], longest = 1.f, total = 0.f, sum = 0.f;
    for (int b = 0; b < p.B; ++b) {
        rounds[b] = (float)((keys[b] + step - 1) / step);
        longest = std::max(longest, rounds[b]);
        total += rounds[b];
        sum += (float)keys[b];
    }
    const float memory = sum * (float)(p.pool.Hkv * p.pool.d * (p.pool.bf16 ? 4 : 8)) / kBytesPerUs;
    // Tiles of 16 rows start sooner and spread few rows over more CUs, tiles of 32
    // bring K and V half as often: 52 rows of a sequence of 1746 keys take 16.3 and
    // 18.6 us, 256 rows of 8 sequences of 1024-4160 keys 127 and 80.  The part length
    // and the tile of least modelled time: a workgroup pays a fixed time and its
    // keys, a CU its share of them, the memory the bytes, and parts pay their merge.
    // Of those within 3 % of it the one of the longest parts (the model does not tell
    // closer, and its near ties go to them: 48 large batches 2 % faster than with the
    // least itself).
    struct Choice { float time, len; int tile, combine; } all[64];
    int n_all = 0;
    for (int tile = 16; tile <= (p.R > 16 ? 32 : 16); tile += 16) {
        const int at = tile / 32, dims = D / 128, rows = std::min(p.R, tile);
        const float n_rb = (float)((p.R + tile - 1) / tile), heads = (float)p.pool.Hkv;
        const float start = kStart[at][type][dims], key = kKey[at][type][dims], gain = kAtOnce[at][type][dims];
        const float record = 4.f * (float)paged_record_floats(rows, D);
        float last = 0.f;
        for (int n = 1; n <= 512; n = n < 8 ? n + 1 : n + n / 4) {
            const float len = up(longest / (float)n), inv = 1.f / len;
            if (len == last) continue;
            last = len;
            float parts = 0.f;
            for (int b = 0; b < p.B; ++b) parts += std::max(1.f, up(rounds[b] * inv));
            const float wgs = parts * heads * n_rb;
            if (n > 1 && wgs * record > (float)most_bytes) break;
            // Row blocks of a (part, KV head) are on one XCD of 8.
            const float on_cu = n_rb > 1.f ? up(up(parts * heads / 8.f) * n_rb * 8.f / (float)cus) : up(wgs / (float)cus);
            const float one = start + key * len * (float)step;
            const float mean = start + key * total * heads * n_rb / wgs * (float)step;
            const float share = on_cu * mean / gain;
            const float stream = memory * (n_rb > 1.f ? kAgain : 1.f) + kUneven * (one - mean) + kTail * one;
            float time = kLaunch + joined(one, share, stream);
            int combine = 0;
            if (n > 1) {
                const float merge = kMerge + (float)n * (kMergePart + kMergeFloat * (float)(rows * D));
                const float launch = kCombine + (float)n * kCombinePart;
                combine = launch < merge;
                time += std::min(merge, launch);
            }
            all[n_all++] = Choice{time, len, tile, combine};
            if (len == 1.f) break;
        }
    }
    float least = all[0].time;
    for (int i = 1; i < n_all; ++i) least = std::min(least, all[i].time);
    const Choice* best = nullptr;
    for (const Choice& c : all) {
        if (&c == all + n_all) break;
        if (c.time <= 1.03f * least && (!best || c.len > best->len || (c.len == best->len && c.time < best->time)))
            best = &c;
    }
    if (!best) best = all;               // (times past the range of a float)
    paged_set_tile(p, best->tile);
    const int64_t units = (int64_t)p.pool.Hkv * p.n_rb, best_len = (int64_t)best->len * step;
    const int64_t record = 4 * paged_record_floats(p.rec_rows, D);
    int64_t n_parts[kPagedSeqs], parts = 0;
    for (int b = 0; b < p.B; ++b) parts += n_parts[b] = std::max<int64_t>(1, (keys[b] + best_len - 1) / best_len);
    if (parts > p.B && (parts > UINT16_MAX || parts * units * record > most_bytes)) {   // (a rounding of the model's)
        parts = p.B;
        std::fill(n_parts, n_parts + p.B, 1);
    }
    order_parts(p, keys, n_parts, units, cus);
    p.combine = parts > p.B ? best->combine : 0;
    return parts > p.B ? parts * units : 0;
}

}  // namespace nne
