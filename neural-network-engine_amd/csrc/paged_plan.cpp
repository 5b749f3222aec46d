// Key split of the paged-attention kernel: how many workgroups share a
// (sequence, KV head, row block).
#include <algorithm>

#include "paged.hpp"

namespace nne {

namespace {
constexpr int kTargetPerCu = 4;    // workgroups per CU that a split may make
}

int64_t paged_max_records(int64_t B, int64_t units, int64_t record_bytes, int cus) {
    const int64_t n = (int64_t)kTargetPerCu * cus + B * units;
    return n * record_bytes <= kPagedRecordBytes ? n : 0;
}

int64_t paged_plan(PagedAttnParams& p, const int64_t* keys, int cus) {
    const int64_t units = (int64_t)p.pool.Hkv * p.n_rb;    // workgroups of a part
    int64_t longest = 1, total = 0;
    for (int b = 0; b < p.B; ++b) {
        longest = std::max(longest, keys[b]);
        total += keys[b];
    }
    // Part lengths from the longest sequence down to 64 keys; the one of least
    // modelled time: a workgroup pays a fixed time and its keys, as many run at
    // once as the device holds, and a sequence in parts pays their merge.
    const int64_t step = p.pool.bf16 ? 128 : 64;           // keys of a round of the waves
    const int64_t slots = 2 * (int64_t)cus;
    const int64_t most = paged_max_records(p.B, units, 4 * paged_record_floats(p.rec_rows, paged_tile_dim(p.pool.d)), cus);
    int64_t best_len = longest;
    double best = 1e300;
    for (int64_t n = 1; n <= 512; n = n < 8 ? n + 1 : n + n / 4) {
        const int64_t len = ((longest + n - 1) / n + step - 1) / step * step;
        int64_t parts = 0;
        for (int b = 0; b < p.B; ++b) parts += std::max<int64_t>(1, (keys[b] + len - 1) / len);
        const int64_t wgs = parts * units;
        if (n > 1 && wgs > most) break;
        const int64_t rounds = (wgs + slots - 1) / slots;
        // Long launches flow through the device, short ones run in rounds.
        const double flow = (double)total * units / slots;
        const double time = 400.0 + (rounds <= 2 ? (double)rounds * (double)(std::min(len, longest) + 150)
                                                 : flow + 150.0 * rounds + 0.5 * (double)len)
                            + (n > 1 ? 100.0 + 12.0 * (double)n : 0.0);
        if (time < best) { best = time; best_len = len; }
        if (len == step) break;
    }
    p.combine = 0;
    p.prefix[0] = 0;
    for (int b = 0; b < p.B; ++b)
        p.prefix[b + 1] = (uint16_t)(p.prefix[b] + std::max<int64_t>(1, (keys[b] + best_len - 1) / best_len));
    if (p.prefix[p.B] == p.B) p.combine = 0;
    return p.prefix[p.B] > p.B ? p.prefix[p.B] * units : 0;
}

}  // namespace nne
