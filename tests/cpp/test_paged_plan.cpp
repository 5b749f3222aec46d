// Invariants of the paged-attention kernel's plan (csrc/paged_plan.cpp) and of its
// divisions without a division (csrc/paged.hpp), on the CPU.
//   * paged_plan, over a seeded sweep of batches (1-128 sequences of 1 to 2^30 keys,
//     1-64 KV heads, 1-2^20 query rows, both types, 8-512 CUs): the tile is 16 or 32
//     rows (16 up to 16 rows) and n_rb, rec_rows and by_rb follow from it; order is a
//     permutation of the sequences; prefix rises by at least one part per sequence and
//     by at most one per round of the waves; the records it returns are every part's,
//     or 0 where nothing is split; they fit paged_record_bytes, which no launch
//     without a split allowance passes; a merge kernel is asked for only where there
//     are records; the longest part is first, and where all workgroups run at once
//     the second ones rise.
//   * paged_record_bytes: within kPagedRecordBytes, and what a larger batch, more rows
//     or heads need is more or nothing.
//   * Divisor: the kernel's quotient(n, d) == n / d.
// Prints "<failed> of <checks> checks failed" and exits non-zero on failure.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "paged.hpp"

using namespace nne;

static int g_checks = 0, g_failed = 0;
static char g_case[256];

#define CHECK(cond, ...)                        \
    do {                                        \
        ++g_checks;                             \
        if (!(cond)) {                          \
            ++g_failed;                         \
            std::printf("FAIL [%s] ", g_case);  \
            std::printf(__VA_ARGS__);           \
            std::printf("\n");                  \
        }                                       \
    } while (0)

// As the kernel computes it (paged_device.hpp): high word of a 32-bit product.
static int quotient(int n, Divisor d) {
    return (int)(((uint64_t)(2u * (uint32_t)n) * d.mul >> 32) >> d.shift);
}

static int g_split = 0, g_whole = 0, g_combined = 0, g_tiles[2] = {0, 0}, g_folded = 0;

static void check_plan(int B, int Hkv, int R, int d, int bf16, int cus, const std::vector<int64_t>& keys) {
    std::snprintf(g_case, sizeof g_case, "B=%d Hkv=%d R=%d d=%d bf16=%d cus=%d keys[0]=%lld", B, Hkv, R, d, bf16, cus,
                  (long long)keys[0]);
    PagedAttnParams p{};
    p.B = B;
    p.R = R;
    p.pool.Hkv = Hkv;
    p.pool.d = d;
    p.pool.bf16 = bf16;
    const int64_t records = paged_plan(p, keys.data(), cus);
    const int64_t step = bf16 ? 128 : 64, units = (int64_t)Hkv * p.n_rb;
    CHECK(p.tile_rows == 16 || (p.tile_rows == 32 && R > 16), "tile of %d rows", p.tile_rows);
    CHECK(p.n_rb == (R + p.tile_rows - 1) / p.tile_rows && p.rec_rows == std::min(R, p.tile_rows), "n_rb %d", p.n_rb);
    CHECK(quotient(R - 1, p.by_rb) == (R - 1) / p.n_rb, "by_rb");
    std::vector<int> seen(B, 0);
    CHECK(p.prefix[0] == 0, "prefix[0] = %d", p.prefix[0]);
    std::vector<int64_t> lengths;
    for (int i = 0; i < B; ++i) {
        const int parts = p.prefix[i + 1] - p.prefix[i], b = p.order[i];
        CHECK(b < B && seen[b]++ == 0, "order[%d] = %d", i, b);
        if (b >= B) return;
        CHECK(parts >= 1 && parts <= std::max<int64_t>(1, (keys[b] + step - 1) / step), "%d parts of %lld keys", parts,
              (long long)keys[b]);
        lengths.push_back(parts > 0 ? (keys[b] + parts - 1) / parts : 0);
    }
    const int64_t all = p.prefix[B], wgs = all * units;
    CHECK(records == (all > B ? wgs : 0), "%lld records of %lld parts", (long long)records, (long long)all);
    CHECK(records * 4 * paged_record_floats(p.rec_rows, paged_tile_dim(d)) <= paged_record_bytes(B, Hkv, R, d, cus),
          "%lld records", (long long)records);
    CHECK(!p.combine || records > 0, "a merge of nothing");
    CHECK(lengths[0] == *std::max_element(lengths.begin(), lengths.end()), "a longer part behind the first");
    const bool folds = wgs > cus && wgs <= 2 * (int64_t)cus;
    int64_t first = 0;
    for (int i = 1; i < B; ++i) {
        first += (int64_t)(p.prefix[i] - p.prefix[i - 1]) * units;
        const bool second = folds && first >= cus;
        if (second && first - (int64_t)(p.prefix[i] - p.prefix[i - 1]) * units < cus) continue;   // the fold
        CHECK(second ? lengths[i] >= lengths[i - 1] : lengths[i] <= lengths[i - 1], "part lengths %lld, %lld",
              (long long)lengths[i - 1], (long long)lengths[i]);
        g_folded += second;
    }
    ++(records ? g_split : g_whole);
    g_combined += p.combine;
    ++g_tiles[p.tile_rows / 32];
}

int main() {
    std::mt19937_64 rng(7);
    const auto pick = [&](int64_t lo, int64_t hi) { return (int64_t)(lo + rng() % (uint64_t)(hi - lo + 1)); };
    const auto log_pick = [&](int bits) { return (int64_t)1 << pick(0, bits) | (rng() & ((1ull << pick(0, bits)) - 1)); };
    for (int i = 0; i < 6000; ++i) {
        const int B = (int)pick(1, i % 3 ? 128 : 8), Hkv = (int)pick(1, i % 5 ? 16 : 64);
        const int R = (int)std::min<int64_t>(log_pick(i % 4 ? 9 : 20), 1 << 20), d = 8 * (int)pick(1, 32);
        const int cus = i % 7 ? 256 : (int)pick(8, 512), bits = (int)pick(3, i % 11 ? 14 : 29);
        std::vector<int64_t> keys(B);
        for (auto& k : keys) k = i % 13 ? log_pick(bits) : (int64_t)1 << bits;
        check_plan(B, Hkv, R, d, (int)(rng() & 1), cus, keys);
    }
    std::snprintf(g_case, sizeof g_case, "record bytes");
    for (int i = 0; i < 2000; ++i) {
        const int64_t B = pick(1, 128), Hkv = pick(1, 64), R = log_pick(20), d = 8 * pick(1, 32);
        const int64_t n = paged_record_bytes(B, Hkv, R, d, 256);
        CHECK(n >= 0 && n <= kPagedRecordBytes, "%lld bytes", (long long)n);
        for (const int64_t m : {paged_record_bytes(B + 1, Hkv, R, d, 256), paged_record_bytes(B, Hkv + 1, R, d, 256),
                                paged_record_bytes(B, Hkv, R + 1, d, 256)})
            CHECK(m == 0 || (n != 0 && m >= n), "%lld then %lld bytes", (long long)n, (long long)m);
    }
    std::snprintf(g_case, sizeof g_case, "divisor");
    for (int i = 0; i < 200000; ++i) {
        const int64_t d = i < 2000 ? i + 1 : std::min<int64_t>(log_pick(30), INT32_MAX);
        const Divisor by = divisor(d);
        for (const int64_t n : {(int64_t)0, d - 1, d, std::min<int64_t>(2 * d - 1, INT32_MAX), (int64_t)INT32_MAX,
                                INT32_MAX / d * d, INT32_MAX / d * d - 1, pick(0, INT32_MAX)})
            if (n >= 0) CHECK(quotient((int)n, by) == n / d, "%lld / %lld", (long long)n, (long long)d);
    }
    std::printf("plans: %d split, %d whole, %d merged by a kernel, %d in 16-row and %d in 32-row tiles, %d places folded\n",
                g_split, g_whole, g_combined, g_tiles[0], g_tiles[1], g_folded);
    std::printf("%d of %d checks failed\n", g_failed, g_checks);
    return g_failed != 0;
}
