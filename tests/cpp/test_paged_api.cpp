// Tests of the paged cache in the C++ host API (neural-network-engine_amd/host/nne.hpp)
// against plain loops in 64 bits, with the bar |gpu - ref| <= 1e-4 + 1e-3 |ref|.
//
//   test_paged_api            run every test (needs a GPU)
//   test_paged_api --cpu      run only the tests that touch no device
// Prints "ok <name>" / "FAIL <name>: <why>" per test; exit status = failures.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <stdexcept>
#include <string>
#include <vector>

#include "nne.hpp"

using namespace nne;

namespace {

struct Failure : std::runtime_error {
    using std::runtime_error::runtime_error;
};

#define CHECK(cond)                                                                                          \
    do {                                                                                                     \
        if (!(cond)) throw Failure(std::string(#cond) + " (line " + std::to_string(__LINE__) + ")");         \
    } while (0)

template <class F>
bool throws(F f) {
    try {
        f();
    } catch (const std::invalid_argument&) {
        return true;
    }
    return false;
}

void close(const std::vector<float>& got, const std::vector<double>& want) {
    CHECK(got.size() == want.size());
    for (size_t i = 0; i < got.size(); ++i)
        if (!(std::fabs(got[i] - want[i]) <= 1e-4 + 1e-3 * std::fabs(want[i])))
            throw Failure("element " + std::to_string(i) + ": " + std::to_string(got[i]) + " for " + std::to_string(want[i]));
}

// Softmax attention of rows q [Hq, T, d] over key lists: sees(t, c) on n keys, whose
// rows are k, v [n][Hkv * d].
std::vector<double> attention(const float* q, size_t hq, size_t t, size_t d, size_t hkv,
                              const std::vector<std::vector<float>>& k, const std::vector<std::vector<float>>& v,
                              const std::function<bool(size_t, size_t)>& sees) {
    std::vector<double> out(hq * t * d, 0);
    for (size_t h = 0; h < hq; ++h)
        for (size_t r = 0; r < t; ++r) {
            const size_t g = h / (hq / hkv) * d;
            std::vector<double> s(k.size(), -INFINITY);
            double m = -INFINITY, l = 0;
            for (size_t c = 0; c < k.size(); ++c) {
                if (!sees(r, c)) continue;
                s[c] = 0;
                for (size_t i = 0; i < d; ++i) s[c] += (double)q[(h * t + r) * d + i] * k[c][g + i];
                s[c] /= std::sqrt((double)d);
                m = std::max(m, s[c]);
            }
            for (size_t c = 0; c < k.size(); ++c) l += s[c] = sees(r, c) ? std::exp(s[c] - m) : 0;
            for (size_t c = 0; c < k.size(); ++c)
                for (size_t i = 0; i < d; ++i) out[(h * t + r) * d + i] += s[c] / l * v[c][g + i];
        }
    return out;
}

// One sequence's row `pos` of a [B, H, T, d] tensor's copy.
std::vector<float> row_of(const std::vector<float>& x, size_t b, size_t h, size_t t, size_t d, size_t pos) {
    std::vector<float> r(h * d);
    for (size_t i = 0; i < h; ++i)
        std::copy_n(x.begin() + ((b * h + i) * t + pos) * d, d, r.begin() + i * d);
    return r;
}

void refusals_without_a_device() {
    CHECK(throws([] { PagedKVCache(1, 4, 2, 8, 12, 2, 4); }));            // head dim
    CHECK(throws([] { PagedKVCache(1, 0, 2, 8, 16, 2, 4); }));
    CHECK(throws([] { PagedKVCache(1, 4, 2, 0, 16, 2, 4); }));
    CHECK(throws([] { PagedKVCache(1, (size_t)1 << 31, 2, 8, 16, 2, 4); }));
    CHECK(throws([] { DraftTree(1, 2, {-1}); }));
    CHECK(throws([] { DraftTree(1, 2, {-1, 1}); }));
    CHECK(throws([] { DraftTree(1, 2, {-2, 0}); }));
    CHECK(throws([] { DraftTree(1, 2, {-1, 0}, {3}); }));
    CHECK(throws([] { DraftTree(1, 2, {-1, 0}, {1, 1}); }));
    CHECK(throws([] { DraftTree::chain(2, 2, {-1, 0}); }));
}

void steps_of_a_serving_loop() {
    const size_t B = 2, hq = 4, hkv = 2, d = 16, layers = 2;
    PagedKVCache cache(layers, 12, hkv, 4, d, B, 8);
    CHECK(cache.num_layers() == layers && cache.capacity() == 32);
    std::vector<std::vector<float>> ks[layers][B], vs[layers][B];       // the rows that count
    const std::vector<int32_t> parents{-1, 0, 0, 2, -1, -1, 0, 1, 1, 3};
    const std::vector<int32_t> paths{0, 2, 3, 0, 1, 4};                 // of trees' tokens
    for (int step = 0; step < 3; ++step) {
        const bool tree = step == 1;
        const size_t t = step == 0 ? 7 : tree ? 5 : 1;
        std::vector<size_t> rows;
        for (size_t b = 0; b < B; ++b) rows.push_back(cache.lengths()[b] + t);
        CHECK(cache.allocate(rows).is_ok());
        const std::vector<int32_t> counts = step == 0 ? std::vector<int32_t>{7, 3} : std::vector<int32_t>{};
        const DraftTree draft = tree ? DraftTree(B, t, parents) : DraftTree::chain(B, t, counts);
        for (size_t layer = 0; layer < layers; ++layer) {
            const RawTensor q = RawTensor::randn({B, hq, t, d}, 0.f, 1.f), k = RawTensor::randn({B, hkv, t, d}, 0.f, 1.f),
                            v = RawTensor::randn({B, hkv, t, d}, 0.f, 1.f);
            CHECK(cache.append(layer, k, v, nullptr, &draft).is_ok());
            const RawTensor o = cache.attend(layer, q, &draft).unwrap();
            CHECK(o.shape() == q.shape());
            const auto qv = q.to_vec(), kv = k.to_vec(), vv = v.to_vec(), ov = o.to_vec();
            for (size_t b = 0; b < B; ++b) {
                const size_t n = counts.empty() ? t : (size_t)counts[b], ctx = ks[layer][b].size();
                auto kk = ks[layer][b], vv2 = vs[layer][b];
                for (size_t i = 0; i < n; ++i) {
                    kk.push_back(row_of(kv, b, hkv, t, d, i));
                    vv2.push_back(row_of(vv, b, hkv, t, d, i));
                }
                const auto sees = [&](size_t r, size_t c) {
                    if (c < ctx) return true;
                    if (!tree) return c - ctx <= r;
                    for (int at = (int)r; at >= 0; at = parents[b * t + at])
                        if ((size_t)at == c - ctx) return true;
                    return false;
                };
                auto want = attention(qv.data() + b * hq * t * d, hq, t, d, hkv, kk, vv2, sees);
                for (size_t h = 0; h < hq; ++h)                        // zeros past the counts
                    std::fill(want.begin() + (h * t + n) * d, want.begin() + (h + 1) * t * d, 0.0);
                close(std::vector<float>(ov.begin() + b * hq * t * d, ov.begin() + (b + 1) * hq * t * d), want);
                if (tree)
                    for (size_t i = 0; i < 3; ++i) {
                        ks[layer][b].push_back(kk[ctx + paths[3 * b + i]]);
                        vs[layer][b].push_back(vv2[ctx + paths[3 * b + i]]);
                    }
                else
                    ks[layer][b] = kk, vs[layer][b] = vv2;
            }
        }
        if (tree) CHECK(cache.commit({3, 3}, paths).is_ok());
        else CHECK(cache.commit(counts.empty() ? std::vector<int32_t>(B, (int32_t)t) : counts).is_ok());
        for (size_t b = 0; b < B; ++b) CHECK((size_t)cache.lengths()[b] == ks[0][b].size());
    }
    // refusals leave the cache as it was
    const auto lens = cache.lengths();
    const RawTensor x = RawTensor::zeros({B, hkv, 1, d}), q = RawTensor::zeros({B, hq, 1, d});
    CHECK(cache.append(2, x, x).is_err() && cache.append(0, q, x).is_err() && cache.append(0, x, q).is_err());
    CHECK(cache.attend(2, q).is_err() && cache.attend(0, RawTensor::zeros({B, 3, 1, d})).is_err());
    const DraftTree two = DraftTree::chain(B, 2);
    CHECK(cache.attend(0, q, &two).error().kind == EngineError::Kind::ShapeMismatch);
    CHECK(cache.commit({1}).is_err() && cache.commit({-1, 0}).is_err() && cache.commit({33, 0}).is_err());
    CHECK(cache.commit({2, 2}, {1, 0, 0, 1}).is_err());
    CHECK(cache.allocate({33, 0}).error().kind == EngineError::Kind::GpuError);
    CHECK(cache.set_lengths({40, 0}).is_err() && cache.set_lengths({32, 32}).is_err() && cache.set_table({0}).is_err());
    CHECK(cache.release(2).is_err());
    CHECK(cache.lengths() == lens);
    CHECK(cache.release(0).is_ok() && cache.lengths()[0] == 0 && cache.lengths()[1] == lens[1]);
}

// A layer's step over a paged cache is its step over a KVCache: a prompt, then tokens.
void layer_steps(PagedKVCache::Dtype dtype, bool drafts) {
    const size_t B = 2, C = 128, hq = 4, hkv = 2, d = 32;
    GroupedQueryAttention gqa(C, hq, hkv, 64);
    KVCache plain(1, B, hkv, 64, d);
    PagedKVCache paged(1, 16, hkv, 8, d, B, 8, dtype);
    size_t len = 0;
    for (size_t t : {6, 1, 3, 1}) {
        const RawTensor x = RawTensor::randn({B, t, C}, 0.f, 1.f);
        const auto want = gqa.forward_gqa_cached(x, len, &plain, 0).unwrap().to_vec();
        CHECK(paged.allocate({len + t, len + t}).is_ok());
        const DraftTree chain = DraftTree::chain(B, t);
        const auto got = gqa.forward_gqa_paged(x, paged, 0, drafts ? &chain : nullptr).unwrap().to_vec();
        if (dtype == PagedKVCache::Dtype::F32) close(got, std::vector<double>(want.begin(), want.end()));
        else CHECK(got.size() == want.size());
        CHECK(paged.commit({(int32_t)t, (int32_t)t}).is_ok());
        len += t;
    }
    CHECK(gqa.forward_gqa_paged(RawTensor::zeros({B, C}), paged).is_err());
    CHECK(gqa.forward_gqa_paged(RawTensor::zeros({1, 1, C}), paged).is_err());
    // with a norm of ones and zeros' weights: heads of zero keys leave equal weights
    gqa.set_qk_norm(RawTensor::zeros({d}), RawTensor::zeros({d}));
    CHECK(paged.allocate({len + 1, len + 1}).is_ok());
    CHECK(gqa.forward_gqa_paged(RawTensor::randn({B, 1, C}, 0.f, 1.f), paged).is_ok());
    gqa.set_qk_norm(RawTensor::zeros({d + 2}), RawTensor::zeros({d}));
    CHECK(gqa.forward_gqa_paged(RawTensor::zeros({B, 1, C}), paged).error().kind == EngineError::Kind::ShapeMismatch);
}

void norm_and_rotation() {
    const size_t B = 2, H = 3, T = 4, d = 8;
    PagedKVCache cache(1, 8, 1, 8, d, B, 4);
    CHECK(cache.allocate({20, 10}).is_ok() && cache.set_lengths({13, 5}).is_ok());
    const RotaryEmbedding rope(d, 32, 10000.f);
    const RawTensor q = RawTensor::randn({B, T, H, d}, 0.f, 2.f).transpose(1, 2).value();
    const RawTensor k = RawTensor::randn({B, 1, T, d}, 0.f, 1.f), w = RawTensor::uniform({d}, 0.5f, 1.5f);
    const DraftTree draft(B, T, {-1, -1, 1, 0, -1, 0, 1, 2});
    const auto got = qk_norm_rope(q, k, &w, nullptr, 1e-5f, &rope, cache, &draft).unwrap();
    const auto cs = rope.cos_cached.to_vec(), sn = rope.sin_cached.to_vec(), wv = w.to_vec();
    const auto expect = [&](const RawTensor& x, size_t heads, bool weighted) {
        const auto xv = x.to_contiguous().to_vec();
        std::vector<double> out(xv.size());
        for (size_t r = 0; r < B * heads * T; ++r) {
            const size_t b = r / (heads * T), t = r % T, at = cache.lengths()[b] + draft.depths[b * T + t];
            double sum = 0, y[8];
            for (size_t i = 0; i < d; ++i) sum += (double)xv[r * d + i] * xv[r * d + i];
            for (size_t i = 0; i < d; ++i)
                y[i] = xv[r * d + i] / std::sqrt(sum / d + 1e-5) * (weighted ? wv[i] : 1.f);
            for (size_t i = 0; i < d; ++i)
                out[r * d + i] = y[i] * cs[at * d + i] + (i < d / 2 ? -y[i + d / 2] : y[i - d / 2]) * sn[at * d + i];
        }
        return out;
    };
    close(got.first.to_vec(), expect(q, H, true));
    close(got.second.to_vec(), expect(k, 1, false));
    const RotaryEmbedding other(16, 32, 10000.f), few(d, 15, 10000.f);
    CHECK(qk_norm_rope(q, k, &w, nullptr, 1e-5f, &other, cache).is_err());
    CHECK(qk_norm_rope(q, k, &w, nullptr, 1e-5f, &few, cache).is_err());       // position 16
    CHECK(qk_norm_rope(q, k, &w, nullptr, std::nullopt, &rope, cache).is_err());
    CHECK(qk_norm_rope(q, RawTensor::zeros({B, 1, T + 1, d}), nullptr, nullptr, 1e-5f, &rope, cache).is_err());
}

struct Test {
    const char* name;
    bool needs_gpu;
    std::function<void()> fn;
};

}  // namespace

int main(int argc, char** argv) {
    const bool cpu = argc > 1 && std::strcmp(argv[1], "--cpu") == 0;
    const std::vector<Test> tests{
        {"refusals_without_a_device", false, refusals_without_a_device},
        {"steps_of_a_serving_loop", true, steps_of_a_serving_loop},
        {"layer_steps", true, [] { layer_steps(PagedKVCache::Dtype::F32, false); }},
        {"layer_steps_drafted", true, [] { layer_steps(PagedKVCache::Dtype::F32, true); }},
        {"layer_steps_bf16", true, [] { layer_steps(PagedKVCache::Dtype::Bf16, false); }},
        {"norm_and_rotation", true, norm_and_rotation},
    };
    int run = 0, failed = 0;
    for (const Test& t : tests) {
        if (cpu && t.needs_gpu) continue;
        ++run;
        std::printf("run %s\n", t.name);
        std::fflush(stdout);
        try {
            t.fn();
            std::printf("ok %s\n", t.name);
        } catch (const std::exception& e) {
            ++failed;
            std::printf("FAIL %s: %s\n", t.name, e.what());
        }
    }
    std::printf("%d of %d tests failed\n", failed, run);
    return failed != 0;
}
