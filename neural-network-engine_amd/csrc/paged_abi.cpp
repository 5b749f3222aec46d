// extern "C" entry points of the paged KV cache (declared in include/nne_attn.h):
// checks, launch planning, launches.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "nne_abi_internal.hpp"
#include "nne_attn.h"
#include "nne_launch.hpp"
#include "paged_launch.hpp"

namespace {

using nne::fail_format;

#define NNE_BAD "Invalid configuration or argument: "

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool vec_view(const void* p, const int64_t* st) {
    return aligned16(p) && st[3] == 1 && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
}

nne::View4 view(const float* p, const int64_t* st) { return nne::View4{p, st[0], st[1], st[2], st[3]}; }
nne::OutView4 out_view(float* p, const int64_t* st) { return nne::OutView4{p, st[0], st[1], st[2], st[3]}; }

struct Strides {
    int64_t v[4];
    Strides(const int64_t* given, int64_t a, int64_t b, int64_t c, int64_t d) {
        const int64_t shape[4] = {a, b, c, d};
        if (given) std::copy(given, given + 4, v);
        else nne::row_major_strides(shape, v);
    }
};

// Geometry of the cache, its lengths, and T tokens behind them.
int check_cache(const nne_paged_cache_t* c, int64_t T) {
    if (!c) return fail_format(NNE_EINVAL, NNE_BAD "null paged cache");
    if (c->dtype != NNE_F32 && c->dtype != NNE_BF16)
        return fail_format(NNE_EINVAL, NNE_BAD "paged cache dtype %lld", (long long)c->dtype);
    if (c->B < 0 || c->n_pages <= 0 || c->Hkv <= 0 || c->page_size <= 0 || c->max_pages <= 0 ||
        c->B > INT32_MAX || c->n_pages > INT32_MAX || c->Hkv > INT32_MAX || c->page_size > INT32_MAX ||
        c->max_pages > INT32_MAX || (c->n_pages * c->Hkv > INT32_MAX) ||
        (c->n_pages * c->Hkv) * c->page_size > INT32_MAX)
        return fail_format(NNE_EINVAL, NNE_BAD "bad paged cache geometry B=%lld n_pages=%lld Hkv=%lld "
                           "page_size=%lld max_pages=%lld (n_pages * Hkv * page_size must be below 2^31)",
                           (long long)c->B, (long long)c->n_pages, (long long)c->Hkv,
                           (long long)c->page_size, (long long)c->max_pages);
    if (c->d <= 0 || c->d % 8 != 0 || c->d > nne::kPagedMaxDim)
        return fail_format(NNE_EINVAL, NNE_BAD "paged cache head dim %lld must be a multiple of 8 up to %d",
                           (long long)c->d, nne::kPagedMaxDim);
    const int64_t bytes = c->n_pages * c->Hkv * c->page_size * c->d * (c->dtype == NNE_BF16 ? 2 : 4);
    if (bytes >= int64_t{1} << 36)
        return fail_format(NNE_EINVAL, NNE_BAD "a layer's pool of %lld bytes: K and V may have 64 GiB each",
                           (long long)bytes);
    if (T < 0 || T > INT32_MAX || c->max_pages * c->page_size + T > INT32_MAX)
        return fail_format(NNE_EINVAL, NNE_BAD "%lld tokens behind %lld pages of %lld rows", (long long)T,
                           (long long)c->max_pages, (long long)c->page_size);
    if (c->B > 0 && !c->lens_host) return fail_format(NNE_EINVAL, NNE_BAD "lens_host is null");
    return NNE_OK;
}

int check_device_side(const nne_paged_cache_t* c) {
    if (!c->k || !c->v || !c->table || !c->lens_dev)
        return fail_format(NNE_EINVAL, NNE_BAD "null tensor pointer");
    if (!aligned16(c->k) || !aligned16(c->v))
        return fail_format(NNE_EINVAL, NNE_BAD "paged cache pools must be 16-byte aligned");
    return NNE_OK;
}

int check_counts(const nne_paged_cache_t* c, int64_t T, const int32_t* dev, const int32_t* host) {
    if (!dev != !host)
        return fail_format(NNE_EINVAL, NNE_BAD "counts are needed on the device and on the host");
    for (int64_t b = 0; host && b < c->B; ++b)
        if (host[b] < 0 || host[b] > T)
            return fail_format(NNE_EINVAL, NNE_BAD "counts[%lld] = %d outside [0, %lld]", (long long)b,
                               host[b], (long long)T);
    return NNE_OK;
}

int64_t count_of(const int32_t* host, int64_t b, int64_t T) { return host ? host[b] : T; }

// Room for the new rows of every sequence.
int check_room(const nne_paged_cache_t* c, int64_t T, const int32_t* counts_host, int code) {
    const int64_t cap = c->max_pages * c->page_size;
    for (int64_t b = 0; b < c->B; ++b) {
        const int64_t n = count_of(counts_host, b, T);
        if (c->lens_host[b] < 0 || c->lens_host[b] + n > cap)
            return fail_format(code, "GPU compute error: %lld new rows of sequence %lld of length %d "
                               "exceed its %lld pages of %lld rows", (long long)n, (long long)b,
                               c->lens_host[b], (long long)c->max_pages, (long long)c->page_size);
    }
    return NNE_OK;
}

// Pages of rows [first, end) of sequence b, where the host has the table.
int check_pages(const nne_paged_cache_t* c, int64_t b, int64_t first, int64_t end) {
    if (!c->table_host || first >= end) return NNE_OK;
    const int32_t* t = c->table_host + b * c->max_pages;
    for (int64_t i = first / c->page_size; i <= (end - 1) / c->page_size; ++i)
        if (t[i] < 0 || t[i] >= c->n_pages)
            return fail_format(NNE_EINVAL, NNE_BAD "row %lld of sequence %lld has no page (entry %lld is %d, "
                               "of %lld pages)", (long long)std::max(first, i * c->page_size), (long long)b,
                               (long long)i, t[i], (long long)c->n_pages);
    return NNE_OK;
}

// The same, and the pages go to `pages`: those that take new rows.
int add_pages(const nne_paged_cache_t* c, int64_t b, int64_t first, int64_t end, std::vector<int32_t>& pages) {
    const int rc = check_pages(c, b, first, end);
    if (rc || !c->table_host || first >= end) return rc;
    const int32_t* t = c->table_host + b * c->max_pages;
    try {
        pages.insert(pages.end(), t + first / c->page_size, t + (end - 1) / c->page_size + 1);
    } catch (const std::bad_alloc&) {
        return fail_format(NNE_EINVAL, NNE_BAD "out of host memory");
    }
    return NNE_OK;
}

// No page takes new rows of two sequences (or through two entries of one).
int check_apart(std::vector<int32_t>& pages) {
    std::sort(pages.begin(), pages.end());
    const auto twice = std::adjacent_find(pages.begin(), pages.end());
    if (twice == pages.end()) return NNE_OK;
    return fail_format(NNE_EINVAL, NNE_BAD "page %d would take new rows of two places", *twice);
}

nne::PagedPool make_pool(const nne_paged_cache_t* c) {
    nne::PagedPool p{};
    p.k = c->k;
    p.v = c->v;
    p.bf16 = c->dtype == NNE_BF16;
    p.n_pages = (int)c->n_pages;
    p.Hkv = (int)c->Hkv;
    p.page_size = (int)c->page_size;
    p.d = (int)c->d;
    p.max_pages = (int)c->max_pages;
    p.table = c->table;
    p.lens = c->lens_dev;
    p.by_page = nne::divisor(c->page_size);
    return p;
}

int check_rotation(const float* cos_table, const float* sin_table, int64_t max_seq_len,
                   int64_t table_head_dim, int64_t d) {
    if (!cos_table != !sin_table)
        return fail_format(NNE_EINVAL, NNE_BAD "the rotation needs both its tables");
    if (!cos_table) return NNE_OK;
    if (d != table_head_dim)   // llama.rs:119-124
        return fail_format(NNE_ESHAPE, "Shape mismatch error: expected shape [%lld], got [%lld]",
                           (long long)table_head_dim, (long long)d);
    if (max_seq_len <= 0 || max_seq_len > INT32_MAX)
        return fail_format(NNE_EINVAL, NNE_BAD "RoPE max_seq_len %lld", (long long)max_seq_len);
    return NNE_OK;
}

// Positions start[b] + depth of n tokens.
int check_positions(const int32_t* start, const int32_t* depths_dev, const int32_t* depths_host,
                    const int32_t* counts_host, int64_t B, int64_t T, int64_t max_seq_len) {
    if (!depths_dev != !depths_host)
        return fail_format(NNE_EINVAL, NNE_BAD "depths are needed on the device and on the host");
    for (int64_t b = 0; b < B; ++b) {
        const int64_t n = count_of(counts_host, b, T);
        if (n == 0) continue;
        int64_t lo = 0, hi = n - 1;
        if (depths_host) {
            const auto mm = std::minmax_element(depths_host + b * T, depths_host + b * T + n);
            lo = *mm.first;
            hi = *mm.second;
        }
        if (start[b] + lo < 0 || start[b] + hi >= max_seq_len)   // llama.rs:131-139
            return fail_format(NNE_EINVAL, NNE_BAD "Sequence range [%lld, %lld) exceeds RoPE max_seq_len %lld",
                               (long long)(start[b] + lo), (long long)(start[b] + hi + 1), (long long)max_seq_len);
    }
    return NNE_OK;
}

int check_attention_heads(const nne_paged_cache_t* c, int64_t Hq, int64_t T) {
    if (Hq <= 0 || Hq > INT32_MAX || Hq % c->Hkv != 0)
        return fail_format(NNE_EINVAL, NNE_BAD "num_heads (%lld) must be divisible by num_kv_heads (%lld) for GQA",
                           (long long)Hq, (long long)c->Hkv);
    if (Hq / c->Hkv * T > INT32_MAX / 2)
        return fail_format(NNE_EINVAL, NNE_BAD "%lld query rows per KV head", (long long)(Hq / c->Hkv * T));
    return NNE_OK;
}

// Workspace of launches over the batch's groups of sequences, with T tokens.
nne_workspace_size_t attention_size(const nne_paged_cache_t* c, int64_t Hq, int64_t T) {
    const int64_t R = Hq / c->Hkv * T;
    const int64_t group = std::min<int64_t>(c->B, nne::kPagedSeqs), rest = c->B % nne::kPagedSeqs;
    const int cus = nne::cus_of_device();
    nne_workspace_size_t s;
    s.records_bytes = (uint64_t)std::max(nne::paged_record_bytes(group, c->Hkv, R, c->d, cus),
                                         rest ? nne::paged_record_bytes(rest, c->Hkv, R, c->d, cus) : 0);
    s.n_counters = (uint64_t)std::max<int64_t>(group * c->Hkv * ((R + 15) / 16), c->B);
    return s;
}

}  // namespace

extern "C" {

int nne_qk_norm_rope(const float* q, const int64_t q_shape[4], const int64_t q_strides[4], float* q_out,
                     const int64_t q_out_strides[4], const float* k, const int64_t k_shape[4],
                     const int64_t k_strides[4], float* k_out, const int64_t k_out_strides[4],
                     const float* q_weight, const float* k_weight, int has_norm, float eps,
                     const float* cos_table, const float* sin_table, int64_t max_seq_len, int64_t table_head_dim,
                     const int32_t* start_dev, const int32_t* start_host, const int32_t* depths_dev,
                     const int32_t* depths_host, void* stream) {
    if (!q_shape || (k && !k_shape))
        return fail_format(NNE_EINVAL, NNE_BAD "qk_norm_rope expects 4D tensors [Batch, Heads, SeqLen, HeadDim]");
    for (int i = 0; i < 4; ++i)
        if (q_shape[i] < 0 || q_shape[i] > INT32_MAX || (k && (k_shape[i] < 0 || k_shape[i] > INT32_MAX)))
            return fail_format(NNE_EINVAL, NNE_BAD "qk_norm_rope dims out of range");
    const int64_t B = q_shape[0], Hq = q_shape[1], T = q_shape[2], d = q_shape[3];
    const int64_t Hk = k ? k_shape[1] : 0;
    if (k && (k_shape[0] != B || k_shape[2] != T || k_shape[3] != d))
        return fail_format(NNE_ESHAPE, "Shape mismatch error: expected shape [%lld, %lld, %lld, %lld], got "
                           "[%lld, %lld, %lld, %lld]", (long long)B, (long long)Hk, (long long)T, (long long)d,
                           (long long)k_shape[0], (long long)k_shape[1], (long long)k_shape[2],
                           (long long)k_shape[3]);
    if (d % 2 != 0)
        return fail_format(NNE_EINVAL, NNE_BAD "qk_norm_rope head_dim (%lld) must be even", (long long)d);
    if (has_norm ? !(eps >= 0.f) : (q_weight || k_weight))
        return fail_format(NNE_EINVAL, NNE_BAD "qk_norm_rope: eps = %g, or weights without a norm", (double)eps);
    int rc = check_rotation(cos_table, sin_table, max_seq_len, table_head_dim, d);
    if (rc) return rc;
    if (B > INT32_MAX / std::max<int64_t>(T, 1) || Hq + Hk > INT32_MAX)
        return fail_format(NNE_EINVAL, NNE_BAD "qk_norm_rope dims out of range");
    if (B * T == 0 || Hq + Hk == 0 || d == 0) return NNE_OK;
    if (cos_table) {
        if (!start_host) return fail_format(NNE_EINVAL, NNE_BAD "start positions are null");
        rc = check_positions(start_host, depths_dev, depths_host, nullptr, B, T, max_seq_len);
        if (rc) return rc;
    }
    if ((Hq > 0 && (!q || !q_out)) || (Hk > 0 && !k_out) || (cos_table && !start_dev))
        return fail_format(NNE_EINVAL, NNE_BAD "null tensor pointer");
    const Strides qs(q_strides, B, Hq, T, d), qo(q_out_strides, B, Hq, T, d);
    const Strides ks(k_strides, B, Hk, T, d), ko(k_out_strides, B, Hk, T, d);
    nne::NormRopeParams p{};
    p.x[0] = view(q, qs.v);
    p.o[0] = out_view(q_out, qo.v);
    p.x[1] = view(k, ks.v);
    p.o[1] = out_view(k_out, ko.v);
    p.w[0] = q_weight;
    p.w[1] = k_weight;
    p.H[0] = (int)Hq;
    p.H[1] = (int)Hk;
    p.B = (int)B;
    p.T = (int)T;
    p.d = (int)d;
    p.by_heads = nne::divisor(Hq + Hk);
    p.by_t = nne::divisor(T);
    p.norm = has_norm != 0;
    p.eps = eps;
    p.cos = cos_table;
    p.sin = sin_table;
    p.max_seq_len = (int)max_seq_len;
    p.start = start_dev;
    p.depths = depths_dev;
    p.vec = vec_view(q, qs.v) && vec_view(q_out, qo.v) &&
            (Hk == 0 || (vec_view(k, ks.v) && vec_view(k_out, ko.v))) && aligned16(q_weight) &&
            aligned16(k_weight) && aligned16(cos_table) && aligned16(sin_table);
    const hipError_t e = nne::launch_qk_norm_rope(p, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? NNE_OK : nne::fail_hip(e, "head norm launch");
}

int nne_paged_append(const nne_paged_cache_t* cache, const float* k_new, const int64_t k_new_strides[4],
                     const float* v_new, const int64_t v_new_strides[4], int64_t T,
                     const int32_t* counts_dev, const int32_t* counts_host, const int32_t* depths_dev,
                     const int32_t* depths_host, const float* cos_table, const float* sin_table,
                     int64_t max_seq_len, int64_t table_head_dim, void* stream) {
    int rc = check_cache(cache, T);
    if (rc == NNE_OK) rc = check_counts(cache, T, counts_dev, counts_host);
    if (rc == NNE_OK) rc = check_room(cache, T, counts_host, NNE_ECAPACITY);
    if (rc == NNE_OK) rc = check_rotation(cos_table, sin_table, max_seq_len, table_head_dim, cache->d);
    if (rc) return rc;
    const int64_t B = cache->B;
    const int64_t per_token = cache->Hkv * (cache->d / 8);
    if (B > 0 && T > INT32_MAX / B / per_token)
        return fail_format(NNE_EINVAL, NNE_BAD "%lld tokens of %lld sequences: K may have 2^34 values", (long long)T,
                           (long long)B);
    if (B == 0 || T == 0) return NNE_OK;
    if (cos_table) {
        rc = check_positions(cache->lens_host, depths_dev, depths_host, counts_host, B, T, max_seq_len);
        if (rc) return rc;
    }
    if (cache->table_host) {
        std::vector<int32_t> pages;
        for (int64_t b = 0; b < B && rc == NNE_OK; ++b)
            rc = add_pages(cache, b, cache->lens_host[b], cache->lens_host[b] + count_of(counts_host, b, T), pages);
        if (rc == NNE_OK) rc = check_apart(pages);
        if (rc) return rc;
    }
    if (!k_new || !v_new) return fail_format(NNE_EINVAL, NNE_BAD "null tensor pointer");
    rc = check_device_side(cache);
    if (rc) return rc;
    const Strides ks(k_new_strides, B, cache->Hkv, T, cache->d), vs(v_new_strides, B, cache->Hkv, T, cache->d);
    nne::PagedAppendParams p{};
    p.k = view(k_new, ks.v);
    p.v = view(v_new, vs.v);
    p.pool = make_pool(cache);
    p.counts = counts_dev;
    p.depths = depths_dev;
    p.cos = cos_table;
    p.sin = sin_table;
    p.max_seq_len = (int)max_seq_len;
    p.B = (int)B;
    p.T = (int)T;
    p.by_token = nne::divisor(cache->Hkv * (cache->d / 8));
    p.by_row = nne::divisor(cache->d / 8);
    p.by_t = nne::divisor(T);
    p.vec = vec_view(k_new, ks.v) && vec_view(v_new, vs.v);
    if (cos_table && (!aligned16(cos_table) || !aligned16(sin_table)))
        return fail_format(NNE_EINVAL, NNE_BAD "RoPE tables must be 16-byte aligned");
    const hipError_t e = nne::launch_paged_append(p, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? NNE_OK : nne::fail_hip(e, "paged append launch");
}

int nne_paged_workspace_size(const nne_paged_cache_t* cache, int64_t Hq, int64_t T, nne_workspace_size_t* out) {
    if (!out) return fail_format(NNE_EINVAL, NNE_BAD "null output pointer");
    *out = nne_workspace_size_t{0, 0};
    int rc = check_cache(cache, T);
    if (rc == NNE_OK) rc = check_attention_heads(cache, Hq, T);
    if (rc) return rc;
    if (cache->B == 0 || T == 0) return NNE_OK;
    // Records grow with the tokens up to where launches no longer split: the most
    // that a step of T tokens or fewer needs is at the last that does.
    *out = attention_size(cache, Hq, T);
    for (int64_t lo = 1, hi = T; lo <= hi;) {
        const int64_t t = lo + (hi - lo) / 2;
        const nne_workspace_size_t s = attention_size(cache, Hq, t);
        out->records_bytes = std::max(out->records_bytes, s.records_bytes);
        if (s.records_bytes) lo = t + 1;
        else hi = t - 1;
    }
    return NNE_OK;
}

int nne_paged_attention(const nne_paged_cache_t* cache, const float* q, const int64_t q_strides[4], float* o,
                        const int64_t o_strides[4], int64_t Hq, int64_t T, const int32_t* counts_dev,
                        const int32_t* counts_host, const int32_t* parents_dev, const int32_t* parents_host,
                        int has_scale, float scale, const nne_workspace_t* ws, void* stream) {
    int rc = check_cache(cache, T);
    if (rc == NNE_OK) rc = check_attention_heads(cache, Hq, T);
    if (rc == NNE_OK) rc = check_counts(cache, T, counts_dev, counts_host);
    if (rc == NNE_OK) rc = check_room(cache, T, counts_host, NNE_EINVAL);
    if (rc) return rc;
    const int64_t B = cache->B, d = cache->d;
    if (!parents_dev != !parents_host)
        return fail_format(NNE_EINVAL, NNE_BAD "parents are needed on the device and on the host");
    if (parents_host && T > nne::kPagedTreeNodes)
        return fail_format(NNE_EINVAL, NNE_BAD "a tree has at most %d tokens, got %lld", nne::kPagedTreeNodes,
                           (long long)T);
    for (int64_t b = 0; parents_host && b < B; ++b)
        for (int64_t t = 0; t < count_of(counts_host, b, T); ++t)
            if (parents_host[b * T + t] < -1 || parents_host[b * T + t] >= t)
                return fail_format(NNE_EINVAL, NNE_BAD "token %lld of sequence %lld follows token %d: a parent "
                                   "comes before its children", (long long)t, (long long)b, parents_host[b * T + t]);
    if (cache->table_host)
        for (int64_t b = 0; b < B; ++b) {
            rc = check_pages(cache, b, 0, cache->lens_host[b] + count_of(counts_host, b, T));
            if (rc) return rc;
        }
    if (B == 0 || T == 0) return NNE_OK;
    if (!q || !o) return fail_format(NNE_EINVAL, NNE_BAD "null tensor pointer");
    rc = check_device_side(cache);
    if (rc) return rc;
    const Strides qs(q_strides, B, Hq, T, d), os(o_strides, B, Hq, T, d);
    nne::PagedAttnParams p{};
    p.q = view(q, qs.v);
    p.o = out_view(o, os.v);
    p.pool = make_pool(cache);
    p.counts = counts_dev;
    p.parents = parents_dev;
    p.G = (int)(Hq / cache->Hkv);
    p.T = (int)T;
    p.R = p.G * p.T;
    p.by_g = nne::divisor(p.G);
    p.by_hkv = nne::divisor(p.pool.Hkv);
    p.vec_q = vec_view(q, qs.v);
    p.vec_o = vec_view(o, os.v);
    p.qscale = (has_scale ? scale : 1.0f / std::sqrt((float)d)) * nne::kLog2e;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    // Launches of up to kPagedSeqs sequences, in stream order on one workspace.
    for (int64_t b0 = 0; b0 < B; b0 += nne::kPagedSeqs) {
        p.b0 = (int)b0;
        p.B = (int)std::min<int64_t>(nne::kPagedSeqs, B - b0);
        int64_t keys[nne::kPagedSeqs];
        for (int i = 0; i < p.B; ++i) {
            const int64_t n = count_of(counts_host, b0 + i, T);
            keys[i] = n > 0 ? cache->lens_host[b0 + i] + n : 1;
        }
        const int64_t n_records = nne::paged_plan(p, keys, nne::cus_of_device());
        p.ws = nullptr;
        p.cnt = nullptr;
        if (n_records > 0) {
            void* records = nullptr;
            const int64_t rec_bytes = 4 * nne::paged_record_floats(p.rec_rows, nne::paged_tile_dim((int)d));
            rc = nne::take_workspace(ws, (uint64_t)(n_records * rec_bytes),
                                     p.combine ? 0 : (int64_t)p.B * p.pool.Hkv * p.n_rb, s, &records, &p.cnt,
                                     "paged attention");
            if (p.combine) p.cnt = nullptr;
            if (rc) return rc;
            p.ws = static_cast<float*>(records);
        }
        const hipError_t e = nne::launch_paged_attention(p, s);
        if (e != hipSuccess) return nne::fail_hip(e, "paged attention launch");
    }
    return NNE_OK;
}

int nne_paged_commit(const nne_paged_cache_t* cache, int64_t n_layers, int64_t layer_stride,
                     const int32_t* counts_dev, const int32_t* counts_host, const int32_t* paths_dev,
                     const int32_t* paths_host, int64_t J, const nne_workspace_t* ws, void* stream) {
    int rc = check_cache(cache, J);
    if (rc) return rc;
    const int64_t B = cache->B, cap = cache->max_pages * cache->page_size;
    if (n_layers < 0 || n_layers > INT32_MAX || layer_stride < 0 ||
        (cache->dtype == NNE_BF16 ? layer_stride % 8 : layer_stride % 4) != 0)
        return fail_format(NNE_EINVAL, NNE_BAD "%lld layers %lld elements apart (16-byte multiples)",
                           (long long)n_layers, (long long)layer_stride);
    if (B == 0) return NNE_OK;
    if (!counts_host) return fail_format(NNE_EINVAL, NNE_BAD "counts_host is null");
    if (!paths_dev != !paths_host)
        return fail_format(NNE_EINVAL, NNE_BAD "paths are needed on the device and on the host");
    std::vector<int32_t> pages;
    for (int64_t b = 0; b < B; ++b) {
        const int64_t n = counts_dev ? counts_host[b] : counts_host[0];
        const int64_t len = cache->lens_host[b];
        if (n < 0 || n > J)
            return fail_format(NNE_EINVAL, NNE_BAD "counts[%lld] = %lld outside [0, %lld]", (long long)b,
                               (long long)n, (long long)J);
        int64_t last = n - 1;
        for (int64_t j = 0; paths_host && j < n; ++j) {
            const int64_t node = paths_host[b * J + j], before = j ? paths_host[b * J + j - 1] : -1;
            if (node <= before)
                return fail_format(NNE_EINVAL, NNE_BAD "path of sequence %lld does not ascend: %lld after %lld",
                                   (long long)b, (long long)node, (long long)before);
            last = node;
        }
        if (len < 0 || len + last + 1 > cap)
            return fail_format(NNE_EINVAL, NNE_BAD "row %lld of sequence %lld is past its %lld pages of %lld rows",
                               (long long)(len + last), (long long)b, (long long)cache->max_pages,
                               (long long)cache->page_size);
        rc = paths_host ? add_pages(cache, b, len, len + last + 1, pages) : check_pages(cache, b, len, len + last + 1);
        if (rc) return rc;
    }
    rc = check_apart(pages);
    if (rc) return rc;
    if (J == 0) return NNE_OK;
    rc = check_device_side(cache);
    if (rc) return rc;
    nne::PagedCommitParams p{};
    p.pool = make_pool(cache);
    p.layer_stride = layer_stride * (cache->dtype == NNE_BF16 ? 2 : 4);
    p.counts = counts_dev;
    p.paths = paths_dev;
    p.count = counts_dev ? 0 : counts_host[0];
    p.J = (int)J;
    p.B = (int)B;
    p.n_layers = (int)n_layers;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (paths_dev) {
        void* records = nullptr;
        rc = nne::take_workspace(ws, 0, B, s, &records, &p.cnt, "paged commit");
        if (rc) return rc;
    }
    const hipError_t e = nne::launch_paged_commit(p, s);
    if (e != hipSuccess) return nne::fail_hip(e, "paged commit launch");
    for (int64_t b = 0; b < B; ++b) cache->lens_host[b] += counts_dev ? counts_host[b] : counts_host[0];
    return NNE_OK;
}

}  // extern "C"
