// Paged KV cache: appending rows with the rotation on the way, committing the
// accepted path of a draft, and the norm of query and key heads with the
// rotation in the same pass.  All three are bound by memory where they are long
// and by latency where they are short; each is one launch that reads and writes
// every value once.
#include <algorithm>
#include <type_traits>

#include "paged_device.hpp"
#include "paged_launch.hpp"

namespace nne {

namespace {

// x * cos + rot * sin, each product and the sum rounded to f32 (the roundings
// of RotaryEmbedding::apply, llama.rs:154-156).
__device__ __forceinline__ float rotated(float x, float c, float rot, float s) {
#pragma clang fp contract(off)
    const float a = x * c;
    const float b = rot * s;
    return a + b;
}

__device__ __forceinline__ vf4 load_row4(const float* row, int64_t sd, int i, bool vec) {
    if (vec) return *reinterpret_cast<const vf4*>(row + i);
    return vf4{row[i * sd], row[(i + 1) * sd], row[(i + 2) * sd], row[(i + 3) * sd]};
}

// Rotates dims i..i+3 (a) and i + d/2.. (b) of a row with the table row.
template <bool VEC>
__device__ __forceinline__ void rotate4(vf4& a, vf4& b, const float* c, const float* s, int i, int half) {
    const vf4 c0 = load_row4(c, 1, i, VEC), s0 = load_row4(s, 1, i, VEC);
    const vf4 c1 = load_row4(c, 1, i + half, VEC), s1 = load_row4(s, 1, i + half, VEC);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float x = a[j], y = b[j];
        a[j] = rotated(x, c0[j], -y, s0[j]);
        b[j] = rotated(y, c1[j], x, s1[j]);
    }
}

// Four values into a pool row: as they are, or rounded to bf16 (to nearest,
// ties to even: the cache's one rounding).
template <bool BF16>
__device__ __forceinline__ void store_row4(void* pool, int64_t at, vf4 x) {
    if constexpr (BF16) {
        const uint2 v{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(pool) + at) = v;
    } else {
        *reinterpret_cast<vf4*>(static_cast<float*>(pool) + at) = x;
    }
}

// One thread: dims i..i+3 and d/2+i..d/2+i+3 of one new row of K and of V.
// Threads run through the dims, then the heads, of a token, so a wave writes
// whole rows.  Bound by memory where it is long: 2 x 2048 tokens of 8 heads of 128
// dims into a bf16 pool, 50 MB, take 10.9 us (4.6 TB/s); by its chain of loads
// (length, page, row) where it is short: 32 tokens 3.5 us.
template <bool BF16>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendParams p) {
    const int per_row = p.pool.d / 8, per_token = per_row * p.pool.Hkv;
    const uint32_t n = (uint32_t)p.B * p.T * per_token;       // (the host keeps this in 31 bits)
    const int half = p.pool.d / 2;
    for (uint32_t e = blockIdx.x * 256 + threadIdx.x; e < n; e += gridDim.x * 256) {
        const int token = quotient(e, p.by_token), in = e - token * per_token;
        const int h = quotient(in, p.by_row), i = 4 * (in - h * per_row);
        const int b = quotient(token, p.by_t), t = token - b * p.T;
        const float* kr = p.k.p + b * p.k.sb + h * p.k.sh + t * p.k.st;
        const float* vr = p.v.p + b * p.v.sb + h * p.v.sh + t * p.v.st;
        const bool vec = p.vec != 0;
        vf4 k0 = load_row4(kr, p.k.sd, i, vec), k1 = load_row4(kr, p.k.sd, i + half, vec);
        const vf4 v0 = load_row4(vr, p.v.sd, i, vec), v1 = load_row4(vr, p.v.sd, i + half, vec);
        const int count = paged_count(p.counts, b, p.T);
        const int len = paged_len(p.pool, b);
        if (t >= count) continue;
        const int row = paged_row(p.pool, p.pool.table + (int64_t)b * p.pool.max_pages, h, len + t);
        if (row < 0) continue;
        if (p.cos) {
            int pos = len + (p.depths ? p.depths[(int64_t)b * p.T + t] : t);
            pos = pos < 0 ? 0 : pos >= p.max_seq_len ? p.max_seq_len - 1 : pos;
            const int64_t at = (int64_t)pos * p.pool.d;
            rotate4<true>(k0, k1, p.cos + at, p.sin + at, i, half);
        }
        const int64_t at = (int64_t)row * p.pool.d + i;
        store_row4<BF16>(p.pool.k, at, k0);
        store_row4<BF16>(p.pool.k, at + half, k1);
        store_row4<BF16>(p.pool.v, at, v0);
        store_row4<BF16>(p.pool.v, at + half, v1);
    }
}

constexpr int kCommitRows = 8;     // rows a thread holds between loads and stores
constexpr int kCommitStage = 256;  // path entries in LDS at a time

// One thread: 16 bytes of every row of one layer's K or V and one head that
// moves.  Paths ascend with paths[j] >= j, so a row is read before a row of a
// lower number could be written over it: rows are read kCommitRows at a time,
// then written, in the order of j, by the one thread that owns these bytes.
// blockIdx.y is the sequence; where its rows lie is looked up once per workgroup
// (each lookup is a chain of two loads: eight in a row, one after the other in
// every thread, took most of the kernel's time), and the last of its workgroups
// to have read lens advances it.  Bound by memory: 32 layers of 8 heads of 16
// sequences, 4.5 rows in the mean, are 19 MB read and written in pieces of 256 bytes
// all over the pools, 11.6 us.
__global__ __launch_bounds__(256) void paged_commit_kernel(const PagedCommitParams p) {
    __shared__ int from_s[kCommitStage], to_s[kCommitStage];
    const int b = blockIdx.y, tid = threadIdx.x;
    const PagedPool& c = p.pool;
    const int32_t* table = c.table + (int64_t)b * c.max_pages;
    const int32_t* path = p.paths + (int64_t)b * p.J;
    int node = tid < p.J ? path[tid] : -1;
    const int len = paged_len(c, b);
    int count = p.counts ? p.counts[b] : p.count;
    count = count < 0 ? 0 : count > p.J ? p.J : count;

    const int vecs = c.d / (c.bf16 ? 8 : 4), in = blockIdx.x * 256 + tid;     // (the host keeps these in 31 bits)
    const int per_layer = 2 * c.Hkv * vecs, layer = in / per_layer, rest = in % per_layer;
    const int h = rest / vecs % c.Hkv;
    const int64_t row_bytes = 16ll * vecs;
    char* const at = static_cast<char*>(rest >= c.Hkv * vecs ? c.v : c.k) + layer * p.layer_stride +
                     (int64_t)h * c.page_size * row_bytes + 16 * (rest % vecs);
    const bool mine = layer < p.n_layers;
    uint32_t arrived = 0;
    for (int j0 = 0; j0 < count; j0 += kCommitStage) {
        const int n = min(kCommitStage, count - j0);
        if (j0 > 0) {
            __syncthreads();
            node = tid < n ? path[j0 + tid] : -1;
        }
        // (rows of head 0; -1: nothing moves)
        int from = -1, to = -1;
        if (tid < n && node > j0 + tid && node <= INT32_MAX - len) {
            from = paged_row(c, table, 0, len + node);
            to = paged_row(c, table, 0, len + j0 + tid);
        }
        from_s[tid] = to < 0 ? -1 : from;
        to_s[tid] = from < 0 ? -1 : to;
        __syncthreads();
        // Every thread of the workgroup has its len: it has arrived (the answer comes
        // while rows move).
        if (j0 == 0 && tid == 0)
            arrived = __hip_atomic_fetch_add(p.cnt + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int j = 0; mine && j < n; j += kCommitRows) {
            vf4 val[kCommitRows];
            int from8[kCommitRows], to8[kCommitRows];
#pragma unroll
            for (int i = 0; i < kCommitRows; ++i) {   // (kCommitRows divides kCommitStage)
                from8[i] = __builtin_amdgcn_readfirstlane(from_s[j + i]);
                to8[i] = __builtin_amdgcn_readfirstlane(to_s[j + i]);
            }
#pragma unroll
            for (int i = 0; i < kCommitRows; ++i)
                if (from8[i] >= 0) val[i] = *reinterpret_cast<const vf4*>(at + from8[i] * row_bytes);
#pragma unroll
            for (int i = 0; i < kCommitRows; ++i)
                if (to8[i] >= 0) *reinterpret_cast<vf4*>(at + to8[i] * row_bytes) = val[i];
        }
    }
    if (tid == 0) {
        if (count == 0) arrived = __hip_atomic_fetch_add(p.cnt + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (arrived == gridDim.x - 1) {
            p.pool.lens[b] = min(len + count, c.max_pages * c.page_size);
            __hip_atomic_store(p.cnt + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// Paths as they lie: only the lengths advance.
__global__ __launch_bounds__(256) void paged_advance_kernel(const PagedCommitParams p) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= p.B) return;
    int count = p.counts ? p.counts[b] : p.count;
    count = count < 0 ? 0 : count > p.J ? p.J : count;
    p.pool.lens[b] = min(paged_len(p.pool, b) + count, p.pool.max_pages * p.pool.page_size);
}

// Position of token t of sequence b in the rotary tables.
__device__ __forceinline__ int64_t norm_table_row(const NormRopeParams& p, int b, int t) {
    const int pos = p.start[b] + (p.depths ? p.depths[(int64_t)b * p.T + t] : t);
    return (int64_t)(pos < 0 ? 0 : pos >= p.max_seq_len ? p.max_seq_len - 1 : pos) * p.d;
}

// LPR lanes hold a head, 4 dims of each half per lane, so both values of a
// rotated pair are in one lane; the sum of squares takes log2(LPR) lane
// exchanges.  A head is read once and written once, and the memory bounds a long
// launch.  STREAM: the outputs are more than the L2s hold, and pass them by.  4
// sequences of 1999 tokens of 32 + 8 heads of 64 dims, 164 MB: 29 us (5.6 TB/s),
// 33 us without; 32 single tokens of 32 + 8 heads of 128 dims: 3.7 us.  VEC: every row
// is 16-byte vectors (the long launch at other addresses: 57 us).
template <int LPR, bool STREAM, bool VEC>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const NormRopeParams p) {
    const int heads = p.H[0] + p.H[1], half = p.d / 2;
    const uint32_t n = (uint32_t)p.B * p.T * heads;           // (the host keeps this in 31 bits)
    const int i = 4 * (threadIdx.x % LPR);
    const bool in = i < half;
    for (uint32_t r = blockIdx.x * (256 / LPR) + threadIdx.x / LPR; r < n; r += gridDim.x * (256 / LPR)) {
        const int token = quotient(r, p.by_heads);
        int h = r - token * heads;
        const int b = quotient(token, p.by_t), t = token - b * p.T;
        const int which = h >= p.H[0];
        if (which) h -= p.H[0];
        const View4 x = which ? p.x[1] : p.x[0];
        const float* row = x.p + b * x.sb + h * x.sh + t * x.st;
        vf4 y0 = vf4{0.f, 0.f, 0.f, 0.f}, y1 = y0;
        if (in) {
            y0 = load_row4(row, x.sd, i, VEC);
            y1 = load_row4(row, x.sd, i + half, VEC);
        }
        const int64_t tab = p.cos ? norm_table_row(p, b, t) : 0;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += y0[j] * y0[j] + y1[j] * y1[j];
#pragma unroll
        for (int m = 1; m < LPR; m <<= 1) sum += __shfl_xor(sum, m);
        const float scale = p.norm ? 1.0f / sqrtf(sum / (float)p.d + p.eps) : 1.f;
        if (!in) continue;
        const float* w = which ? p.w[1] : p.w[0];
        const vf4 one = vf4{1.f, 1.f, 1.f, 1.f};
        y0 = y0 * scale * (w ? load_row4(w, 1, i, VEC) : one);
        y1 = y1 * scale * (w ? load_row4(w, 1, i + half, VEC) : one);
        if (p.cos) rotate4<VEC>(y0, y1, p.cos + tab, p.sin + tab, i, half);
        const OutView4 o = which ? p.o[1] : p.o[0];
        float* out = o.p + b * o.sb + h * o.sh + t * o.st;
        if constexpr (!VEC) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                out[(i + j) * o.sd] = y0[j];
                out[(i + half + j) * o.sd] = y1[j];
            }
        } else if constexpr (STREAM) {
            __builtin_nontemporal_store(y0, reinterpret_cast<vf4*>(out + i));
            __builtin_nontemporal_store(y1, reinterpret_cast<vf4*>(out + i + half));
        } else {
            *reinterpret_cast<vf4*>(out + i) = y0;
            *reinterpret_cast<vf4*>(out + i + half) = y1;
        }
    }
}

// Any other even d: a wave per head, which reads it twice.
__global__ __launch_bounds__(256) void qk_norm_rope_any_kernel(const NormRopeParams p) {
    const int heads = p.H[0] + p.H[1], half = p.d / 2, lane = threadIdx.x & 63;
    const int64_t n = (int64_t)p.B * p.T * heads;
    for (int64_t r = (blockIdx.x * 256ll + threadIdx.x) / 64; r < n; r += gridDim.x * 4ll) {
        const int token = (int)(r / heads);
        int h = (int)(r % heads);
        const int b = token / p.T, t = token % p.T;
        const int which = h >= p.H[0];
        if (which) h -= p.H[0];
        const View4 x = which ? p.x[1] : p.x[0];
        const OutView4 o = which ? p.o[1] : p.o[0];
        const float* row = x.p + b * x.sb + h * x.sh + t * x.st;
        float* out = o.p + b * o.sb + h * o.sh + t * o.st;
        float sum = 0.f;
        for (int i = lane; i < p.d; i += 64) sum += row[i * x.sd] * row[i * x.sd];
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
        const float scale = p.norm ? 1.0f / sqrtf(sum / (float)p.d + p.eps) : 1.f;
        const float* w = which ? p.w[1] : p.w[0];
        const int64_t at = p.cos ? norm_table_row(p, b, t) : 0;
        for (int i = lane; i < half; i += 64) {
            const float a = row[i * x.sd] * scale * (w ? w[i] : 1.f);
            const float c = row[(i + half) * x.sd] * scale * (w ? w[i + half] : 1.f);
            float ra = a, rc = c;
            if (p.cos) {
                ra = rotated(a, p.cos[at + i], -c, p.sin[at + i]);
                rc = rotated(c, p.cos[at + i + half], a, p.sin[at + i + half]);
            }
            out[i * o.sd] = ra;
            out[(i + half) * o.sd] = rc;
        }
    }
}

constexpr int64_t kL2Bytes = int64_t{32} << 20;   // the L2s of 8 XCDs

unsigned grid_for(int64_t threads, int64_t most) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, most));
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendParams& p, hipStream_t stream) {
    const int64_t n = (int64_t)p.B * p.T * p.pool.Hkv * (p.pool.d / 8);
    if (n <= 0) return hipSuccess;
    const dim3 grid(grid_for(n, 1 << 20));
    if (p.pool.bf16) hipLaunchKernelGGL(paged_append_kernel<true>, grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(paged_append_kernel<false>, grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_paged_commit(const PagedCommitParams& p, hipStream_t stream) {
    if (p.B <= 0) return hipSuccess;
    if (!p.paths || p.J == 0 || p.n_layers == 0) {
        hipLaunchKernelGGL(paged_advance_kernel, dim3((p.B + 255) / 256), dim3(256), 0, stream, p);
        return hipGetLastError();
    }
    const int64_t n = 2ll * p.n_layers * p.pool.Hkv * (p.pool.d / (p.pool.bf16 ? 8 : 4));
    if (n > INT32_MAX - 256) return hipErrorInvalidValue;
    for (int b0 = 0; b0 < p.B; b0 += 32768) {     // grid.y is below 65536
        PagedCommitParams q = p;
        q.B = std::min(32768, p.B - b0);
        q.pool.table += (int64_t)b0 * p.pool.max_pages;
        q.pool.lens += b0;
        if (q.counts) q.counts += b0;
        q.paths += (int64_t)b0 * p.J;
        q.cnt += b0;
        hipLaunchKernelGGL(paged_commit_kernel, dim3((unsigned)((n + 255) / 256), q.B), dim3(256), 0, stream, q);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_qk_norm_rope(const NormRopeParams& p, hipStream_t stream) {
    const int64_t n = (int64_t)p.B * p.T * (p.H[0] + p.H[1]);
    if (n <= 0) return hipSuccess;
    const int64_t most = 1 << 20;
    if (p.d % 8 != 0 || p.d > 512 || n > INT32_MAX) {
        hipLaunchKernelGGL(qk_norm_rope_any_kernel, dim3(grid_for(n * 64, most)), dim3(256), 0, stream, p);
        return hipGetLastError();
    }
    const bool streams = n * p.d * 4 > kL2Bytes;
    const auto launch = [&](auto lpr) {
        constexpr int LPR = decltype(lpr)::value;
        const dim3 grid(grid_for(n * LPR, most));
        if (!p.vec) hipLaunchKernelGGL((qk_norm_rope_kernel<LPR, false, false>), grid, dim3(256), 0, stream, p);
        else if (streams) hipLaunchKernelGGL((qk_norm_rope_kernel<LPR, true, true>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((qk_norm_rope_kernel<LPR, false, true>), grid, dim3(256), 0, stream, p);
    };
    if (p.d <= 64) launch(std::integral_constant<int, 8>());
    else if (p.d <= 128) launch(std::integral_constant<int, 16>());
    else if (p.d <= 256) launch(std::integral_constant<int, 32>());
    else launch(std::integral_constant<int, 64>());
    return hipGetLastError();
}

}  // namespace nne
