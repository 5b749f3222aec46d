// Attention over a paged KV cache: a step's new tokens -- one, a chain, or a
// tree -- against their sequence's rows and the new ones on their path.
//
//   o[r] = sum_c 2^(s[r,c] - m[r]) v[c] / sum_c 2^(s[r,c] - m[r]),   any m[r],
//   s[r,c] = (scale log2(e) q[r]) . k[c] where r sees c, else -inf,
//
// in one pass over the keys, with m[r] kept above the scores seen so far.
//
// A KV head's G * T query rows (row r: token r / G of query head r % G) are the
// columns of MFMA tiles, its keys the rows:  S^T = K Q^T, O^T += V^T P^T.  Both
// products take K and V from registers as they come from memory, with no LDS:
//   * K: lane l (column l % 16, group g = l / 16) holds dims of key l % 16;
//     which dims sit in which step does not matter as long as Q agrees;
//   * S^T arrives as 4 keys (4 g + i) of row l % 16 per lane, which is how the
//     second product takes P^T, if its step pairs those keys: lane group g loads
//     V rows 4 g + i, and the lane's consecutive dims become the tiles' rows.
// f32 pools run on the f32 MFMAs (16x16x4, exact products, 16 keys a block).
// bf16 pools run on the bf16 MFMAs (16x16x32, 32 keys a block): K and V are
// exact there, Q and P are the exact sums of three bf16 parts, so products are
// exact and sums f32, at three MFMAs a product.  P's parts lose bits only of
// weights below 2^-110 of the row's largest.
//
// A workgroup is 4 waves that take blocks of its part of the keys in turn and
// meet only at the end.  Parts of a sequence (paged_plan.cpp) leave records that
// the last workgroup to arrive merges in the order of the parts, so results do
// not depend on who that is.
//
// Single tokens are bound by memory: 32 sequences of 512-4096 keys, 32 / 8 heads of
// 128 dims, take 107 us on an f32 pool (606 MB, 5.7 TB/s; a large copy runs at 4.9)
// and 59 on a bf16 one (5.1 TB/s); 5 tokens of 16 of them 37 us (4.1 TB/s).  Trees of
// many rows are bound by the matrix cores and what they wait for: 64 tokens of 8
// sequences of 1024-4096 keys take 80 us, 825 TFLOP/s of bf16 products (31 % of the
// MFMAs' cycles; a large library product of that type reaches 1146).  Two waves per
// SIMD is what the registers of 32 rows allow.  Bringing K to LDS in whole lines
// first was level (79 us), 128 rows per workgroup with K and V in LDS slower (99 us).
#include <algorithm>
#include <cstddef>
#include <type_traits>

#include "paged_device.hpp"
#include "paged_launch.hpp"

namespace nne {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

constexpr int kStage = 1024;     // keys whose pool rows are in LDS at a time
constexpr int kTable = 512;      // pages of a sequence whose table row goes to LDS whole
// A row's weights are taken relative to 2^8 times the largest so far (they cancel
// in the quotient), so that a larger one changes nothing until it passes that:
// nearly every block skips the scaling of O, and no weight is above 1.
constexpr float kSlack = 8.f;

__device__ __forceinline__ float row_groups_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    return pair_max(x);
}
__device__ __forceinline__ float row_groups_sum(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    return pair_sum(x);
}

__device__ __forceinline__ floatx4 mfma_part(uintx4 a, uintx4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <bool NT, typename V>
__device__ __forceinline__ V load_vec(const void* p) {
    if constexpr (NT) return __builtin_nontemporal_load(static_cast<const V*>(p));
    else return *static_cast<const V*>(p);
}

// 16- and 8-byte forms of store_coherent (buffer stores with the same policy).
__device__ __forceinline__ void store_coherent4(__amdgpu_buffer_rsrc_t range, uint32_t byte_offset, vf4 x) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uintx4, x), range, byte_offset, 0, 16);
}
__device__ __forceinline__ void store_coherent2(__amdgpu_buffer_rsrc_t range, uint32_t byte_offset, float x, float y) {
    __builtin_amdgcn_raw_buffer_store_b64(uintx2{__float_as_uint(x), __float_as_uint(y)}, range, byte_offset, 0, 16);
}

// What differs between the pools' types.  KB: keys of a block, JN: keys of a
// block per lane, VE: consecutive dims of a V load.
template <bool BF16, int D>
struct Shape {
    static constexpr int KB = BF16 ? 32 : 16;
    static constexpr int JN = KB / 4;
    static constexpr int VE = BF16 ? (D >= 128 ? 8 : 4) : 4;
    static constexpr int NV = D / (16 * VE);          // V loads per key
    static constexpr int KT = KB / 16;                // 16-key tiles
    static constexpr int KS = BF16 ? D / 32 : D / 16; // K loads per tile
    static constexpr int NO = D / 16;                 // 16-dim tiles of O
    static constexpr int ES = BF16 ? 2 : 4;           // bytes of an element
    static constexpr int QP = BF16 ? 3 : 1;           // parts of Q
};

// Key of a block that slot j of lane group g stands for.
template <bool BF16>
__device__ __forceinline__ int slot_key(int g, int j) {
    return BF16 ? 16 * (j >> 2) + 4 * g + (j & 3) : 4 * g + j;
}

// n / d for uniform n >= 0, d > 0 with a quotient below 2^16 (off by one at most
// before it is put right).
__device__ __forceinline__ int small_quotient(int n, int d) {
    int q = __builtin_amdgcn_readfirstlane((int)((float)n * __builtin_amdgcn_rcpf((float)d)));
    q -= q * (int64_t)d > n;
    q += (q + 1) * (int64_t)d <= n;
    return q;
}

__device__ __forceinline__ bool not_finite(float x) {
    return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
}

// Writes dims dd..dd+3 of row r of a KV head: O over the sum of weights, zeros
// where nothing was seen.
__device__ __forceinline__ void put_row4(const PagedAttnParams& p, int b, int h, int r, int count, int dd, vf4 x, float l) {
    const int t = quotient(r, p.by_g);
    if (t >= count) return;
    float* const out = p.o.p + b * p.o.sb + (h * p.G + r - t * p.G) * p.o.sh + t * p.o.st;
    x = l == 0.f ? vf4{0.f, 0.f, 0.f, 0.f} : x * (1.f / l);
    if (p.vec_o) {
        if (dd < p.pool.d) *reinterpret_cast<vf4*>(out + dd) = x;
    } else {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            if (dd + i < p.pool.d) out[(dd + i) * p.o.sd] = x[0];
            x = vf4{x[1], x[2], x[3], x[0]};
        }
    }
}

// Keys that some row of the block sees (0: none of its tokens exists).
__device__ __forceinline__ int block_keys(const PagedAttnParams& p, int row0, int n_rows, int len, int count) {
    if (quotient(row0, p.by_g) >= count) return 0;
    return len + (p.parents ? count : min(count, quotient(row0 + n_rows - 1, p.by_g) + 1));
}

// How many parts a (sequence, KV head, row block)'s keys are in, of how many keys
// (whole rounds of the waves), and where their records lie.  n: its parts as planned.
struct Parts {
    int live, length;
    int64_t rec0, rec_step;
};

__device__ __forceinline__ Parts even_parts(const PagedAttnParams& p, int before, int n, int h, int rb, int n_keys, int round) {
    Parts r;
    const int even = __builtin_amdgcn_readfirstlane((int)((float)n_keys * __builtin_amdgcn_rcpf((float)n) * 1.000002f));
    r.length = (even + round - 1) & ~(round - 1);
    if (r.length * (int64_t)n < n_keys) r.length += round;
    r.live = n_keys > 0 ? small_quotient(n_keys + r.length - 1, r.length) : 0;
    r.rec_step = p.pool.Hkv * p.n_rb;
    r.rec0 = ((int64_t)before * p.pool.Hkv + h) * p.n_rb + rb;
    return r;
}

// BF16: the pools' type.  D: dims, padded.  NRT: 16-row tiles of query rows.
// FULL: d == D.  NT: no other workgroup reads these keys.  DRAFT: T > 1, rows may see
// different keys (its masks cost a third wave per SIMD in registers, at 256 dims the
// second: 33 single tokens over 612 keys there 38.1 us with one wave, 37.2 with two).
template <bool BF16, int D, int NRT, bool FULL, bool NT, bool DRAFT>
__global__ __launch_bounds__(256, D > 128 ? (DRAFT ? 1 : 2) : DRAFT ? 2 : 3) void paged_attention_kernel(const PagedAttnParams p) {
    using S = Shape<BF16, D>;
    constexpr int KB = S::KB, JN = S::JN, VE = S::VE, NV = S::NV, KT = S::KT, KS = S::KS, NO = S::NO;
    constexpr int OS = D + 4;                        // row stride of the merge buffer
    constexpr int ROWS = 16 * NRT;

    // Q^T in operand order, [row tile][step][part][lane], until the last block;
    // then the waves' O.
    constexpr int QN = NRT * KS * S::QP * 64;
    constexpr int ON = 4 * 16 * OS / 4;
    __shared__ uintx4 smem[QN > ON ? QN : ON];
    float* const ob = reinterpret_cast<float*>(smem);
    __shared__ __attribute__((aligned(16))) uint32_t rows_s[kStage];   // 16-byte units from the pool
    __shared__ uint32_t gone_s[kStage / 32];     // keys without a row, a bit each
    __shared__ float ml_s[4][16][2];
    __shared__ uint32_t anc_s[kPagedTreeNodes][kPagedTreeNodes / 32];
    __shared__ int nxt_s[kPagedTreeNodes];
    __shared__ int table_s[kTable];
    __shared__ int last_s, odd_s;

    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Everything up to the first K and V is latency: one trip for the arguments,
    // one for the length, the page table and Q together, one for K and V.
    const int pref_lo = p.prefix[min(lane + 1, kPagedSeqs)], pref_hi = p.prefix[min(lane + 65, kPagedSeqs)];
    const int order_lo = p.order[lane], order_hi = p.order[lane + 64];
    warm_kernargs<0, sizeof(PagedAttnParams)>();
    asm volatile("" ::"v"(pref_lo), "v"(pref_hi), "v"(order_lo), "v"(order_hi));
    const PagedPool& pool = p.pool;

    // Workgroup -> (part of a sequence and KV head, row block).  With several row
    // blocks, the ones that read the same keys follow each other on one XCD
    // (workgroups go to the 8 XCDs in turn), whose L2 then serves them.
    int unit = blockIdx.x, rb = 0;
    if (p.n_rb > 1) {
        const int x = unit & 7, y = unit >> 3, z = quotient(y, p.by_rb);
        rb = y - z * p.n_rb;
        unit = z * 8 + x;
    }
    if (unit >= p.prefix[p.B] * pool.Hkv) return;
    const int part_all = quotient(unit, p.by_hkv), h = unit - part_all * pool.Hkv;
    const int place = __popcll(__builtin_amdgcn_ballot_w64(lane < p.B && pref_lo <= part_all)) +
                      __popcll(__builtin_amdgcn_ballot_w64(lane + 64 < p.B && pref_hi <= part_all));
    const int b = p.b0 + __builtin_amdgcn_readlane(place < 64 ? order_lo : order_hi, place & 63);
    const int row0 = rb * ROWS;
    const int n_rows = min(ROWS, p.R - row0);
    const int raw_len = pool.lens[b];
    const int count = paged_count(p.counts, b, p.T);
    const int32_t* const table = pool.table + (int64_t)b * pool.max_pages;
    const bool table_fits = pool.max_pages <= kTable;
    int page[kTable / 256];
#pragma unroll
    for (int i = 0; i < kTable / 256; ++i)
        page[i] = table_fits && tid + 256 * i < pool.max_pages ? table[tid + 256 * i] : -1;

    // Q^T, the second operand of S^T, scaled: 4 or 8 dims of a row per thread and
    // turn, every load issued before the first use.
    constexpr int QT = (NRT * KS * 64 + 255) / 256;
    vf4 qx[QT][BF16 ? 2 : 1];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        const int e = tid + 256 * i, qc = e & 15, qg = (e >> 4) & 3, st = (e >> 6) % KS, rt = (e >> 6) / KS;
        const bool rok = rt < NRT && 16 * rt + qc < n_rows;
        const int r = rok ? row0 + 16 * rt + qc : row0, t = quotient(r, p.by_g);
        const float* const qp = p.q.p + b * p.q.sb + (h * p.G + r - t * p.G) * p.q.sh + t * p.q.st;
#pragma unroll
        for (int y = 0; y < (BF16 ? 2 : 1); ++y) {
            const int c = BF16 ? 32 * st + 8 * qg + 4 * y : 16 * st + 4 * qg;
            vf4 x = vf4{0.f, 0.f, 0.f, 0.f};
            if (rok && (FULL || c < pool.d)) {
                if (p.vec_q) {
                    x = *reinterpret_cast<const vf4*>(qp + c);
                } else {
#pragma unroll 1
                    for (int k = 0; k < 4; ++k) x = vf4{x[1], x[2], x[3], qp[(c + k) * p.q.sd]};
                }
            }
            qx[i][y] = x;
        }
    }
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        const int e = tid + 256 * i;
        if (NRT * KS * 64 % 256 != 0 && e >= NRT * KS * 64) break;
        uintx4* const to = smem + (e >> 6) * S::QP * 64 + (e & 63);
        if constexpr (BF16) {
            const vf4 x = qx[i][0] * p.qscale, y = qx[i][1] * p.qscale;
            uint32_t w[3][4];
            split3(x[0], x[1], w[0][0], w[1][0], w[2][0]);
            split3(x[2], x[3], w[0][1], w[1][1], w[2][1]);
            split3(y[0], y[1], w[0][2], w[1][2], w[2][2]);
            split3(y[2], y[3], w[0][3], w[1][3], w[2][3]);
#pragma unroll
            for (int k = 0; k < 3; ++k) to[64 * k] = uintx4{w[k][0], w[k][1], w[k][2], w[k][3]};
        } else {
            *to = __builtin_bit_cast(uintx4, qx[i][0] * p.qscale);
        }
    }
#pragma unroll
    for (int i = 0; i < kTable / 256; ++i) table_s[tid + 256 * i] = page[i];

    // This part's keys, k0 to k1 of those that some row sees.
    const int len = paged_clamp(pool, raw_len);
    const int n_keys = block_keys(p, row0, n_rows, len, count);
    const Parts parts = even_parts(p, p.prefix[place], p.prefix[place + 1] - p.prefix[place], h, rb, n_keys, 4 * KB);
    const int part = part_all - p.prefix[place], live = parts.live;
    const int k0 = min(part * (int64_t)parts.length, (int64_t)n_keys);
    const int k1 = min((int64_t)n_keys, k0 + (int64_t)parts.length);
    if (k0 >= k1) return;
    int tok[NRT];                        // token of row col of tile rt
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) tok[rt] = quotient(min(row0 + 16 * rt + col, p.R - 1), p.by_g);

    if (tid == 0) odd_s = 0;             // (the stage's barriers follow)

    // Which drafted tokens precede a token: bit u of anc_s[t].  Pointer
    // doubling: after k rounds a row holds its 2^k nearest.
    if (DRAFT && p.parents && k1 > len) {
        constexpr int W = kPagedTreeNodes / 32;
        const int words = (p.T + 31) / 32;
        uint32_t own[W];
        int next = -1;
        if (tid < p.T) {
            next = p.parents[(int64_t)b * p.T + tid];
            if (next >= tid) next = -1;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) own[w] = w == tid >> 5 ? 1u << (tid & 31) : 0u;
        for (int span = 1;; span *= 2) {
#pragma unroll
            for (int w = 0; w < W; ++w)
                if (w < words) anc_s[tid][w] = own[w];
            nxt_s[tid] = next;
            __syncthreads();
            if (span >= p.T) break;
            const int at = next;
            if (at >= 0) {
#pragma unroll
                for (int w = 0; w < W; ++w)
                    if (w < words) own[w] |= anc_s[at][w];
                next = nxt_s[at];
            }
            __syncthreads();
        }
    }
    // Whether token t sees drafted token u (u < 0: a counted row).  Without
    // branches: lanes differ.
    auto sees = [&](int t, int u) __attribute__((always_inline)) -> bool {
        if (!p.parents) return u <= t;
        const int at = min(max(u, 0), kPagedTreeNodes - 1);
        return (u < 0) | (((anc_s[t][at >> 5] >> (at & 31)) & 1u) != 0);
    };

    // The same for drafted tokens u0, u0 + 1, ..., a bit each.
    auto sees_from = [&](int t, int u0) __attribute__((always_inline)) -> uint32_t {
        if (!p.parents) {
            const int n = t - u0 + 1;
            return n >= 32 ? ~0u : (1u << max(n, 0)) - 1u;
        }
        const int w = u0 >> 5;           // (uniform; u0 > -32)
        const uint32_t lo = w < 0 ? ~0u : anc_s[t][min(w, kPagedTreeNodes / 32 - 1)];
        const uint32_t hi = w + 1 < kPagedTreeNodes / 32 ? anc_s[t][w + 1] : 0u;
        return __builtin_amdgcn_alignbit(hi, lo, (uint32_t)u0 & 31u);
    };

    floatx4 o[NRT][NO];
    float m_run[NRT], l_run[NRT];
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
        m_run[rt] = kNegInf;
        l_run[rt] = 0.f;
#pragma unroll
        for (int c = 0; c < NO; ++c) o[rt][c] = floatx4{0.f, 0.f, 0.f, 0.f};
    }

    // Dims past d: any of the row's own (their Q is zero, their O is not kept).
    const auto clamp_dim = [&](int c) __attribute__((always_inline)) { return FULL || c < pool.d ? c : 0; };
    const char* const kbase = static_cast<const char*>(pool.k);
    const char* const vbase = static_cast<const char*>(pool.v);
    const uint32_t row_units = (uint32_t)pool.d * S::ES / 16;      // (the host keeps pools below 2^32 units)
    // A row's address: one shift-and-add where row numbers would take a 64-bit
    // multiplication (16 cycles a wave) for each of a block's rows.
    const auto row_at = [](const char* base, uint32_t at) __attribute__((always_inline)) { return base + ((uint64_t)at << 4); };
    typedef typename std::conditional<BF16 && VE == 4, uintx2, uintx4>::type VReg;

    for (int kc = k0; kc < k1; kc += kStage) {
        const int n_stage = min(kStage, k1 - kc);
        const int n_blocks = (n_stage + KB - 1) / KB;
        __syncthreads();                 // table_s is there; rows_s is done with
        for (int i = tid; i < n_blocks * KB; i += 256) {
            int row = -1;
            if (i < n_stage) row = table_fits ? paged_row(pool, table_s, h, kc + i) : paged_row(pool, table, h, kc + i);
            rows_s[i] = (uint32_t)max(row, 0) * row_units;           // (row 0 where there is none: not used)
            const uint64_t gone = __builtin_amdgcn_ballot_w64(row < 0);
            if ((lane & 31) == 0) gone_s[i >> 5] = (uint32_t)(gone >> (lane & 32));
        }
        __syncthreads();

        uintx4 kreg[KT][KS];
        VReg vreg[JN][NV];
        auto load_k = [&](int blk) __attribute__((always_inline)) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const char* row = row_at(kbase, rows_s[blk * KB + 16 * kt + col]);
#pragma unroll
                for (int s = 0; s < KS; ++s)
                    kreg[kt][s] = load_vec<false, uintx4>(row + S::ES * clamp_dim(BF16 ? 32 * s + 8 * g : 16 * s + 4 * g));
            }
        };
        auto load_v = [&](int blk) __attribute__((always_inline)) {
#pragma unroll
            for (int q = 0; q < JN / 4; ++q) {
                const uintx4 r4 = *reinterpret_cast<const uintx4*>(rows_s + blk * KB + 16 * q + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const char* row = row_at(vbase, r4[i]);
#pragma unroll
                    for (int c = 0; c < NV; ++c)
                        vreg[4 * q + i][c] = load_vec<NT, VReg>(row + S::ES * clamp_dim(16 * VE * c + VE * col));
                }
            }
        };

        int blk = wave;
        if (blk < n_blocks) {
            load_k(blk);
            load_v(blk);
        }
        for (; blk < n_blocks; blk += 4) {
            const int kb = kc + blk * KB;
            // ---- S^T = K Q^T (Q is read again for each block: held in registers
            // it would cost a wave per SIMD, so its address is kept from being hoisted)
            int qlane = lane;
            asm volatile("" : "+v"(qlane));
            floatx4 s[NRT][KT];
#pragma unroll
            for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) s[rt][kt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < KS; ++st)
#pragma unroll
                for (int rt = 0; rt < NRT; ++rt) {
                    const uintx4* const qa = smem + (rt * KS + st) * S::QP * 64 + qlane;
                    if constexpr (BF16) {
                        const uintx4 q2 = qa[128], q1 = qa[64], q0 = qa[0];
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) s[rt][kt] = mfma_part(kreg[kt][st], q2, s[rt][kt]);
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) s[rt][kt] = mfma_part(kreg[kt][st], q1, s[rt][kt]);
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) s[rt][kt] = mfma_part(kreg[kt][st], q0, s[rt][kt]);
                    } else {
                        const vf4 kv = __builtin_bit_cast(vf4, kreg[0][st]), qv = __builtin_bit_cast(vf4, *qa);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[rt][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv[i], qv[i], s[rt][0], 0, 0, 0);
                    }
                }
            // Q two steps ahead of the products: read where it is used, each step
            // waited for the LDS.
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * S::QP, 0);
#pragma unroll
            for (int i = 0; i < KS * NRT - 2; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, BF16 ? 3 * KT : 4, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, S::QP, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, BF16 ? 6 * KT : 8, 0);
            const bool more = blk + 4 < n_blocks;
            if (more) load_k(blk + 4);

            // ---- masks: only the last blocks have any
            const bool drafted = DRAFT && p.T > 1 && kb + KB > len;
            const uint32_t gone = (uint32_t)__builtin_amdgcn_readfirstlane((int)gone_s[blk * KB >> 5]) >> (blk * KB & 31);
            if (__builtin_expect((gone << (32 - KB)) != 0 || drafted, 0)) {
                // A word of bits per row tile, bit i for the block's key i, so that a
                // lane's keys are at constant places from 4 g on.
                int gm = g;              // (nothing of this is worth a register in the other blocks)
                asm volatile("" : "+v"(gm));
                const uint32_t there = ~gone >> (4 * gm);
                uint32_t ok[NRT];
#pragma unroll
                for (int rt = 0; rt < NRT; ++rt) ok[rt] = there;
                if (drafted)
#pragma unroll
                    for (int rt = 0; rt < NRT; ++rt) ok[rt] &= sees_from(tok[rt], kb - len) >> (4 * gm);
#pragma unroll
                for (int j = 0; j < JN; ++j) {
                    const int at = 31 - slot_key<BF16>(0, j);
#pragma unroll
                    for (int rt = 0; rt < NRT; ++rt) {
                        const uint32_t m = (uint32_t)((int)(ok[rt] << at) >> 31), x = __float_as_uint(s[rt][j >> 2][j & 3]);
                        s[rt][j >> 2][j & 3] = __uint_as_float((x & m) | (~m & 0xff800000u));     // (-infinity)
                    }
                    const uint32_t m = (uint32_t)((int)(there << at) >> 31);
#pragma unroll
                    for (int c = 0; c < NV; ++c)
#pragma unroll
                        for (int w = 0; w < (int)(sizeof(VReg) / 4); ++w) vreg[j][c][w] &= m;
                }
            }

            // ---- softmax: 2^(s - m), row col's other keys are in lanes l ^ 16, l ^ 32
            bool grow = false;
            float m_blk[NRT];
#pragma unroll
            for (int rt = 0; rt < NRT; ++rt) {
                float m = s[rt][0][0];
#pragma unroll
                for (int j = 1; j < JN; ++j) m = fmaxf(m, s[rt][j >> 2][j & 3]);
                m_blk[rt] = row_groups_max(m);
                grow |= m_blk[rt] > m_run[rt];
            }
            if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
                for (int rt = 0; rt < NRT; ++rt) {
                    const float m_new = m_blk[rt] > m_run[rt] ? m_blk[rt] + kSlack : m_run[rt];
                    const float alpha = fast_exp2(m_run[rt] - (m_new == kNegInf ? 0.f : m_new));
                    m_run[rt] = m_new;
                    l_run[rt] *= alpha;
#pragma unroll
                    for (int c = 0; c < NO; ++c) o[rt][c] *= alpha;
                }
            }
#pragma unroll
            for (int rt = 0; rt < NRT; ++rt) {
                const float m_use = m_run[rt] == kNegInf ? 0.f : m_run[rt];
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < JN; ++j) {
                    const float w = fast_exp2(s[rt][j >> 2][j & 3] - m_use);
                    s[rt][j >> 2][j & 3] = w;
                    sum += w;
                }
                l_run[rt] += sum;
            }

            // ---- where rows see different keys: a V that is not finite would
            // reach the rows that do not see it as 0 * inf.  Such values are taken
            // out here and added to the rows that see them at the end.
            if (__builtin_expect(drafted, 0)) {
                uint32_t fine = ~0u;
#pragma unroll
                for (int j = 0; j < JN; ++j) {
#pragma unroll
                    for (int c = 0; c < NV; ++c)
#pragma unroll
                        for (int w = 0; w < (int)(sizeof(VReg) / 4); ++w) {
                            // (all ones where the exponent is not: no comparison, whose
                            // results would take scalar registers)
                            const uint32_t x = vreg[j][c][w];
                            const uint32_t hi = (uint32_t)((int)((x & 0x7f800000u) - 0x7f800000u) >> 31);
                            const uint32_t lo = BF16 ? (uint32_t)((int)((x & 0x7f80u) - 0x7f80u) >> 31) : hi;
                            fine &= hi & lo;
                            vreg[j][c][w] = x & (BF16 ? (hi & 0xffff0000u) | (lo & 0xffffu) : hi);
                        }
                }
                if (fine != ~0u) odd_s = 1;
            }

            // ---- O^T += V^T P^T
            if constexpr (BF16) {
                uintx4 pb[NRT][3];
#pragma unroll
                for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t w0, w1, w2;
                        split3(s[rt][k >> 1][2 * (k & 1)], s[rt][k >> 1][2 * (k & 1) + 1], w0, w1, w2);
                        pb[rt][0][k] = w0;
                        pb[rt][1][k] = w1;
                        pb[rt][2][k] = w2;
                    }
                // Dims 2 c and 2 c + 1 of each load, two keys a register.
#pragma unroll
                for (int c = 0; c < NO; c += 2) {
                    uintx4 even, odd;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t x = vreg[2 * k][c / VE][(c % VE) / 2], y = vreg[2 * k + 1][c / VE][(c % VE) / 2];
                        even[k] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                        odd[k] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                    }
#pragma unroll
                    for (int i = 2; i >= 0; --i)
#pragma unroll
                        for (int rt = 0; rt < NRT; ++rt) {
                            o[rt][c] = mfma_part(even, pb[rt][i], o[rt][c]);
                            o[rt][c + 1] = mfma_part(odd, pb[rt][i], o[rt][c + 1]);
                        }
                }
            } else {
#pragma unroll
                for (int j = 0; j < JN; ++j)
#pragma unroll
                    for (int c = 0; c < NO; ++c) {
                        const float v = __builtin_bit_cast(vf4, vreg[j][c / 4])[c % 4];
#pragma unroll
                        for (int rt = 0; rt < NRT; ++rt)
                            o[rt][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, s[rt][0][j], o[rt][c], 0, 0, 0);
                    }
            }
            if (more) load_v(blk + 4);
        }
    }

    // ---- the 4 waves' (m, l, O), one tile of rows at a time
    const int64_t rec_floats = paged_record_floats(p.rec_rows, D);
    const int o_at = (2 * p.rec_rows + 3) & ~3;          // O of a record
    const __amdgpu_buffer_rsrc_t rec_range = coherent_range(p.ws + (parts.rec0 + part * parts.rec_step) * rec_floats,
                                                            live > 1 ? (uint32_t)rec_floats * 4u : 0u);
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
        if (16 * rt >= n_rows) break;
        const float l_all = row_groups_sum(l_run[rt]);
        __syncthreads();                 // Q, or the tile before, is done with
#pragma unroll
        for (int c = 0; c < NO; c += 4)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<vf4*>(ob + (wave * 16 + col) * OS + 16 * VE * (c / VE) + VE * (4 * g + i) + c % VE) =
                    vf4{o[rt][c][i], o[rt][c + 1][i], o[rt][c + 2][i], o[rt][c + 3][i]};
        if (g == 0) {
            ml_s[wave][col][0] = m_run[rt];
            ml_s[wave][col][1] = l_all;
        }
        __syncthreads();
        for (int f = tid; f < 16 * (D / 4); f += 256) {
            const int lr = f / (D / 4), dd = 4 * (f % (D / 4)), rr = 16 * rt + lr;
            if (rr >= n_rows) continue;
            float M = kNegInf;
#pragma unroll
            for (int w = 0; w < 4; ++w) M = fmaxf(M, ml_s[w][lr][0]);
            const float M_use = M == kNegInf ? 0.f : M;
            float l = 0.f;
            vf4 acc = vf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = fast_exp2(ml_s[w][lr][0] - M_use);
                l += f * ml_s[w][lr][1];
                acc += f * *reinterpret_cast<const vf4*>(ob + (w * 16 + lr) * OS + dd);
            }
            if (DRAFT && odd_s) {        // values that are not finite, for the rows that see them
                const int t = quotient(row0 + rr, p.by_g);
                for (int key = max(k0, len); key < k1; ++key) {
                    const int row = paged_row(pool, table, h, key);
                    if (row < 0 || !sees(t, key - len)) continue;
#pragma unroll 1
                    for (int i = 0; i < 4; ++i) {
                        const int64_t at = row * (int64_t)pool.d + clamp_dim(dd + i);
                        const float v = BF16 ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(vbase)[at] << 16)
                                             : reinterpret_cast<const float*>(vbase)[at];
                        if (not_finite(v)) acc[i] += v;
                    }
                }
            }
            if (live == 1) {
                put_row4(p, b, h, row0 + rr, count, dd, acc, l);
            } else {
                store_coherent4(rec_range, (uint32_t)(4 * (o_at + rr * D + dd)), acc);
                if (dd == 0) store_coherent2(rec_range, (uint32_t)(8 * rr), M, l);
            }
        }
    }
    if (live == 1 || !p.cnt) return;     // (without counters paged_combine_kernel merges)

    // ---- the last of the parts to arrive merges their records in order
    wait_stores_performed();
    __syncthreads();
    uint32_t* const cnt = p.cnt + ((int64_t)place * pool.Hkv + h) * p.n_rb + rb;
    if (tid == 0)
        last_s = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)live - 1;
    __syncthreads();
    if (!last_s) return;
    if (tid == 0) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // Each thread combines EV groups of 4 dims, with the loads of NR records of
    // all of them in flight (a trip to the coherence point is about 1.2 us: with 8
    // loads a trip the merge of 14 records of 32 rows took 13 us of a 26 us launch).
    constexpr int VPT = (ROWS * D / 4 + 255) / 256, EV = VPT < 4 ? VPT : 4, NR = (NRT == 1 ? 16 : 32) / EV;
    const uint32_t step = (uint32_t)(parts.rec_step * rec_floats * 4);     // bytes between two parts' records
    const __amdgpu_buffer_rsrc_t range = coherent_range(p.ws + parts.rec0 * rec_floats,
                                                        (uint32_t)(live - 1) * step + (uint32_t)rec_floats * 4u);
    for (int f0 = tid; f0 < n_rows * (D / 4); f0 += 256 * EV) {
        float M[EV], l[EV];
        vf4 acc[EV];
#pragma unroll
        for (int v = 0; v < EV; ++v) {
            M[v] = kNegInf;
            l[v] = 0.f;
            acc[v] = vf4{0.f, 0.f, 0.f, 0.f};
        }
        for (int c0 = 0; c0 < live; c0 += NR) {
            float2 ml[EV][NR];
            vf4 x[EV][NR];
#pragma unroll
            for (int c = 0; c < NR; ++c)
#pragma unroll
                for (int v = 0; v < EV; ++v) {       // (past the last record: zeros, without an access)
                    const int f = f0 + 256 * v, rr = f / (D / 4), dd = 4 * (f % (D / 4));
                    const uint32_t at = f < n_rows * (D / 4) ? (uint32_t)(c0 + c) * step : 0xfffffff0u - 4u * ROWS * (D + 2);
                    ml[v][c] = load_coherent2(range, at + 8u * rr);
                    x[v][c] = load_coherent4(range, at + 4u * (o_at + rr * D + dd));
                }
#pragma unroll
            for (int v = 0; v < EV; ++v) {
                float M_new = M[v];
#pragma unroll
                for (int c = 0; c < NR; ++c) {
                    ml[v][c].x = c0 + c < live ? ml[v][c].x : kNegInf;
                    M_new = fmaxf(M_new, ml[v][c].x);
                }
                const float M_use = M_new == kNegInf ? 0.f : M_new;
                const float old = fast_exp2(M[v] - M_use);
                l[v] *= old;
                acc[v] *= old;
                M[v] = M_new;
#pragma unroll
                for (int c = 0; c < NR; ++c) {
                    const float f = fast_exp2(ml[v][c].x - M_use);
                    l[v] += f * ml[v][c].y;
                    acc[v] += f * x[v][c];
                }
            }
        }
#pragma unroll
        for (int v = 0; v < EV; ++v) {
            const int f = f0 + 256 * v, rr = f / (D / 4), dd = 4 * (f % (D / 4));
            if (rr < n_rows) put_row4(p, b, h, row0 + rr, count, dd, acc[v], l[v]);
        }
    }
}

// Merges the records of a (sequence, KV head, row block), in the order of the
// parts: one thread per 4 dims of a row.  Behind launches whose merge is long:
// many records of many values, which one workgroup would be reading for longer than
// a launch takes (42 records of 8 rows of 256 dims: 21.4 us in all, 25.8 merged by
// the last to arrive).
template <int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(const PagedAttnParams p, int tile_rows) {
    int unit = blockIdx.x, rb = 0;
    if (p.n_rb > 1) {
        const int z = quotient(unit, p.by_rb);
        rb = unit - z * p.n_rb;
        unit = z;
    }
    const int place = quotient(unit, p.by_hkv), h = unit - place * p.pool.Hkv, b = p.b0 + p.order[place];
    const int ROUND = p.pool.bf16 ? 128 : 64, row0 = rb * tile_rows, n_rows = min(tile_rows, p.R - row0);
    const int count = paged_count(p.counts, b, p.T), len = paged_len(p.pool, b);
    const int n_keys = block_keys(p, row0, n_rows, len, count);
    const Parts parts = even_parts(p, p.prefix[place], p.prefix[place + 1] - p.prefix[place], h, rb, n_keys, ROUND);
    const int f = blockIdx.y * 256 + threadIdx.x, rr = f / (D / 4), dd = 4 * (f % (D / 4));
    if (parts.live <= 1 || rr >= n_rows) return;
    const int64_t rec_floats = paged_record_floats(p.rec_rows, D), step = parts.rec_step * rec_floats;
    const float* const rec = p.ws + parts.rec0 * rec_floats;
    const int o_at = (2 * p.rec_rows + 3) & ~3;
    constexpr int NR = 16;
    float M = kNegInf, l = 0.f;
    vf4 acc = vf4{0.f, 0.f, 0.f, 0.f};
    for (int c0 = 0; c0 < parts.live; c0 += NR) {
        vf2 ml[NR];
        vf4 x[NR];
#pragma unroll
        for (int c = 0; c < NR; ++c) {
            const float* const at = rec + min(c0 + c, parts.live - 1) * step;
            ml[c] = *reinterpret_cast<const vf2*>(at + 2 * rr);
            x[c] = *reinterpret_cast<const vf4*>(at + o_at + rr * D + dd);
        }
        float M_new = M;
#pragma unroll
        for (int c = 0; c < NR; ++c) M_new = fmaxf(M_new, ml[c][0]);
        const float M_use = M_new == kNegInf ? 0.f : M_new;
        const float old = fast_exp2(M - M_use);
        l *= old;
        acc *= old;
        M = M_new;
#pragma unroll
        for (int c = 0; c < NR; ++c) {
            const float w = c0 + c < parts.live ? fast_exp2(ml[c][0] - M_use) : 0.f;
            l += w * ml[c][1];
            acc += w * x[c];
        }
    }
    put_row4(p, b, h, row0 + rr, count, dd, acc, l);
}

template <bool BF16, int D, int NRT, bool NT, bool DRAFT>
hipError_t launch_tile(const PagedAttnParams& p, hipStream_t stream) {
    const int64_t units = (int64_t)p.prefix[p.B] * p.pool.Hkv;
    const int64_t wgs = p.n_rb > 1 ? (units + 7) / 8 * 8 * p.n_rb : units;
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    if (p.pool.d == D)
        hipLaunchKernelGGL((paged_attention_kernel<BF16, D, NRT, true, NT, DRAFT>), dim3((unsigned)wgs), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((paged_attention_kernel<BF16, D, NRT, false, NT, DRAFT>), dim3((unsigned)wgs), dim3(256), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.combine) return e;
    const int64_t all = (int64_t)p.B * p.pool.Hkv * p.n_rb;
    if (all > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL(paged_combine_kernel<D>, dim3((unsigned)all, (p.rec_rows * D / 4 + 255) / 256), dim3(256), 0,
                       stream, p, 16 * NRT);
    return hipGetLastError();
}

template <bool BF16, int D>
hipError_t launch_dim(const PagedAttnParams& p, hipStream_t stream) {
    // One row block: each byte of K and V is read by one workgroup, once (5 tokens of 16
    // sequences of 512-4096 keys, bf16: 37 us, 43 through the caches).
    const bool once = p.n_rb == 1;
    if (p.tile_rows == 32)
        return once ? launch_tile<BF16, D, 2, true, true>(p, stream) : launch_tile<BF16, D, 2, false, true>(p, stream);
    if (p.T == 1 && once) return launch_tile<BF16, D, 1, true, false>(p, stream);
    return once ? launch_tile<BF16, D, 1, true, true>(p, stream) : launch_tile<BF16, D, 1, false, true>(p, stream);
}

template <bool BF16>
hipError_t launch_type(const PagedAttnParams& p, hipStream_t stream) {
    switch (paged_tile_dim(p.pool.d)) {
    case 64: return launch_dim<BF16, 64>(p, stream);
    case 128: return launch_dim<BF16, 128>(p, stream);
    default: return launch_dim<BF16, 256>(p, stream);
    }
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttnParams& p, hipStream_t stream) {
    if (p.B <= 0 || p.R <= 0) return hipSuccess;
    return p.pool.bf16 ? launch_type<true>(p, stream) : launch_type<false>(p, stream);
}

}  // namespace nne
