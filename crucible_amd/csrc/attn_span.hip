// Windowed attention over the paged cache (span_attend.hpp): one new token a request, and chunks
// of rows packed back to back. No counterpart in the reference, whose rows see every earlier token.
//
// span_kernel: a workgroup takes 16 QB columns of one (request, KV head) over one split of the
// pages they see; its waves take pairs of pages in turn and merge through LDS. Where the splits are
// more than one, span_join_kernel joins them in a second launch: nothing has to be cleared or
// counted between calls, so a call's scratch can be any memory of its own.
// Bound: a launch and its chain of loads (lengths, table, keys and values) where the bytes are few,
// 5.5 us for one request behind a 256-token window; HBM where they are many, 53.5 us and a join of
// 4.8 for 32 requests of up to 4,100 visible tokens, 16 / 4 heads of 128: 264 MB, partly from the
// last-level cache, where a copy reaches 4.7 TB/s. 16 x 5 drafted rows over up to 258 pages, 33 MB,
// stay with the chain: 14.2 and 3.9 us.
#include <cmath>

#include "generic_attend.hpp"
#include "span_attend.hpp"

namespace crucible {
namespace {

struct SpanArgs {
    const void* q;
    const half_t* k_pool;
    const half_t* v_pool;
    void* out;
    const int32_t* tables;
    const int32_t* lens;      // one row a request, at position lens[b] - 1; or
    const int32_t* segments;  // {packed row, rows, first position, table}
    PoolAddr addr;
    SpanMask mask;
    int32_t n_head, n_kv_head, group, max_chunk, table_stride;
    int32_t max_seq;      // tokens that the grid's splits cover, within the table
    int32_t head_dim;
    int32_t n_tiles;      // column tiles of a (request, KV head)
    int32_t split_pages, n_splits;
    int32_t q_f32, out_f16;
    float scale_log2;
    float *po, *pm, *pl;  // partials [request][kv head][tile][split][column]; null: one split
    // weighing: scores in log2 units [request][query head][padded tokens], the pools they go to
    float* scores;
    int64_t score_stride;
    float* w_pool;
    int32_t* pos_pool;
    const int32_t* positions;
    int32_t n_layer, layer;
};

template <int QB>
struct SpanTile {
    int c0, n_cols, p0, p1;  // first column, columns, positions of the first and last row

    __device__ __forceinline__ SpanTile(const SpanArgs& a, const SpanRows& r, int tile) {
        c0 = tile * 16 * QB;
        n_cols = (int)min((int64_t)16 * QB, (int64_t)r.rows * a.group - c0);
        p0 = r.first + c0 / a.group;
        p1 = r.first + (c0 + n_cols - 1) / a.group;
    }
};

// Output offset of column c of a tile that starts at c0.
__device__ __forceinline__ int64_t column_row(const SpanArgs& a, const SpanRows& r, int g, int c, int hd) {
    return ((int64_t)(r.packed + c / a.group) * a.n_head + g * a.group + c % a.group) * hd;
}

__device__ __forceinline__ void store_one(const SpanArgs& a, int64_t at, float v) {
    if (a.out_f16)
        static_cast<half_t*>(a.out)[at] = (half_t)v;
    else
        static_cast<float*>(a.out)[at] = v;
}

__device__ __forceinline__ void store_four(const SpanArgs& a, int64_t at, float4_t v) {
    if (a.out_f16)
        *reinterpret_cast<half4_any_t*>(static_cast<half_t*>(a.out) + at) =
            half4_t{(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]};
    else
        *reinterpret_cast<float4_any_t*>(static_cast<float*>(a.out) + at) = v;
}

// The columns of `bad`, again: their outputs are not finite, by what they see or by a masked value
// that met a weight of 0.
__device__ void redo_columns(RowLds& lds, const SpanArgs& a, const SpanRows& r, const int g, const int c0,
                             const uint64_t bad, const int hd) {
    for (uint64_t left = bad; left; left &= left - 1) {
        const int c = c0 + __builtin_ctzll(left);
        const int64_t at = column_row(a, r, g, c, hd);
        const void* q = static_cast<const char*>(a.q) + at * (a.q_f32 ? 4 : 2);
        span_row(lds, q, a.q_f32, a.k_pool, a.v_pool, a.addr, r.table, g, hd, a.mask, r.first + c / a.group,
                 a.scale_log2, [&](int d, float v) { store_one(a, at + d, v); });
    }
}

// (m, l) of two disjoint sets of keys, as one; w, v: what sums under the first and the second are
// worth in it.
__device__ __forceinline__ float join_max(float m, float n, float& w, float& v) {
    const float mx = fmaxf(m, n), at = mx == -INFINITY ? 0.0f : mx;
    w = fast_exp2(m - at);
    v = fast_exp2(n - at);
    return mx;
}

// The waves' states of one column block, which meet in LDS.
template <int HD, int W>
struct MergeLds {
    alignas(16) float o[W][16][HD + 4];  // the columns start in different banks
    float m[W][16], l[W][16];
};

template <int HD, bool PAD, bool F32, int QB, bool WEIGH>
__global__ __launch_bounds__(64 * hd_waves(HD)) void span_kernel(SpanArgs a) {
    constexpr int W = hd_waves(HD);
    __shared__ union {
        MergeLds<HD, W> merge;
        RowLds row;
    } lds;
    __shared__ uint32_t bad_cols[QB];
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = blockIdx.x, b = blockIdx.z;
    const int g = blockIdx.y / a.n_tiles, tile = blockIdx.y % a.n_tiles;
    const SpanRows r(a, b);
    const SpanTile<QB> t(a, r, tile);
    if (t.n_cols <= 0) return;
    const SpanPages sp(a.mask, t.p0, t.p1);
    const int i0 = split * a.split_pages, n = min(a.split_pages, sp.count - i0);  // pages of the split
    if (n <= 0 && split > 0) return;
    // page ids of the split, one a lane, 64 at a time
    int id = 0;
    if (lane < n) id = r.table[sp.page(i0 + lane)];
    if (threadIdx.x < QB) bad_cols[threadIdx.x] = 0;

    const SpanDim<HD, PAD> dim{a.head_dim};
    const int head_off = g * dim.hd(), kv_dim = a.addr.kv_dim;
    // Keys and values of the pair at hand. Both are loaded as soon as their registers are free:
    // the next keys before the softmax, the next values after the products with the last.
    SpanKeys<HD, PAD> ks;
    SpanValues<HD, PAD> vs;
    int idx0, idx1;
    int64_t base0, base1;
    const auto find = [&](int i) {
        if (i >= 64 && (i & 63) == 2 * wave) {
            const int next = (i & ~63) + lane;
            if (next < n) id = r.table[sp.page(i0 + next)];
        }
        const bool two = i + 1 < n;
        idx0 = sp.page(i0 + i);
        idx1 = two ? sp.page(i0 + i + 1) : 0x7fffff0;  // past every row
        base0 = block_base(a.addr, __builtin_amdgcn_readlane(id, i & 63));
        base1 = two ? block_base(a.addr, __builtin_amdgcn_readlane(id, (i & 63) + 1)) : base0;
    };
    int i = 2 * wave;
    if (i < n) {
        find(i);
        ks.load(dim, a.k_pool, col >= 8 ? base1 : base0, kv_dim, head_off, col, grp);
        vs.load(dim, a.v_pool, grp >= 2 ? base1 : base0, head_off, col, grp);
    }
    HdQuery<HD, F32> q[QB];
    int pos[QB];
#pragma unroll
    for (int k = 0; k < QB; ++k) {
        const int c = 16 * k + col;
        const bool on = c < t.n_cols;
        span_query(q[k], dim, a.q, on ? column_row(a, r, g, t.c0 + c, dim.hd()) : 0, on, grp, a.scale_log2);
        pos[k] = on ? r.first + (t.c0 + c) / a.group : -1;
    }
    HdState<HD> st[QB];
#pragma unroll
    for (int k = 0; k < QB; ++k) st[k].clear();

    while (i < n) {
        const int key = (grp >= 2 ? idx1 : idx0) * kPageTokens + 8 * (grp & 1);
        const int64_t base = grp >= 2 ? base1 : base0;
        // every row sees both pages?
        const auto whole = [&](int idx) {
            const int j = idx * kPageTokens;
            return j + kPageMask <= t.p0 && (j + kPageMask < a.mask.n_sink || t.p1 - j < a.mask.window);
        };
        const bool masked = !(whole(idx0) && whole(idx1));
        float4_t s[QB][2];
#pragma unroll
        for (int k = 0; k < QB; ++k) {
            span_scores(s[k], q[k], ks);
            if constexpr (WEIGH)
                span_exact_scores(s[k], q[k], dim, a.q, a.k_pool, base, kv_dim, head_off, pos[k] >= 0,
                                  column_row(a, r, g, t.c0 + 16 * k + col, dim.hd()), grp, a.scale_log2, F32);
        }
        const bool held = i + 1 < n || grp < 2;
        i += 2 * W;
        if (i < n) {
            find(i);
            ks.load(dim, a.k_pool, col >= 8 ? base1 : base0, kv_dim, head_off, col, grp);
        }
        if (masked) vs.zero_unseen(a.mask, sp, t.p1, key);
#pragma unroll
        for (int k = 0; k < QB; ++k) {
            if (masked) span_mask(s[k], a.mask, pos[k], key);
            span_accumulate(st[k], s[k], q[k].scale, vs);
            if constexpr (WEIGH)
                if (pos[k] >= 0 && held) {
                    float* to = a.scores + ((int64_t)b * a.n_head + g * a.group + t.c0 + col) * a.score_stride + key;
                    *reinterpret_cast<float4_t*>(to) = s[k][0];
                    *reinterpret_cast<float4_t*>(to + 4) = s[k][1];
                }
        }
        if (i < n) vs.load(dim, a.v_pool, grp >= 2 ? base1 : base0, head_off, col, grp);
    }

    // The waves meet, one column block at a time: every thread joins 4 dimensions of a column.
    const int64_t unit = (((int64_t)b * a.n_kv_head + g) * a.n_tiles + tile) * a.n_splits + split;
#pragma unroll
    for (int k = 0; k < QB; ++k) {
        const int cols = min(16, t.n_cols - 16 * k);
        if (cols <= 0) break;
        if (k > 0) __syncthreads();
        const float l_wave = group_sum4(st[k].l);
        if (col < cols) {
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
                *reinterpret_cast<float4_t*>(&lds.merge.o[wave][col][16 * d + 4 * grp]) = st[k].o[d];
            if (grp == 0) {
                lds.merge.m[wave][col] = st[k].m;
                lds.merge.l[wave][col] = l_wave;
            }
        }
        __syncthreads();
        for (int x = threadIdx.x; x < cols * (HD / 4); x += 64 * W) {
            const int c = x / (HD / 4), d = 4 * (x % (HD / 4));
            float m = lds.merge.m[0][c];
#pragma unroll
            for (int w = 1; w < W; ++w) m = fmaxf(m, lds.merge.m[w][c]);
            const float at = m == -INFINITY ? 0.0f : m;
            float l = 0.0f;
            float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float f = fast_exp2(lds.merge.m[w][c] - at);
                const float4_t y = *reinterpret_cast<const float4_t*>(&lds.merge.o[w][c][d]);
                l = __builtin_fmaf(lds.merge.l[w][c], f, l);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(y[e], f, o[e]);
            }
            if (a.po) {
                const int64_t to = unit * 16 * QB + 16 * k + c;
                *reinterpret_cast<float4_t*>(a.po + to * HD + d) = o;
                if (d == 0) {
                    a.pm[to] = m;
                    a.pl[to] = l;
                }
                continue;
            }
            const float z = (o[0] * 0.0f + o[1] * 0.0f) + (o[2] * 0.0f + o[3] * 0.0f) + l * 0.0f;
            if (!(z == 0.0f)) atomicOr(&bad_cols[k], 1u << c);
            else if (dim.has(d))
                store_four(a, column_row(a, r, g, t.c0 + 16 * k + c, dim.hd()) + d, o * (l == 0.0f ? 0.0f : 1.0f / l));
        }
    }
    if (a.po) return;
    __syncthreads();
    uint64_t bad = 0;
#pragma unroll
    for (int k = 0; k < QB; ++k) bad |= (uint64_t)bad_cols[k] << (16 * k);
    if (bad) redo_columns(lds.row, a, r, g, t.c0, bad, dim.hd());
}

// ---------------------------------------------------------------- many rows
//
// span_tile_kernel: for chunks whose rows fill the chip by themselves. A workgroup of four waves
// takes 128 columns, 32 a wave, over every page they see; keys and values pass through LDS, where
// each byte serves the four waves, in the order in which the lanes want them as operands: a
// direct-to-LDS load a fragment, 16 bytes a lane, read back without bank conflicts. Three stages of
// 32 or 64 keys: one is computed on, the next is there or on its way, the third is being loaded;
// one barrier a stage.
//
// Bound by the vector units: 8 scores a lane and 16 columns cost 8 exponentials (a quarter of the
// rate), 8 FMAs, 7 maxima and 12 operations for fp16 hi and lo, against 10 products of 16 cycles at
// head_dim 64. So the running maximum moves, and sums are rescaled, only when a score passes it by
// more than 2^kLazy (weights up to 256 are fine in fp16 hi + lo), and the sum of weights comes from
// a product with ones. 8,192 rows behind a 1,024-token window, 12 / 3 heads of 64: 57 us, 420
// TFLOP/s of the formula's products; on a SIMD 65,000 cycles of vector issue and 42,000 of products,
// which barely overlap.
constexpr int kTileWaves = 4, kTileQb = 2, kTileColumns = 16 * kTileQb * kTileWaves;
constexpr float kLazy = 8.0f;

template <int HD>
constexpr int tile_pairs() {  // of a stage
    return HD <= 32 ? 4 : HD <= 64 ? 2 : 1;
}

template <int HD, bool PAD, bool F32>
__global__ __launch_bounds__(64 * kTileWaves, HD <= 64 ? 3 : 2) void span_tile_kernel(SpanArgs a) {
    constexpr int QB = kTileQb, NP = tile_pairs<HD>(), KF = 2 * (HD / 32), VF = HD / 16, PF = KF + VF;
    constexpr int FW = NP * PF / kTileWaves;  // fragments of a stage that a wave loads
    static_assert(NP * PF % kTileWaves == 0, "");
    __shared__ union {
        half8_t stage[3][NP * PF][64];
        RowLds row;
    } lds;
    __shared__ uint32_t bad_cols[kTileWaves * QB];
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.z, g = blockIdx.y, tile = blockIdx.x / a.n_splits, split = blockIdx.x % a.n_splits;
    const SpanRows r(a, b);
    const SpanTile<QB * kTileWaves> t(a, r, tile);
    if (t.n_cols <= 0) return;
    const SpanPages sp(a.mask, t.p0, t.p1);
    const int first = split * a.split_pages;  // of the list
    const int n = min(a.split_pages, sp.count - first), stages = (n + 2 * NP - 1) / (2 * NP);
    if (n <= 0 && split > 0) return;
    const SpanDim<HD, PAD> dim{a.head_dim};
    const int head_off = g * dim.hd(), kv_dim = a.addr.kv_dim;
    const uint32_t lds0 = lds_offset(&lds.stage[0][0][0]);
    // A wave loads FW fragments of one pair of the stage: at these places of the pages' blocks, keys
    // from the page that row `col` lies in, values from the one that the lane group covers.
    static_assert(PF % FW == 0, "");
    const int pair_of = wave * FW / PF, f0 = wave * FW % PF;
    int off[FW];
    bool is_v[FW];
#pragma unroll
    for (int x = 0; x < FW; ++x) {
        const int w = f0 + x;
        is_v[x] = w >= KF;
        if (!is_v[x]) {
            const int d = 32 * (w % (HD / 32)) + 8 * grp;
            const int slot = 8 * ((col >> 2) & 1) + (col & 3) + 4 * (w / (HD / 32));
            off[x] = slot * kv_dim + head_off + (dim.has(d) ? d : 0);
        } else {
            const int d = 16 * (w - KF) + col;
            off[x] = (head_off + (dim.has(d) ? d : 0)) * kPageTokens + 8 * (grp & 1);
        }
    }
    // block offsets of pages id_at .. + 63 of the split, one a lane
    uint32_t lo = 0, hi = 0;
    int id_at = -64;
    const auto issue = [&](int s) {
        const int i0 = 2 * NP * s;
        if (i0 >= id_at + 64) {  // stages divide 64 pages
            id_at = i0 & ~63;
            if (id_at + lane < n) {
                const int64_t base = block_base(a.addr, r.table[sp.page(first + id_at + lane)]);
                lo = (uint32_t)base;
                hi = (uint32_t)(base >> 32);
            }
        }
        // past the split: its last page again, masked
        const int i = min(i0 + 2 * pair_of, n - 1) - id_at, j = min(i0 + 2 * pair_of + 1, n - 1) - id_at;
        const uint32_t lo0 = __builtin_amdgcn_readlane(lo, i), hi0 = __builtin_amdgcn_readlane(hi, i);
        const uint32_t lo1 = __builtin_amdgcn_readlane(lo, j), hi1 = __builtin_amdgcn_readlane(hi, j);
        const int64_t kb = (int64_t)((uint64_t)(col >= 8 ? hi1 : hi0) << 32 | (col >= 8 ? lo1 : lo0));
        const int64_t vb = (int64_t)((uint64_t)(grp >= 2 ? hi1 : hi0) << 32 | (grp >= 2 ? lo1 : lo0));
        const uint32_t to = lds0 + (uint32_t)(((s % 3) * NP * PF + wave * FW) * 64 * sizeof(half8_t));
#pragma unroll
        for (int x = 0; x < FW; ++x)
            lds_dma16((is_v[x] ? a.v_pool + vb : a.k_pool + kb) + off[x], to + x * 64 * (uint32_t)sizeof(half8_t));
    };
    if (stages > 0) issue(0);

    HdQuery<HD, F32> q[QB];
    int pos[QB];
    const int w0 = 32 * wave;  // the wave's first column of the tile
#pragma unroll
    for (int k = 0; k < QB; ++k) {
        const int c = w0 + 16 * k + col;
        const bool on = c < t.n_cols;
        span_query(q[k], dim, a.q, on ? column_row(a, r, g, t.c0 + c, dim.hd()) : 0, on, grp, a.scale_log2);
        pos[k] = on ? r.first + (t.c0 + c) / a.group : -1;
    }
    // positions of the wave's first and last row
    const int wp0 = r.first + (t.c0 + min(w0, t.n_cols - 1)) / a.group;
    const int wp1 = w0 < t.n_cols ? r.first + (t.c0 + min(w0 + 31, t.n_cols - 1)) / a.group : -1;
    // The pages of the split that all of its rows see whole: [plain0, plain1), of the windows' part.
    const int plain0 = sp.n_head - first + max(0, ((max(wp1 - a.mask.window, -1) + kPageTokens) >> kPageShift) - sp.first);
    const int plain1 = wp1 < 0 ? 0 : min(n, sp.n_head - first + ((wp0 + 1) >> kPageShift) - sp.first);
    HdState<HD> st[QB];
    float4_t sum[QB];
#pragma unroll
    for (int k = 0; k < QB; ++k) {
        st[k].clear();
        sum[k] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    half8_t ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = (half_t)1.0f;

    if (stages > 1) issue(1);
    for (int s = 0; s < stages; ++s) {
        // this stage's fragments have arrived, the wave's own and, past the barrier, everyone's; and
        // everyone is done with the stage before, whose place the one after next takes
        if (s + 1 < stages)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(FW) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s + 2 < stages) issue(s + 2);
#pragma unroll
        for (int pair = 0; pair < NP; ++pair) {
            const int i = 2 * NP * s + 2 * pair;
            if (i >= n) break;
            int key = 0;
            bool masked = false;
            if (i < plain0 || i + 2 > plain1) {
                const int j0 = sp.page(first + i) * kPageTokens;
                const int j1 = i + 1 < n ? sp.page(first + i + 1) * kPageTokens : 0x7fffff00;  // past every row
                const auto none = [&](int j) {
                    return j > wp1 || (j >= a.mask.n_sink && wp0 - (j + kPageMask) >= a.mask.window);
                };
                if (none(j0) && none(j1)) continue;
                masked = true;
                key = (grp >= 2 ? j1 : j0) + 8 * (grp & 1);
            }
            const half8_t* f = &lds.stage[s % 3][pair * PF][lane];
            SpanKeys<HD, PAD> ks;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int x = 0; x < HD / 32; ++x) ks.k[u][x] = f[64 * (u * (HD / 32) + x)];
            float4_t sc[QB][2];
#pragma unroll
            for (int k = 0; k < QB; ++k) span_scores(sc[k], q[k], ks);
            SpanValues<HD, PAD> vs;
#pragma unroll
            for (int x = 0; x < VF; ++x) vs.v[x] = f[64 * (KF + x)];
            if (masked) {
                vs.zero_unseen(a.mask, sp, t.p1, key);
#pragma unroll
                for (int k = 0; k < QB; ++k) span_mask(sc[k], a.mask, pos[k], key);
            }
            // one branch for all blocks, so that the products of one fill the waits of another
            float mx[QB];
            bool past = false;
#pragma unroll
            for (int k = 0; k < QB; ++k) {
                mx[k] = fmaxf(sc[k][0][0], sc[k][0][1]);
#pragma unroll
                for (int e = 2; e < 8; ++e) mx[k] = fmaxf(mx[k], sc[k][e >> 2][e & 3]);
                past = past || mx[k] * q[k].scale > st[k].m + kLazy;
            }
            if (__ballot(past)) {
#pragma unroll
                for (int k = 0; k < QB; ++k) {
                    const float mn = fmaxf(st[k].m, group_max4(mx[k]) * q[k].scale);
                    const float alpha = fast_exp2(st[k].m - (mn == -INFINITY ? 0.0f : mn));
                    st[k].m = mn;
                    sum[k] *= alpha;
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d) st[k].o[d] *= alpha;
                }
            }
#pragma unroll
            for (int k = 0; k < QB; ++k) {
                const float at = st[k].m == -INFINITY ? 0.0f : st[k].m;
                u32x4_t hw, lw;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float pf[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) pf[e] = fast_exp2(__builtin_fmaf(sc[k][u][e], q[k].scale, -at));
                    const uint32_t h01 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(pf[0], pf[1]));
                    const uint32_t h23 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(pf[2], pf[3]));
                    uint32_t l01, l23;
                    split_lo4(pf, h01, h23, l01, l23);
                    hw[2 * u] = h01;
                    hw[2 * u + 1] = h23;
                    lw[2 * u] = l01;
                    lw[2 * u + 1] = l23;
                }
                const half8_t ph = __builtin_bit_cast(half8_t, hw), pl = __builtin_bit_cast(half8_t, lw);
                sum[k] = mfma_16x16x32(ones, ph, sum[k]);
                sum[k] = mfma_16x16x32(ones, pl, sum[k]);
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) {
                    st[k].o[d] = mfma_16x16x32(vs.v[d], ph, st[k].o[d]);
                    st[k].o[d] = mfma_16x16x32(vs.v[d], pl, st[k].o[d]);
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < QB; ++k) {
        const int c = w0 + 16 * k + col;
        const bool on = c < t.n_cols;
        st[k].l = sum[k][0];
        if (a.po) {
            if (!on) continue;
            const int64_t unit = (((int64_t)b * a.n_kv_head + g) * a.n_tiles + tile) * a.n_splits + split;
            const int64_t to = unit * kTileColumns + c;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
                *reinterpret_cast<float4_t*>(a.po + to * HD + 16 * i + 4 * grp) = st[k].o[i];
            if (grp == 0) {
                a.pm[to] = st[k].m;
                a.pl[to] = st[k].l;
            }
            continue;
        }
        const uint32_t bad = hd_not_finite(st[k], on);
        if (lane == 0) bad_cols[QB * wave + k] = bad;
        if (!on || (bad >> col & 1)) continue;
        const float inv = st[k].l == 0.0f ? 0.0f : 1.0f / st[k].l;
        const int64_t at = column_row(a, r, g, t.c0 + c, dim.hd());
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
            if (dim.has(16 * i + 4 * grp)) store_four(a, at + 16 * i + 4 * grp, st[k].o[i] * inv);
    }
    if (a.po) return;
    __syncthreads();
    for (int k = 0; k < QB * kTileWaves; ++k)
        if (bad_cols[k]) redo_columns(lds.row, a, r, g, t.c0 + 16 * k, bad_cols[k], dim.hd());
}

// Joins the splits of up to C columns of a tile, from column cb of it, with HD / 4 threads a column.
// Where the columns are fewer, several threads share the splits of one and meet in LDS: a join waits
// for loads, and this way fewer follow each other.
template <int HD>
struct JoinLds {
    static constexpr int C = kRowThreads / (HD / 4);
    float4_t o[C][HD / 4];
    float m[C], l[C];
    uint32_t bad;
};

template <int HD, int QB>
__device__ void join_columns(RowLds& row_lds, JoinLds<HD>& lds, const SpanArgs& a, const SpanRows& r, int b, int g,
                             int tile, int cb) {
    constexpr int T = HD / 4, C = JoinLds<HD>::C;
    const SpanTile<QB> t(a, r, tile);
    if (cb >= t.n_cols) return;
    if (threadIdx.x == 0) lds.bad = 0;
    const SpanPages sp(a.mask, t.p0, t.p1);
    const int n = (sp.count + a.split_pages - 1) / a.split_pages;
    const int cols = min(C, t.n_cols - cb), parts = C / cols;
    const int i = threadIdx.x / T, d = 4 * (threadIdx.x % T), part = i / cols;
    const int cl = i % cols, c = cb + cl;
    const bool on = part < parts;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;
    if (on) {
        const int64_t unit = (((int64_t)b * a.n_kv_head + g) * a.n_tiles + tile) * a.n_splits;
        constexpr int U = 4;  // splits on their way at a time
        for (int s0 = part; s0 < n; s0 += U * parts) {
            float pm[U], pl[U];
            float4_t po[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = s0 + u * parts;
                const int64_t k = (unit + min(s, n - 1)) * 16 * QB + c;
                pm[u] = s < n ? a.pm[k] : -INFINITY;
                pl[u] = s < n ? a.pl[k] : 0.0f;
                po[u] = s < n ? *reinterpret_cast<const float4_t*>(a.po + k * HD + d) : float4_t{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float w, v;
                m = join_max(m, pm[u], w, v);
                l = __builtin_fmaf(pl[u], v, l * w);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(po[u][e], v, o[e] * w);
            }
        }
        if (parts > 1) {
            lds.o[i][d / 4] = o;
            if (d == 0) {
                lds.m[i] = m;
                lds.l[i] = l;
            }
        }
    }
    __syncthreads();
    const bool mine = on && part == 0;
    if (mine) {
        for (int j = 1; j < parts; ++j) {
            const int k = j * cols + cl;
            const float4_t po = lds.o[k][d / 4];
            float w, v;
            m = join_max(m, lds.m[k], w, v);
            l = __builtin_fmaf(lds.l[k], v, l * w);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(po[e], v, o[e] * w);
        }
        const float z = (o[0] * 0.0f + o[1] * 0.0f) + (o[2] * 0.0f + o[3] * 0.0f) + l * 0.0f;
        if (!(z == 0.0f)) atomicOr(&lds.bad, 1u << cl);
    }
    __syncthreads();
    const uint32_t bad = lds.bad;
    if (mine && d < a.head_dim && !(bad >> cl & 1))
        store_four(a, column_row(a, r, g, t.c0 + c, a.head_dim) + d, o * (l == 0.0f ? 0.0f : 1.0f / l));
    if (bad) redo_columns(row_lds, a, r, g, t.c0 + cb, bad, a.head_dim);
}

template <int HD, int QB>
__global__ __launch_bounds__(kRowThreads) void span_join_kernel(SpanArgs a) {
    __shared__ RowLds row_lds;
    __shared__ JoinLds<HD> lds;
    const SpanRows r(a, blockIdx.z);
    join_columns<HD, QB>(row_lds, lds, a, r, blockIdx.z, blockIdx.y / a.n_tiles, blockIdx.y % a.n_tiles,
                         blockIdx.x * JoinLds<HD>::C);
}

// The second launch of a weighing call, one new token a request. The first workgroups of a (request,
// KV head) take kRowThreads tokens each: the weights that the group's heads gave them go to the
// pool, the newest token's as its first. The others join the output. The first launch leaves the
// scores, 4 bytes a head and token against 4 head_dim of K and V a KV head, as weights need the row's
// maximum and sum. 16 requests of up to 2,048 tokens, 12 / 3 heads of 64: 8.3 and 4.4 us; 4 of up
// to 32,768, 16 / 4 of 128, 253 MB: 53.8 and 10.1, 84% of a copy's rate over both.
template <int HD>
__global__ __launch_bounds__(kRowThreads) void weigh_join_kernel(SpanArgs a, int token_blocks) {
    constexpr int kHeads = 64, kAhead = 4;
    __shared__ RowLds row_lds;
    __shared__ JoinLds<HD> lds;
    __shared__ float sm[kHeads], sl[kHeads];
    const int b = blockIdx.z, g = blockIdx.y;
    const SpanRows r(a, b);
    if (r.rows <= 0) return;
    if ((int)blockIdx.x >= token_blocks) {
        constexpr int C = JoinLds<HD>::C, N = (16 + C - 1) / C;
        const int i = blockIdx.x - token_blocks;
        join_columns<HD, 1>(row_lds, lds, a, r, b, g, i / N, i % N * C);
        return;
    }
    const int p = r.first, t = threadIdx.x, lane = t & 63, j = blockIdx.x * kRowThreads + t;
    if ((int)blockIdx.x * kRowThreads > p) return;
    const int n = (p / kPageTokens + a.split_pages) / a.split_pages;
    const float* scores = a.scores + ((int64_t)b * a.n_head + g * a.group) * a.score_stride + j;
    // what does not wait for the maxima: the first heads' scores, the old sum
    float ahead[kAhead];
    float old = 0.0f;
    int64_t at = 0;
    if (j <= p) {
#pragma unroll
        for (int h = 0; h < kAhead; ++h) ahead[h] = h < a.group ? scores[h * a.score_stride] : 0.0f;
        const int64_t page = r.table[j >> kPageShift];
        at = ((page * a.n_layer + a.layer) * a.n_kv_head + g) * kPageTokens + (j & kPageMask);
        if (j < p) old = a.w_pool[at];
    }
    float sum = 0.0f;
    for (int h0 = 0; h0 < a.group; h0 += kHeads) {
        const int heads = min(kHeads, a.group - h0);
        __syncthreads();
        for (int h = t >> 6; h < heads; h += kRowThreads / 64) {  // a wave a head, a lane a split
            const int c = h0 + h;
            const int64_t k = ((((int64_t)b * a.n_kv_head + g) * a.n_tiles + c / 16) * a.n_splits) * 16 + c % 16;
            float m = -INFINITY, l = 0.0f, w, v;
            for (int s = lane; s < n; s += 64) {
                m = join_max(m, a.pm[k + 16 * s], w, v);
                l = __builtin_fmaf(a.pl[k + 16 * s], v, l * w);
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) {
                const float m2 = __shfl_xor(m, d), l2 = __shfl_xor(l, d);
                m = join_max(m, m2, w, v);
                l = __builtin_fmaf(l2, v, l * w);
            }
            if (lane == 0) {
                sm[h] = m == -INFINITY ? 0.0f : m;
                sl[h] = l == 0.0f ? 0.0f : 1.0f / l;
            }
        }
        __syncthreads();
        if (j <= p) {
            if (h0 == 0) {
#pragma unroll
                for (int h = 0; h < kAhead; ++h)
                    if (h < heads) sum = __builtin_fmaf(fast_exp2(ahead[h] - sm[h]), sl[h], sum);
            }
            for (int h = h0 == 0 ? kAhead : 0; h < heads; ++h)
                sum = __builtin_fmaf(fast_exp2(scores[(h0 + h) * a.score_stride] - sm[h]), sl[h], sum);
        }
    }
    if (j > p) return;
    a.w_pool[at] = j == p ? sum : old + sum;
    if (j == p) a.pos_pool[at] = a.positions[b];
}

// ---------------------------------------------------------------- launches

struct SpanShape {
    int qb, n_tiles, split_pages, n_splits;
    int64_t partials;  // floats; 0: none
};

// Columns of a tile: as few 16-column blocks as hold a request's rows, at most what the registers
// take beside a pair of pages.
int span_qb(int64_t columns, int64_t hd) {
    const int most = hd <= 64 ? 4 : hd <= 128 ? 2 : 1;
    int qb = 1;
    while (qb < most && 16 * qb < columns) qb *= 2;
    return qb;
}

// head_dim as the kernels' operands hold it.
int64_t span_wide(int64_t hd) { return (hd + 31) / 32 * 32; }

bool span_shape(SpanShape& s, int64_t requests, int64_t max_chunk, int64_t n_head, int64_t n_kv_head, int64_t hd,
                int64_t table_pages, int64_t window, int64_t n_sink, bool weigh) {
    const int64_t columns = checked_mul(max_chunk, n_head / n_kv_head);
    if (columns < 0) return false;
    const int64_t cus = device_cu_count();
    // More columns than a span_kernel tile holds: tiles of 128. us against span_kernel, 12 / 3 heads
    // of 64: 1,500 rows 37 / 62, 4,000 rows 111 / 124, behind a 256-token window 27 / 50, 8 x 40 rows
    // behind histories 33 / 32; 16 / 4 heads of 128: 4,000 rows 200 / 241, but 300 rows 24 / 19.
    if (!weigh && span_wide(hd) <= 128 && columns > 16 * span_qb(columns, span_wide(hd))) {
        s.qb = kTileQb * kTileWaves;
        const int64_t tiles = (columns + kTileColumns - 1) / kTileColumns;
        const int64_t units = checked_mul(requests, n_kv_head, tiles);
        const int64_t rows = (kTileColumns + n_head / n_kv_head - 1) / (n_head / n_kv_head) + 1;
        const int64_t pages = span_pages_bound(window, n_sink, rows, table_pages);
        if (units < 0 || tiles * n_kv_head > 65535 || requests > 65535) return false;
        // Splits as many as the workgroups that the registers let a CU hold, of 32 pages at least.
        // us without / with them, launch overhead included, 12 / 3 heads of 64: 512 rows behind
        // 12,000 tokens 195 / 55, 2,048 rows there 198 / 136, 1,500 rows alone 46 / 37, 4,000 rows
        // 134 / 111; 300 rows, 19 pages, stay at 19.
        const int64_t slots = (span_wide(hd) <= 64 ? 3 : 2) * cus;
        const int64_t n = units < slots ? slots / units : 1;
        int64_t sp = ((pages + n - 1) / n + 7) / 8 * 8;  // whole stages
        sp = sp < 32 ? 32 : sp;
        s.n_tiles = (int)tiles;
        s.split_pages = (int)sp;
        s.n_splits = (int)((pages + sp - 1) / sp);
        s.partials = s.n_splits > 1 ? checked_mul(units, s.n_splits, kTileColumns * (span_wide(hd) + 2)) : 0;
        return s.partials >= 0 && s.partials <= INT64_MAX / 8 && tiles * s.n_splits <= INT32_MAX;
    }
    s.qb = weigh ? 1 : span_qb(columns, span_wide(hd));
    const int64_t tiles = (columns + 16 * s.qb - 1) / (16 * s.qb);
    const int64_t tile_rows = (16 * s.qb + n_head / n_kv_head - 1) / (n_head / n_kv_head) + 1;
    const int64_t pages = span_pages_bound(window, n_sink, tile_rows, table_pages);
    const int64_t units = checked_mul(requests, n_kv_head, tiles);
    if (units < 0 || tiles * n_kv_head > 65535 || requests > 65535) return false;
    s.n_tiles = (int)tiles;
    const int waves = hd_waves((int)span_wide(hd));
    // Splits of 2 to 6 steps of what the waves take at once, or none, by what they cost in steps: the
    // CUs take a workgroup each, round after round, a round costs its steps and one to start (its
    // chain of loads), and a join 1.75. Not more than 6, as lengths may be far below their bound; one
    // split where the units alone fill the chip twice. us for splits of 2 / 3 / 4 / 5 / 6 / 9 / 17
    // steps, launch overhead included, windows of 258 pages (17: one split): 128 units of 128 dims
    // 61.7 / 57.6 / 62.3 / 57.7 / 61.3 / 55.3 / 63.9, 80 units 40.8 / 38.0 / 42.0 / 48.7 / 36.3 /
    // 42.2 / 58.3, 192 units 88 / 86 / 87 / 85 / 86 / 91 / 77; 72 units of 64 dims 19.7 / 17.9 /
    // 20.1 / 23.0 / 17.7 / 19.6 / 25.7, 16 x 5 drafted rows 22.3 / 20.9 / 16.6 / 18.2 / 19.5 / 24.3 /
    // 31.3; weighing 16 requests of up to 128 pages 14.3 / 14.4 / 14.6 / 16.2 / 17.7 / 19.9 / 19.8.
    const int64_t step = 2 * waves;
    int64_t sp = pages;
    if (units < 2 * cus) {
        const auto rounds = [&](int64_t n) { return (units * n + cus - 1) / cus; };
        // in quarters of a step
        int64_t least = 4 * rounds(1) * pages / step + (weigh ? 4 * rounds(1) + 7 : 0);
        for (int64_t k = 2; k <= 6 && k * step < pages; ++k) {
            const int64_t cost = 4 * rounds((pages + k * step - 1) / (k * step)) * (k + 1) + 7;
            if (cost <= least) {
                least = cost;
                sp = k * step;
            }
        }
    }
    s.split_pages = (int)sp;
    s.n_splits = (int)((pages + sp - 1) / sp);
    s.partials = 0;
    if (weigh || s.n_splits > 1) {
        s.partials = checked_mul(units, s.n_splits, 16 * s.qb * (span_wide(hd) + 2));
        if (s.partials < 0 || s.partials > INT64_MAX / 8) return false;
    }
    return true;
}

template <int HD, bool PAD, bool F32, int QB>
void launch_tiles(const SpanArgs& a, int requests, hipStream_t stream) {
    const dim3 grid((unsigned)a.n_splits, (unsigned)(a.n_kv_head * a.n_tiles), (unsigned)requests);
    if constexpr (QB == 1) {
        if (a.scores) {
            hipLaunchKernelGGL((span_kernel<HD, PAD, F32, 1, true>), grid, dim3(64 * hd_waves(HD)), 0, stream, a);
            constexpr int C = JoinLds<HD>::C, N = (16 + C - 1) / C;
            const int blocks = (int)((a.score_stride + kRowThreads - 1) / kRowThreads);
            const dim3 join((unsigned)(blocks + N * a.n_tiles), (unsigned)a.n_kv_head, grid.z);
            hipLaunchKernelGGL((weigh_join_kernel<HD>), join, dim3(kRowThreads), 0, stream, a, blocks);
            return;
        }
    }
    hipLaunchKernelGGL((span_kernel<HD, PAD, F32, QB, false>), grid, dim3(64 * hd_waves(HD)), 0, stream, a);
    if (a.n_splits > 1) {
        constexpr int C = JoinLds<HD>::C;
        const dim3 join((16 * QB + C - 1) / C, grid.y, grid.z);
        hipLaunchKernelGGL((span_join_kernel<HD, QB>), join, dim3(kRowThreads), 0, stream, a);
    }
}

template <int HD, bool PAD, bool F32>
void launch_qb(const SpanArgs& a, int qb, int requests, hipStream_t stream) {
    if constexpr (HD <= 128) {
        if (qb == kTileQb * kTileWaves) {
            const dim3 grid((unsigned)(a.n_tiles * a.n_splits), (unsigned)a.n_kv_head, (unsigned)requests);
            hipLaunchKernelGGL((span_tile_kernel<HD, PAD, F32>), grid, dim3(64 * kTileWaves), 0, stream, a);
            if (a.n_splits > 1) {
                constexpr int QB = kTileQb * kTileWaves, C = JoinLds<HD>::C;
                const dim3 join((16 * QB + C - 1) / C, (unsigned)(a.n_kv_head * a.n_tiles), grid.z);
                hipLaunchKernelGGL((span_join_kernel<HD, QB>), join, dim3(kRowThreads), 0, stream, a);
            }
            return;
        }
    }
    constexpr int M = HD <= 64 ? 4 : HD <= 128 ? 2 : 1;
    if (qb == 1) return launch_tiles<HD, PAD, F32, 1>(a, requests, stream);
    if (qb == 2) return launch_tiles<HD, PAD, F32, M >= 2 ? 2 : 1>(a, requests, stream);
    return launch_tiles<HD, PAD, F32, M>(a, requests, stream);
}

template <int HD>
void launch_hd(const SpanArgs& a, int qb, int requests, hipStream_t stream) {
    if (a.head_dim == HD)
        a.q_f32 ? launch_qb<HD, false, true>(a, qb, requests, stream)
                : launch_qb<HD, false, false>(a, qb, requests, stream);
    else
        a.q_f32 ? launch_qb<HD, true, true>(a, qb, requests, stream)
                : launch_qb<HD, true, false>(a, qb, requests, stream);
}

int check_span(const char* what, int q_dtype, int out_dtype, int64_t requests, int64_t max_chunk, int64_t n_head,
               int64_t n_kv_head, int64_t head_dim, int64_t table_stride, int64_t kv_dim, int64_t window,
               int64_t n_sink) {
    CRUCIBLE_CHECK(dtype_ok(q_dtype) && dtype_ok(out_dtype), CRUCIBLE_ERR_INVALID, "%s: bad dtype", what);
    CRUCIBLE_CHECK(requests >= 0 && requests <= 65535 && max_chunk >= 0 && max_chunk <= INT32_MAX &&
                       table_stride > 0 && table_stride <= kMaxTablePages,
                   CRUCIBLE_ERR_INVALID, "%s: requests=%lld rows=%lld table_stride=%lld", what,
                   (long long)requests, (long long)max_chunk, (long long)table_stride);
    CRUCIBLE_CHECK(n_head > 0 && n_kv_head > 0 && n_head <= (1 << 20) && n_head % n_kv_head == 0,
                   CRUCIBLE_ERR_INVALID, "%s: n_head %lld must be a positive multiple of n_kv_head %lld", what,
                   (long long)n_head, (long long)n_kv_head);
    CRUCIBLE_CHECK(generic_head_dim_ok(head_dim), CRUCIBLE_ERR_UNSUPPORTED,
                   "%s: head_dim %lld unsupported (a multiple of 8 up to 256)", what, (long long)head_dim);
    CRUCIBLE_CHECK(kv_dim == n_kv_head * head_dim, CRUCIBLE_ERR_INVALID,
                   "%s: kv_dim %lld != n_kv_head * head_dim", what, (long long)kv_dim);
    CRUCIBLE_CHECK(window >= 0 && window <= INT32_MAX && n_sink >= 0 && n_sink <= INT32_MAX - kPageTokens,
                   CRUCIBLE_ERR_INVALID, "%s: window=%lld n_sink=%lld", what, (long long)window,
                   (long long)n_sink);
    return CRUCIBLE_OK;
}

size_t span_workspace(int64_t requests, int64_t max_chunk, int64_t n_head, int64_t n_kv_head, int64_t head_dim,
                      int64_t table_pages, int64_t window, int64_t n_sink, bool weigh = false) {
    if (requests <= 0 || max_chunk <= 0 || n_head <= 0 || n_head > (1 << 20) || n_kv_head <= 0 ||
        n_head % n_kv_head ||
        !generic_head_dim_ok(head_dim) || table_pages <= 0 || window < 0 || n_sink < 0)
        return 0;
    SpanShape s;
    if (!span_shape(s, requests, max_chunk, n_head, n_kv_head, head_dim, table_pages, window, n_sink, weigh))
        return 0;
    const int64_t scores = weigh ? checked_mul(requests * n_head, table_pages, kPageTokens) : 0;
    if (scores < 0 || scores > INT64_MAX / 16) return SIZE_MAX;
    return ((size_t)s.partials + (size_t)scores) * sizeof(float);
}

int launch_span(const char* what, SpanArgs& a, int64_t requests, int64_t max_chunk, int64_t head_dim,
                int64_t table_pages, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const bool weigh = a.w_pool != nullptr;
    SpanShape s;
    CRUCIBLE_CHECK(span_shape(s, requests, max_chunk, a.n_head, a.n_kv_head, head_dim, table_pages, a.mask.window,
                              a.mask.n_sink, weigh),
                   CRUCIBLE_ERR_INVALID, "%s: %lld requests of %lld rows and %d heads are past the grid", what,
                   (long long)requests, (long long)max_chunk, a.n_head);
    CRUCIBLE_CHECK((((uintptr_t)a.k_pool | (uintptr_t)a.v_pool) & 15) == 0, CRUCIBLE_ERR_INVALID,
                   "%s: pools must be 16-byte aligned", what);
    a.n_tiles = s.n_tiles;
    a.split_pages = s.split_pages;
    a.n_splits = s.n_splits;
    const int wide = (int)span_wide(head_dim);
    const size_t need = span_workspace(requests, max_chunk, a.n_head, a.n_kv_head, head_dim, table_pages,
                                       a.mask.window, a.mask.n_sink, weigh);
    if (need) {
        CRUCIBLE_CHECK(workspace && workspace_bytes >= need, CRUCIBLE_ERR_WORKSPACE,
                       "%s: workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : 0, need);
        CRUCIBLE_CHECK(((uintptr_t)workspace & 15) == 0, CRUCIBLE_ERR_INVALID,
                       "%s: workspace must be 16-byte aligned", what);
        const size_t n = (size_t)s.partials / (wide + 2);
        a.po = static_cast<float*>(workspace);
        a.pm = a.po + n * wide;
        a.pl = a.pm + n;
        if (weigh) {
            a.scores = a.pl + n;
            a.score_stride = table_pages * kPageTokens;
        }
    }
    const int r = (int)requests;
    switch (wide) {
        case 32: launch_hd<32>(a, s.qb, r, stream); break;
        case 64: launch_hd<64>(a, s.qb, r, stream); break;
        case 96: launch_hd<96>(a, s.qb, r, stream); break;
        case 128: launch_hd<128>(a, s.qb, r, stream); break;
        case 160: launch_hd<160>(a, s.qb, r, stream); break;
        case 192: launch_hd<192>(a, s.qb, r, stream); break;
        case 224: launch_hd<224>(a, s.qb, r, stream); break;
        default: launch_hd<256>(a, s.qb, r, stream); break;
    }
    return fail_launch(what);
}

SpanArgs span_args(const void* q, int q_dtype, const void* k_pool, const void* v_pool, void* out, int out_dtype,
                   const int32_t* tables, int64_t n_head, int64_t n_kv_head, int64_t head_dim, int64_t table_stride,
                   const PoolAddr& addr, int64_t kv_dim, int64_t window, int64_t n_sink) {
    SpanArgs a{};
    a.q = q;
    a.k_pool = static_cast<const half_t*>(k_pool);
    a.v_pool = static_cast<const half_t*>(v_pool);
    a.out = out;
    a.tables = tables;
    a.addr = addr;
    a.addr.kv_dim = (int32_t)kv_dim;
    a.mask = SpanMask{(int)window, (int)n_sink};
    a.n_head = (int)n_head;
    a.n_kv_head = (int)n_kv_head;
    a.group = (int)(n_head / n_kv_head);
    a.max_chunk = 1;
    a.table_stride = (int)table_stride;
    a.q_f32 = q_dtype == CRUCIBLE_F32;
    a.out_f16 = out_dtype == CRUCIBLE_F16;
    a.head_dim = (int)head_dim;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)head_dim));
    a.n_splits = 1;
    a.n_tiles = 1;
    return a;
}

int64_t pages_of(int64_t tokens) { return (tokens + kPageMask) / kPageTokens; }

}  // namespace
}  // namespace crucible

using namespace crucible;

extern "C" size_t crucible_attention_decode_window_workspace_bytes(int64_t batch, int64_t n_head, int64_t n_kv_head,
                                                                   int64_t head_dim, int64_t max_seq,
                                                                   int64_t window, int64_t n_sink) {
    if (max_seq <= 0 || max_seq > kMaxTablePages * kPageTokens || window > INT32_MAX || n_sink > INT32_MAX || batch > 65535) return 0;
    return span_workspace(batch, 1, n_head, n_kv_head, head_dim, pages_of(max_seq), window, n_sink);
}

extern "C" int crucible_attention_decode_window_paged(
    const void* q, int q_dtype, const void* k_pool, const void* v_pool, void* out, int out_dtype,
    const int32_t* page_tables, const int32_t* seq_lens, int64_t batch, int64_t n_head, int64_t n_kv_head,
    int64_t head_dim, int64_t table_stride, int64_t n_layer, int64_t layer, int64_t kv_dim, int64_t max_seq,
    int64_t window, int64_t n_sink, void* workspace, size_t workspace_bytes, crucible_stream_t stream) {
    const char* what = "attention_decode_window_paged";
    if (int rc = check_span(what, q_dtype, out_dtype, batch, 1, n_head, n_kv_head, head_dim, table_stride, kv_dim,
                            window, n_sink))
        return rc;
    PoolAddr addr;
    CRUCIBLE_CHECK(paged_addr(n_layer, layer, kv_dim, addr), CRUCIBLE_ERR_INVALID, "%s: layer %lld of %lld", what,
                   (long long)layer, (long long)n_layer);
    CRUCIBLE_CHECK(max_seq > 0 && max_seq <= table_stride * kPageTokens, CRUCIBLE_ERR_INVALID,
                   "%s: max_seq %lld past the table's %lld pages", what, (long long)max_seq,
                   (long long)table_stride);
    if (batch == 0) return CRUCIBLE_OK;
    CRUCIBLE_CHECK(q && k_pool && v_pool && out && page_tables && seq_lens, CRUCIBLE_ERR_INVALID, "%s: null buffer",
                   what);
    SpanArgs a = span_args(q, q_dtype, k_pool, v_pool, out, out_dtype, page_tables, n_head, n_kv_head, head_dim,
                           table_stride, addr, kv_dim, window, n_sink);
    a.lens = seq_lens;
    a.max_seq = (int)max_seq;
    return launch_span(what, a, batch, 1, head_dim, pages_of(max_seq), workspace, workspace_bytes, stream);
}

extern "C" size_t crucible_attention_prefill_window_workspace_bytes(int64_t requests, int64_t max_chunk,
                                                                    int64_t table_stride, int64_t n_head,
                                                                    int64_t n_kv_head, int64_t head_dim,
                                                                    int64_t window, int64_t n_sink) {
    if (table_stride <= 0 || table_stride > kMaxTablePages || window > INT32_MAX ||
        n_sink > INT32_MAX || requests > 65535 || max_chunk > INT32_MAX)
        return 0;
    return span_workspace(requests, max_chunk, n_head, n_kv_head, head_dim, table_stride, window, n_sink);
}

extern "C" int crucible_attention_prefill_window_tiled(
    const void* q, int q_dtype, const void* k_pool, const void* v_pool, void* out, int out_dtype,
    const int32_t* tables, const int32_t* segments, int64_t requests, int64_t max_chunk, int64_t table_stride,
    int64_t n_head, int64_t n_kv_head, int64_t head_dim, int64_t n_layer, int64_t layer, int64_t kv_dim,
    int64_t window, int64_t n_sink, void* workspace, size_t workspace_bytes, crucible_stream_t stream) {
    const char* what = "attention_prefill_window_tiled";
    if (int rc = check_span(what, q_dtype, out_dtype, requests, max_chunk, n_head, n_kv_head, head_dim,
                            table_stride, kv_dim, window, n_sink))
        return rc;
    PoolAddr addr;
    CRUCIBLE_CHECK(paged_addr(n_layer, layer, kv_dim, addr), CRUCIBLE_ERR_INVALID, "%s: layer %lld of %lld", what,
                   (long long)layer, (long long)n_layer);
    if (requests == 0 || max_chunk == 0) return CRUCIBLE_OK;
    CRUCIBLE_CHECK(q && k_pool && v_pool && out && tables && segments, CRUCIBLE_ERR_INVALID, "%s: null buffer",
                   what);
    SpanArgs a = span_args(q, q_dtype, k_pool, v_pool, out, out_dtype, tables, n_head, n_kv_head, head_dim,
                           table_stride, addr, kv_dim, window, n_sink);
    a.segments = segments;
    a.max_chunk = (int)max_chunk;
    a.max_seq = (int)(table_stride * kPageTokens);
    return launch_span(what, a, requests, max_chunk, head_dim, table_stride, workspace, workspace_bytes, stream);
}

extern "C" size_t crucible_attention_decode_weigh_workspace_bytes(int64_t batch, int64_t n_head, int64_t n_kv_head,
                                                                  int64_t head_dim, int64_t max_seq) {
    if (max_seq <= 0 || max_seq > kMaxTablePages * kPageTokens || batch > 65535 || n_head > (1 << 20)) return 0;
    return span_workspace(batch, 1, n_head, n_kv_head, head_dim, pages_of(max_seq), INT32_MAX, 0, true);
}

extern "C" int crucible_attention_decode_weigh_paged(
    const void* q, int q_dtype, const void* k_pool, const void* v_pool, float* w_pool, int32_t* pos_pool, void* out,
    int out_dtype, const int32_t* page_tables, const int32_t* positions, const int32_t* seq_lens, int64_t batch,
    int64_t n_head, int64_t n_kv_head, int64_t head_dim, int64_t table_stride, int64_t n_layer, int64_t layer,
    int64_t kv_dim, int64_t max_seq, void* workspace, size_t workspace_bytes, crucible_stream_t stream) {
    const char* what = "attention_decode_weigh_paged";
    if (int rc = check_span(what, q_dtype, out_dtype, batch, 1, n_head, n_kv_head, head_dim, table_stride, kv_dim,
                            INT32_MAX, 0))
        return rc;
    PoolAddr addr;
    CRUCIBLE_CHECK(paged_addr(n_layer, layer, kv_dim, addr), CRUCIBLE_ERR_INVALID, "%s: layer %lld of %lld", what,
                   (long long)layer, (long long)n_layer);
    CRUCIBLE_CHECK(max_seq > 0 && max_seq <= table_stride * kPageTokens, CRUCIBLE_ERR_INVALID,
                   "%s: max_seq %lld past the table's %lld pages", what, (long long)max_seq,
                   (long long)table_stride);
    if (batch == 0) return CRUCIBLE_OK;
    CRUCIBLE_CHECK(q && k_pool && v_pool && w_pool && pos_pool && out && page_tables && positions && seq_lens,
                   CRUCIBLE_ERR_INVALID, "%s: null buffer", what);
    SpanArgs a = span_args(q, q_dtype, k_pool, v_pool, out, out_dtype, page_tables, n_head, n_kv_head, head_dim,
                           table_stride, addr, kv_dim, INT32_MAX, 0);
    a.lens = seq_lens;
    a.max_seq = (int)max_seq;
    a.w_pool = w_pool;
    a.pos_pool = pos_pool;
    a.positions = positions;
    a.n_layer = (int)n_layer;
    a.layer = (int)layer;
    return launch_span(what, a, batch, 1, head_dim, pages_of(max_seq), workspace, workspace_bytes, stream);
}
