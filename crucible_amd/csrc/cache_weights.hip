// The sums of attention weights beside a paged cache: what a prompt's rows give its tokens, and the
// cut of a cache to its heaviest tokens. No counterpart in the reference, whose caches only grow.
//
// Pools of sums (f32) and of positions (int32) lie like the KV pools' pages:
// [page][layer][kv head][16]. Keys are stored with their rotation, so a slot's place in the cache
// means nothing to attention: a cut moves as few tokens as it can, and the pool of positions keeps
// what place they had.
#include <cmath>
#include <type_traits>

#include "generic_attend.hpp"
#include "span_attend.hpp"

namespace crucible {
namespace {

int64_t wide_dim(int64_t hd) { return (hd + 31) / 32 * 32; }

// ---------------------------------------------------------------- a prompt's weights
//
// w[g][j] += sum over the last n_observe rows r of a chunk and the heads h of group g of
//   exp(s(r, h, j) - m(r, h)) / l(r, h),   m and l the row's maximum and sum over j <= its position.
// The sum runs over rows, so m and l come first: observe_rows_kernel forms them (keys split over
// workgroups, joined by observe_join_kernel), and observe_keys_kernel forms the scores again, with
// the keys of a workgroup in registers and the rows going by: their fp16 halves, laid down by the
// first kernel as the lanes load them, and their m and 1 / l. Twice the score products cost less
// than scores in memory: 4 bytes a score against head_dim / 16 MFMA flops of a 16-wide tile.
// Bound: chains of loads, on which the rows' waves spend 63% of their time. Eight prompts of 46 to
// 420 rows, all observed, 16 / 4 heads of 64: rows 17.3 us, keys 14.0; the last 64 of 16,384 rows,
// 12 / 3 heads: rows 13.6, join 3.9, keys 12.2. Rows with 8 or 2 waves a workgroup: 25.7 and 15.4
// in the first, 16.6 and 17.5 in the second; operands of four tiles ahead instead of one: 21 to
// 24 for the keys' 14.

struct ObserveArgs {
    const void* q;
    const half_t* k_pool;
    float* w_pool;
    int32_t* pos_pool;
    const int32_t* tables;
    const int32_t* segments;
    const int32_t* lens;  // unused: SpanRows reads segments
    const int32_t* positions;
    PoolAddr addr;
    int32_t n_head, n_kv_head, group, max_chunk, table_stride, max_seq;
    int32_t n_observe, n_layer, layer, head_dim;
    int32_t n_tiles, split_pages, n_splits;
    int32_t columns;  // of a (request, KV head), at most, in whole tiles
    float scale_log2;
    float2* part;   // [request][kv head][tile][split][column] m, l
    float4* norm;   // [request][kv head][column] m, 1 / l, score -> log2 units, position (as int bits)
    half8_t* frag;  // [request][kv head][16 columns][hi, lo][32 dimensions][lane]
};

// The observed rows of request b: `n` of them from row `skip` of its chunk on.
struct Observed {
    int skip, n;
    __device__ __forceinline__ Observed(const ObserveArgs& a, const SpanRows& r) {
        n = min(a.n_observe, r.rows);
        skip = r.rows - n;
    }
};

__device__ __forceinline__ int64_t observe_row(const ObserveArgs& a, const SpanRows& r, const Observed& o, int g,
                                               int c) {
    return ((int64_t)(r.packed + o.skip + c / a.group) * a.n_head + g * a.group + c % a.group) * a.head_dim;
}

template <int HD, bool PAD, bool F32, int QB>
__global__ __launch_bounds__(256, HD <= 64 ? (F32 && QB == 2 ? 3 : 4) : 2) void observe_rows_kernel(ObserveArgs a) {
    constexpr int W = 4;
    __shared__ float sm[W][16 * QB], sl[W][16 * QB];
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = blockIdx.x, b = blockIdx.z;
    const int g = blockIdx.y / a.n_tiles, tile = blockIdx.y % a.n_tiles;
    const SpanRows r(a, b);
    const Observed o(a, r);
    const int c0 = tile * 16 * QB;
    const int n_cols = (int)min((int64_t)16 * QB, (int64_t)o.n * a.group - c0);
    if (n_cols <= 0) return;
    const int p0 = r.first + o.skip + c0 / a.group;
    const int p1 = r.first + o.skip + (c0 + n_cols - 1) / a.group;
    const int pages = (p1 >> kPageShift) + 1;
    const int i0 = split * a.split_pages, i1 = min(i0 + a.split_pages, pages);
    if (i0 >= i1) return;
    // page ids, one a lane, 64 at a time
    int id = 0, at_id = 2 * wave;
    if (lane < i1 - i0) id = r.table[i0 + lane];
    const SpanDim<HD, PAD> dim{a.head_dim};
    const int64_t unit = (int64_t)b * a.n_kv_head + g;
    HdQuery<HD, F32> q[QB];
    int pos[QB];
    float m[QB], l[QB];
#pragma unroll
    for (int k = 0; k < QB; ++k) {
        const int c = 16 * k + col;
        const bool on = c < n_cols;
        span_query(q[k], dim, a.q, on ? observe_row(a, r, o, g, c0 + c) : 0, on, grp, a.scale_log2);
        pos[k] = on ? r.first + o.skip + (c0 + c) / a.group : -1;
        m[k] = -INFINITY;
        l[k] = 0.0f;
        if (split == 0 && wave == 0) {
            constexpr int N = (F32 ? 2 : 1) * (HD / 32);
            half8_t* to = a.frag + ((unit * a.columns + c0) / 16 + k) * N * 64 + lane;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                to[64 * i] = q[k].hi[i];
                if constexpr (F32) to[64 * (HD / 32 + i)] = q[k].lo[i];
            }
            if (grp == 0) {
                float4& to = a.norm[unit * a.columns + c0 + c];
                to.z = q[k].scale;
                to.w = __builtin_bit_cast(float, pos[k]);
            }
        }
    }
    const int head_off = g * dim.hd(), kv_dim = a.addr.kv_dim, n = i1 - i0;
    int64_t base0, base1;
    const auto find = [&](int i) {
        if ((i & 63) == 2 * wave && i != at_id) {
            at_id = i;
            const int next = (i & ~63) + lane;
            if (next < n) id = r.table[i0 + next];
        }
        base0 = block_base(a.addr, __builtin_amdgcn_readlane(id, i & 63));
        base1 = i + 1 < n ? block_base(a.addr, __builtin_amdgcn_readlane(id, (i & 63) + 1)) : base0;
    };
    // EXACT: with the scores that f32 sums give where an operand is infinite
    const auto run = [&](auto exact) {
        SpanKeys<HD, PAD> ks;
        int i = 2 * wave;
        if (i < n) {
            find(i);
            ks.load(dim, a.k_pool, col >= 8 ? base1 : base0, kv_dim, head_off, col, grp);
        }
        while (i < n) {
            const int key = (i0 + i) * kPageTokens + 8 * grp;  // of a page that is none: past every row
            const bool masked = (i0 + i + 2) * kPageTokens > p0 + 1;
            float4_t s[QB][2];
#pragma unroll
            for (int k = 0; k < QB; ++k) {
                span_scores(s[k], q[k], ks);
                if constexpr (exact.value)
                    span_exact_scores(s[k], q[k], dim, a.q, a.k_pool, grp >= 2 ? base1 : base0, kv_dim, head_off,
                                      pos[k] >= 0, observe_row(a, r, o, g, c0 + 16 * k + col), grp, a.scale_log2, F32);
            }
            i += 2 * W;
            if (i < n) {  // the next keys, while these scores are summed
                find(i);
                ks.load(dim, a.k_pool, col >= 8 ? base1 : base0, kv_dim, head_off, col, grp);
            }
#pragma unroll
            for (int k = 0; k < QB; ++k) {
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[k][t][e] = masked && key + 4 * t + e > pos[k] ? -INFINITY : s[k][t][e] * q[k].scale;
                        mx = fmaxf(mx, s[k][t][e]);
                    }
                const float mn = fmaxf(m[k], mx);
                const float at = mn == -INFINITY ? 0.0f : mn;
                float sum = 0.0f;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += fast_exp2(s[k][t][e] - at);
                l[k] = __builtin_fmaf(l[k], fast_exp2(m[k] - at), sum);
                m[k] = mn;
            }
        }
    };
    run(std::false_type{});
    float z = 0.0f;
#pragma unroll
    for (int k = 0; k < QB; ++k) z = __builtin_fmaf(l[k], 0.0f, z);
    if (__ballot(!(z == 0.0f))) {
#pragma unroll
        for (int k = 0; k < QB; ++k) {
            m[k] = -INFINITY;
            l[k] = 0.0f;
        }
        run(std::true_type{});
    }
    // the lane groups, then the waves
#pragma unroll
    for (int k = 0; k < QB; ++k) {
        const float mn = group_max4(m[k]);
        const float at = mn == -INFINITY ? 0.0f : mn;
        const float sum = group_sum4(l[k] * fast_exp2(m[k] - at));
        if (grp == 0) {
            sm[wave][16 * k + col] = mn;
            sl[wave][16 * k + col] = sum;
        }
    }
    __syncthreads();
    const int c = threadIdx.x;
    if (c >= n_cols) return;
    float mn = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) mn = fmaxf(mn, sm[w][c]);
    const float at = mn == -INFINITY ? 0.0f : mn;
#pragma unroll
    for (int w = 0; w < W; ++w) sum = __builtin_fmaf(sl[w][c], fast_exp2(sm[w][c] - at), sum);
    if (a.n_splits == 1) {
        float4& to = a.norm[unit * a.columns + c0 + c];
        to.x = at;
        to.y = sum == 0.0f ? 0.0f : 1.0f / sum;
    } else {
        a.part[((unit * a.n_tiles + tile) * a.n_splits + split) * 16 * QB + c] = float2{mn, sum};
    }
}

template <int QB>
__global__ __launch_bounds__(256) void observe_join_kernel(ObserveArgs a) {
    const int b = blockIdx.z, g = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x;
    const SpanRows r(a, b);
    const Observed o(a, r);
    if (c >= (int64_t)o.n * a.group) return;
    const int tile = c / (16 * QB);
    const int last = min((tile + 1) * 16 * QB, o.n * a.group) - 1;
    const int pages = ((r.first + o.skip + last / a.group) >> kPageShift) + 1;
    const int n = (pages + a.split_pages - 1) / a.split_pages;
    const int64_t unit = (int64_t)b * a.n_kv_head + g;
    const float2* p = a.part + (unit * a.n_tiles + tile) * a.n_splits * 16 * QB + c % (16 * QB);
    float m = -INFINITY, l = 0.0f;
    constexpr int U = 8;  // splits on their way at a time
    for (int s0 = 0; s0 < n; s0 += U) {
        float2 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = s0 + u < n ? p[(int64_t)(s0 + u) * 16 * QB] : float2{-INFINITY, 0.0f};
        float mx = m;
#pragma unroll
        for (int u = 0; u < U; ++u) mx = fmaxf(mx, x[u].x);
        const float at = mx == -INFINITY ? 0.0f : mx;
        l *= fast_exp2(m - at);
#pragma unroll
        for (int u = 0; u < U; ++u) l = __builtin_fmaf(x[u].y, fast_exp2(x[u].x - at), l);
        m = mx;
    }
    float4& to = a.norm[unit * a.columns + c];
    to.x = m == -INFINITY ? 0.0f : m;
    to.y = l == 0.0f ? 0.0f : 1.0f / l;
}

// 32 KP keys of a (request, KV head) against every observed row that sees one of them. A wave takes
// every W-th tile of 16 columns, the next tile's operands on their way while one is summed.
template <int HD, bool PAD, bool F32, int KP, int W>
__global__ __launch_bounds__(64 * W, HD <= 64 && KP <= 2 ? 4 : 2) void observe_keys_kernel(ObserveArgs a) {
    constexpr int N = (F32 ? 2 : 1) * (HD / 32);
    __shared__ float part[W][32 * KP];
    __shared__ int s_bad;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.z, g = blockIdx.y;
    const SpanRows r(a, b);
    const Observed o(a, r);
    const int key0 = blockIdx.x * 32 * KP, end = r.first + r.rows;
    if (r.rows <= 0 || key0 >= end) return;
    if (threadIdx.x == 0) s_bad = 0;
    const SpanDim<HD, PAD> dim{a.head_dim};
    const int head_off = g * dim.hd(), kv_dim = a.addr.kv_dim;
    const int64_t unit = (int64_t)b * a.n_kv_head + g;
    const float4* norm = a.norm + unit * a.columns;
    const half8_t* frag = a.frag + unit * a.columns / 16 * N * 64 + lane;
    const int n_cols = o.n * a.group, first = r.first + o.skip;
    const int from = key0 > first ? (int)min((int64_t)(key0 - first) * a.group, (int64_t)n_cols) / 16 : 0;
    half8_t q[N];
    float4 nm = {0.f, 0.f, 0.f, 0.f};
    const auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = frag[((int64_t)t * N + i) * 64];
        nm = norm[16 * t + col];
    };
    int t = from + wave;
    if (t * 16 < n_cols) load(t);
    SpanKeys<HD, PAD> ks[KP];
#pragma unroll
    for (int k = 0; k < KP; ++k) {
        const int last = (end - 1) >> kPageShift, page = (key0 >> kPageShift) + 2 * k;
        const int64_t base0 = block_base(a.addr, r.table[min(page, last)]);
        const int64_t base1 = block_base(a.addr, r.table[min(page + 1, last)]);
        ks[k].load(dim, a.k_pool, col >= 8 ? base1 : base0, kv_dim, head_off, col, grp);
    }
    float acc[KP][2][4] = {};
    while (t * 16 < n_cols) {
        float4_t s[KP][2];
#pragma unroll
        for (int k = 0; k < KP; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s[k][u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    s[k][u] = mfma_16x16x32(ks[k].k[u][i], q[i], s[k][u]);
                    if constexpr (F32) s[k][u] = mfma_16x16x32(ks[k].k[u][i], q[HD / 32 + i], s[k][u]);
                }
            }
        const bool on = 16 * t + col < n_cols;
        const float m = on ? nm.x : 0.0f, inv = on ? nm.y : 0.0f, scale = nm.z;
        const int pos = on ? __builtin_bit_cast(int, nm.w) : -1;
        const bool masked = key0 + 32 * KP > first + 16 * t / a.group + 1;
        t += W;
        if (t * 16 < n_cols) load(t);
        if (masked) {
#pragma unroll
            for (int k = 0; k < KP; ++k)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float w = fast_exp2(__builtin_fmaf(s[k][u][e], scale, -m)) * inv;
                        acc[k][u][e] += key0 + 32 * k + 8 * grp + 4 * u + e > pos ? 0.0f : w;
                    }
        } else {
#pragma unroll
            for (int k = 0; k < KP; ++k)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[k][u][e] = __builtin_fmaf(fast_exp2(__builtin_fmaf(s[k][u][e], scale, -m)), inv, acc[k][u][e]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KP; ++k)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = acc[k][u][e];
#pragma unroll
                for (int off = 1; off < 16; off <<= 1) x += __shfl_xor(x, off);
                if (col == 0) {
                    part[wave][32 * k + 8 * grp + 4 * u + e] = x;
                    if (!(x * 0.0f == 0.0f)) s_bad = 1;
                }
            }
    __syncthreads();
    const int i = threadIdx.x, j = key0 + i;
    if (i >= 32 * KP || j >= end) return;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += part[w][i];
    if (s_bad) {
        // A sum that is not finite may be what f32 gives, or an infinite key's product with a lo
        // half of 0: once more, plainly.
        sum = 0.0f;
        const half_t* kr = a.k_pool + block_base(a.addr, r.table[j >> kPageShift]) +
                           (int64_t)(j & kPageMask) * kv_dim + head_off;
        for (int c = j > first ? (j - first) * a.group : 0; c < n_cols; ++c) {
            const int64_t at = observe_row(a, r, o, g, c);
            float s = 0.0f;
            for (int d = 0; d < dim.hd(); ++d) {
                const float x = F32 ? static_cast<const float*>(a.q)[at + d]
                                    : (float)static_cast<const half_t*>(a.q)[at + d];
                s = __builtin_fmaf(x, (float)kr[d], s);
            }
            sum = __builtin_fmaf(fast_exp2(s * a.scale_log2 - norm[c].x), norm[c].y, sum);
        }
    }
    const int64_t page = r.table[j >> kPageShift];
    const int64_t at = ((page * a.n_layer + a.layer) * a.n_kv_head + g) * kPageTokens + (j & kPageMask);
    if (j < r.first) {
        a.w_pool[at] += sum;
    } else {
        a.w_pool[at] = sum;
        a.pos_pool[at] = a.positions[r.packed + j - r.first];
    }
}

struct ObserveShape {
    int qb, n_tiles, split_pages, n_splits, kp;
    int64_t columns, part, norm, frag;  // part: float2s, norm: float4s, frag: half8_ts
};

bool observe_shape(ObserveShape& s, int64_t requests, int64_t max_chunk, int64_t n_head, int64_t n_kv_head,
                   int64_t hd, int64_t table_pages, int64_t n_observe) {
    const int64_t rows = n_observe < max_chunk ? n_observe : max_chunk, wide = wide_dim(hd);
    const int64_t columns = checked_mul(rows, n_head / n_kv_head);
    if (columns < 0 || columns > INT32_MAX - 256) return false;
    s.qb = wide <= 128 && columns > 16 ? 2 : 1;
    const int64_t tiles = (columns + 16 * s.qb - 1) / (16 * s.qb);
    const int64_t units = checked_mul(requests, n_kv_head, tiles > 0 ? tiles : 1);
    if (units < 0 || tiles * n_kv_head > 65535 || requests > 65535 || n_kv_head > 65535) return false;
    s.n_tiles = (int)tiles;
    s.columns = tiles * 16 * s.qb;
    // Splits as many as give every CU two workgroups of four waves, of 2 to 8 steps of 8 pages.
    const int64_t cus = device_cu_count();
    int64_t sp = table_pages;
    if (units < 2 * cus) {
        const int64_t n = 2 * cus / units;
        sp = ((table_pages + n - 1) / n + 7) / 8 * 8;
        sp = sp < 16 ? 16 : sp > 64 ? 64 : sp;
    }
    s.split_pages = (int)sp;
    s.n_splits = (int)((table_pages + sp - 1) / sp);
    // Keys of a workgroup: the more, the fewer times a row's operands are loaded; but few
    // workgroups walk their rows one after another.
    s.kp = wide <= 64 ? 4 : wide <= 128 ? 2 : 1;
    while (s.kp > 1 && requests * n_kv_head * ((table_pages + 2 * s.kp - 1) / (2 * s.kp)) < 2 * cus) s.kp /= 2;
    s.part = s.n_splits > 1 ? checked_mul(units, s.n_splits, 16 * s.qb) : 0;
    s.norm = checked_mul(requests, n_kv_head, s.columns);
    s.frag = checked_mul(s.norm, wide / 32 * 8);  // hi and lo: 2 x 64 lanes for 16 columns
    return s.part >= 0 && s.frag >= 0 && s.part < INT64_MAX / 64 && s.frag < INT64_MAX / 64;
}

size_t observe_bytes(const ObserveShape& s) {
    return (size_t)s.frag * sizeof(half8_t) + (size_t)s.norm * sizeof(float4) + (size_t)s.part * sizeof(float2);
}

template <int HD, bool PAD, bool F32, int KP>
void launch_keys(const ObserveArgs& a, int requests, hipStream_t stream) {
    const dim3 keys((unsigned)((a.max_seq + 32 * KP - 1) / (32 * KP)), (unsigned)a.n_kv_head, (unsigned)requests);
    // Eight waves where the rows are many; where each would have two tiles or none, four, so that
    // twice the workgroups fit.
    if (a.columns > 512)
        hipLaunchKernelGGL((observe_keys_kernel<HD, PAD, F32, KP, 8>), keys, dim3(512), 0, stream, a);
    else
        hipLaunchKernelGGL((observe_keys_kernel<HD, PAD, F32, KP, 4>), keys, dim3(256), 0, stream, a);
}

template <int HD, bool PAD, bool F32>
void launch_observe(const ObserveArgs& a, int qb, int kp, int requests, hipStream_t stream) {
    constexpr int QB = HD <= 128 ? 2 : 1;
    if (a.columns) {
        const dim3 rows((unsigned)a.n_splits, (unsigned)(a.n_kv_head * a.n_tiles), (unsigned)requests);
        const dim3 join((unsigned)((a.columns + 255) / 256), (unsigned)a.n_kv_head, (unsigned)requests);
        if (qb == 1) {
            hipLaunchKernelGGL((observe_rows_kernel<HD, PAD, F32, 1>), rows, dim3(256), 0, stream, a);
            if (a.n_splits > 1) hipLaunchKernelGGL((observe_join_kernel<1>), join, dim3(256), 0, stream, a);
        } else {
            hipLaunchKernelGGL((observe_rows_kernel<HD, PAD, F32, QB>), rows, dim3(256), 0, stream, a);
            if (a.n_splits > 1) hipLaunchKernelGGL((observe_join_kernel<QB>), join, dim3(256), 0, stream, a);
        }
    }
    if constexpr (HD <= 64) {
        if (kp == 4) return launch_keys<HD, PAD, F32, 4>(a, requests, stream);
    }
    if constexpr (HD <= 128) {
        if (kp == 2) return launch_keys<HD, PAD, F32, 2>(a, requests, stream);
    }
    launch_keys<HD, PAD, F32, 1>(a, requests, stream);
}

template <int HD>
void launch_observe_hd(const ObserveArgs& a, bool f32, const ObserveShape& s, int requests, hipStream_t stream) {
    if (a.head_dim == HD)
        f32 ? launch_observe<HD, false, true>(a, s.qb, s.kp, requests, stream)
            : launch_observe<HD, false, false>(a, s.qb, s.kp, requests, stream);
    else
        f32 ? launch_observe<HD, true, true>(a, s.qb, s.kp, requests, stream)
            : launch_observe<HD, true, false>(a, s.qb, s.kp, requests, stream);
}

// ---------------------------------------------------------------- the cut
//
// A request of n > keep tokens keeps, in every layer and KV head, the tokens at positions below
// n_sink, those at the n_recent newest positions, and of the others the heaviest (equal sums: the
// lower slot; NaN below every number). The i-th free slot below `keep` takes the i-th kept token at
// or past it, so what is read lies past `keep` and what is written below it: no order between moves.

// Sums as unsigned whole numbers of the same order: 0 is no token, NaN is 1, protected tokens are
// above all.
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int n_sink, int newest, int n_recent) {
    if (pos < n_sink || pos > (int64_t)newest - n_recent) return 0xffffffffu;
    if (w != w) return 1u;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct EvictArgs {
    half_t* k_pool;
    half_t* v_pool;
    float* w_pool;
    int32_t* pos_pool;
    const int32_t* tables;
    const int32_t* lens;
    int32_t* new_lens;
    int32_t n_kv_head, head_dim, kv_dim, table_stride, n_layer, max_seq;
    int32_t keep, n_sink, n_recent;
    int32_t max_moves;
    int32_t write_lens;  // the selecting launch writes new_lens (it is not seq_lens)
    int32_t* count;      // [request][layer][kv head]
    int2* moves;         // [request][layer][kv head][max_moves] free slot, kept slot
};

__device__ __forceinline__ int evict_len(int n, int keep, int max_seq) { return n > keep && n <= max_seq ? keep : n; }

// Up to kMoveChunk moves of a (layer, KV head), by the whole workgroup. A lane keeps its move's
// addresses: keys go in 16-byte pieces, a token's side by side; values lie 16 tokens to a row, so the
// lanes of a wave take one dimension of neighbouring moves, whose slots share rows.
// Bound: those rows. Of a page that keeps 2.6 of 16 tokens all 2 KB of a head's values are fetched:
// 4 prompts of up to 16,384 tokens cut to 2,048, 12 layers x 3 KV heads, take 84 us, 66 without the
// stores of values and 19 without values, whose 132 MB thus come at 2.8 TB/s (blocks of 2 KB here
// and there reach 3.4 to 4). The same through LDS, in 16-byte pieces (84) or with the lanes on
// dimensions on either side (92 to 112). Of 23 us for 16 requests of up to 64 tokens too many, 13
// are moves, with stores of 2 bytes into as many different rows.
constexpr int kMoveChunk = 64;

struct MoveLds {
    int64_t src_page[kMoveChunk], dst_page[kMoveChunk];
    int src_slot[kMoveChunk], dst_slot[kMoveChunk];
};

template <class Moves>
__device__ __forceinline__ void evict_move(MoveLds& lds, const EvictArgs& a, int b, int unit, int n, Moves moves) {
    const int t = threadIdx.x, layer = unit / a.n_kv_head, g = unit % a.n_kv_head;
    __syncthreads();
    if (t < n) {
        const int2 mv = moves(t);
        const int32_t* table = a.tables + (int64_t)b * a.table_stride;
        const int64_t dp = (int64_t)table[mv.x >> kPageShift] * a.n_layer + layer;
        const int64_t sp = (int64_t)table[mv.y >> kPageShift] * a.n_layer + layer;
        const int ds = mv.x & kPageMask, ss = mv.y & kPageMask;
        const int64_t from = (sp * a.n_kv_head + g) * kPageTokens + ss, to = (dp * a.n_kv_head + g) * kPageTokens + ds;
        const float w = a.w_pool[from];
        const int pos = a.pos_pool[from];
        lds.dst_page[t] = dp;
        lds.src_page[t] = sp;
        lds.dst_slot[t] = ds;
        lds.src_slot[t] = ss;
        a.w_pool[to] = w;
        a.pos_pool[to] = pos;
    }
    __syncthreads();
    const int64_t block = (int64_t)kPageTokens * a.kv_dim;
    // 64 dimensions at a time; everything a thread moves of them is on its way before it stores.
    constexpr int S = 64, KU = S / 8 * kMoveChunk / 256, VU = S * kMoveChunk / 256;
    // As many lanes a dimension as there are moves, in powers of two; of a 1024-thread workgroup
    // the first 256 threads.
    if (t >= 256) return;
    int lanes = 64;
    while (lanes > 8 && lanes / 2 >= n) lanes /= 2;
    const int m = t % lanes, step = 256 / lanes;
    const half_t* src = a.v_pool;
    half_t* dst = a.v_pool;
    if (m < n) {
        src += lds.src_page[m] * block + lds.src_slot[m];
        dst += lds.dst_page[m] * block + lds.dst_slot[m];
    }
    for (int s = 0; s < a.head_dim; s += S) {
        const int d0 = g * a.head_dim + s, dims = min(S, a.head_dim - s), units = dims / 8;
        half8_t k[KU];
        half_t v[VU];
#pragma unroll
        for (int x = 0; x < KU; ++x) {
            const int i = t + 256 * x, j = i / units;
            if (j < n)
                k[x] = *reinterpret_cast<const half8_t*>(a.k_pool + lds.src_page[j] * block +
                                                         (int64_t)lds.src_slot[j] * a.kv_dim + d0 + 8 * (i % units));
        }
#pragma unroll
        for (int x = 0; x < VU; ++x) {
            const int d = t / lanes + x * step;
            if (m < n && d < dims) v[x] = src[(d0 + d) * kPageTokens];
        }
#pragma unroll
        for (int x = 0; x < KU; ++x) {
            const int i = t + 256 * x, j = i / units;
            if (j < n)
                *reinterpret_cast<half8_t*>(a.k_pool + lds.dst_page[j] * block + (int64_t)lds.dst_slot[j] * a.kv_dim +
                                            d0 + 8 * (i % units)) = k[x];
        }
#pragma unroll
        for (int x = 0; x < VU; ++x) {
            const int d = t / lanes + x * step;
            if (m < n && d < dims) dst[(d0 + d) * kPageTokens] = v[x];
        }
    }
}

// The sums over W waves of three counts each, from LDS: a lane reads one, 16 (4) lanes add up.
template <int W>
__device__ __forceinline__ void wave_counts(const int (&c)[4][W], int lane, int (&all)[3]) {
    static_assert(W == 4 || W == 16, "");
    int v = lane < 4 * W ? c[lane / W][lane % W] : 0;
#pragma unroll
    for (int d = 1; d < W; d <<= 1) v += __shfl_xor(v, d);
#pragma unroll
    for (int x = 0; x < 3; ++x) all[x] = __builtin_amdgcn_readlane(v, x * W);
}

// Selection of a (request, layer, KV head), whose T R keys stay in registers: a wave has 64 R tokens
// side by side, lane l of it tokens 64 i + l. The threshold is the largest key that `keep` keys
// reach, found two bits at a time by counting (a ballot and a bit count a register, no atomics, one
// barrier a step), until the count is `keep` exactly: for sums that differ, after about half of the
// 16 steps. 144 selections from up to 16,384 tokens take 33 us; 576 from up to 1,088, 10 of which 7
// are the chain of loads. Few moves follow in the same launch (FUSE), many in one of their own.
template <int T, int R, bool FUSE>
__global__ __launch_bounds__(T) void evict_select_kernel(EvictArgs a) {
    constexpr int W = T / 64;
    __shared__ int cnt[2][4][W];  // three are used
    __shared__ int red[3][W];
    __shared__ uint16_t list[FUSE ? 2 : 1][FUSE ? T * R : 1];
    __shared__ MoveLds move_lds;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int unit = blockIdx.x, b = blockIdx.y;  // unit: layer * n_kv_head + g
    const int n = a.lens[b];
    const int64_t u = (int64_t)b * gridDim.x + unit;
    if (a.write_lens && unit == 0 && t == 0) a.new_lens[b] = evict_len(n, a.keep, a.max_seq);
    if (n <= a.keep || n > a.max_seq) {
        if (!FUSE && t == 0) a.count[u] = 0;
        return;
    }
    const int32_t* table = a.tables + (int64_t)b * a.table_stride;
    const int64_t stride = (int64_t)a.n_layer * a.n_kv_head * kPageTokens, off = (int64_t)unit * kPageTokens;
    const int j0 = wave * 64 * R + lane;
    float w[R];
    int pos[R];
    {
        int page[R];
#pragma unroll
        for (int i = 0; i < R; ++i) page[i] = j0 + 64 * i < n ? table[(j0 + 64 * i) >> kPageShift] : 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t at = page[i] * stride + off + (lane & kPageMask);
            w[i] = 0.0f;
            pos[i] = INT32_MIN;
            if (j0 + 64 * i < n) {
                w[i] = a.w_pool[at];
                pos[i] = a.pos_pool[at];
            }
        }
    }
    int newest = INT32_MIN;
#pragma unroll
    for (int i = 0; i < R; ++i) newest = max(newest, pos[i]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) newest = max(newest, __shfl_xor(newest, d));
    if (lane == 0) red[0][wave] = newest;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < W; ++x) newest = max(newest, red[0][x]);
    uint32_t key[R];
#pragma unroll
    for (int i = 0; i < R; ++i)
        key[i] = j0 + 64 * i < n ? evict_key(w[i], pos[i], a.n_sink, newest, a.n_recent) : 0u;

    uint32_t threshold = 0;
    int above = 0;  // keys that reach it
    for (int shift = 30; shift >= 0 && above != a.keep; shift -= 2) {
        int (&c)[4][W] = cnt[shift >> 1 & 1];
        int own[3] = {0, 0, 0};
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int x = 0; x < 3; ++x)
                own[x] += __builtin_popcountll(__ballot(key[i] >= (threshold | (uint32_t)(x + 1) << shift)));
        if (lane < 3) c[lane][wave] = lane == 0 ? own[0] : lane == 1 ? own[1] : own[2];
        __syncthreads();
        int all[3];
        wave_counts<W>(c, lane, all);
        const int digit = all[2] >= a.keep ? 3 : all[1] >= a.keep ? 2 : all[0] >= a.keep ? 1 : 0;
        if (digit) above = all[digit - 1];
        threshold |= (uint32_t)digit << shift;
    }
    // Where more keys reach the threshold than are kept, those equal to it go by slot.
    const bool ties = above != a.keep;
    int free_ties = 0, before = 0;  // equal keys that stay; equal keys of the waves before
    if (ties) {
        int eq = 0, gt = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            eq += __builtin_popcountll(__ballot(key[i] == threshold));
            gt += __builtin_popcountll(__ballot(key[i] > threshold));
        }
        __syncthreads();  // red[0] has been read by everyone
        if (lane == 0) {
            red[0][wave] = eq;
            red[1][wave] = gt;
        }
        __syncthreads();
        free_ties = a.keep;
#pragma unroll
        for (int x = 0; x < W; ++x) {
            free_ties -= red[1][x];
            if (x < wave) before += red[0][x];
        }
    }
    const uint64_t below = (1ull << lane) - 1;
    uint32_t kept = 0;  // bit i: token i of the lane (R <= 32)
    int holes = 0, movers = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        bool k = key[i] >= threshold && key[i] > 0;
        if (ties) {
            const uint64_t eq = __ballot(key[i] == threshold);
            if (key[i] == threshold) k = before + __builtin_popcountll(eq & below) < free_ties;
            before += __builtin_popcountll(eq);
        }
        kept |= (uint32_t)k << i;
        const int j = j0 + 64 * i;
        holes += __builtin_popcountll(__ballot(j < a.keep && !k));
        movers += __builtin_popcountll(__ballot(j >= a.keep && k));
    }
    __syncthreads();  // red and cnt have been read by everyone
    if (lane == 0) {
        red[0][wave] = holes;
        red[1][wave] = movers;
    }
    __syncthreads();
    holes = movers = 0;
    int total = 0;
#pragma unroll
    for (int x = 0; x < W; ++x) {
        if (x < wave) {
            holes += red[0][x];
            movers += red[1][x];
        }
        total += red[1][x];
    }
    int2* moves = FUSE ? nullptr : a.moves + u * a.max_moves;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int j = j0 + 64 * i;
        const bool k = kept >> i & 1, hole = j < a.keep && !k, mover = j >= a.keep && k;
        const uint64_t hb = __ballot(hole), mb = __ballot(mover);
        const int h = holes + __builtin_popcountll(hb & below), m = movers + __builtin_popcountll(mb & below);
        if constexpr (FUSE) {
            if (hole) list[0][h] = (uint16_t)j;
            if (mover) list[1][m] = (uint16_t)j;
        } else {
            if (hole) moves[h].x = j;
            if (mover) moves[m].y = j;
        }
        holes += __builtin_popcountll(hb);
        movers += __builtin_popcountll(mb);
    }
    if constexpr (FUSE) {
        for (int m0 = 0; m0 < total; m0 += kMoveChunk)
            evict_move(move_lds, a, b, unit, min(kMoveChunk, total - m0),
                       [&](int i) { return int2{list[0][m0 + i], list[1][m0 + i]}; });
    } else {
        if (t == 0) a.count[u] = total;
    }
}

// The same for more tokens than registers hold: keys are formed again in every step.
__global__ __launch_bounds__(1024) void evict_select_long_kernel(EvictArgs a) {
    constexpr int T = 1024, W = T / 64;
    __shared__ int cnt[2][4][W];
    __shared__ int red[3][W];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int unit = blockIdx.x, b = blockIdx.y;
    const int n = a.lens[b];
    const int64_t u = (int64_t)b * gridDim.x + unit;
    if (a.write_lens && unit == 0 && t == 0) a.new_lens[b] = evict_len(n, a.keep, a.max_seq);
    if (n <= a.keep || n > a.max_seq) {
        if (t == 0) a.count[u] = 0;
        return;
    }
    const int32_t* table = a.tables + (int64_t)b * a.table_stride;
    const int64_t stride = (int64_t)a.n_layer * a.n_kv_head * kPageTokens, off = (int64_t)unit * kPageTokens;
    const auto place = [&](int j) { return table[j >> kPageShift] * stride + off + (j & kPageMask); };
    int newest = INT32_MIN;
    for (int j = t; j < n; j += T) newest = max(newest, a.pos_pool[place(j)]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) newest = max(newest, __shfl_xor(newest, d));
    if (lane == 0) red[0][wave] = newest;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < W; ++x) newest = max(newest, red[0][x]);
    const auto form = [&](int j) {
        const int64_t at = place(j);
        return evict_key(a.w_pool[at], a.pos_pool[at], a.n_sink, newest, a.n_recent);
    };
    uint32_t threshold = 0;
    int above = 0;
    for (int shift = 30; shift >= 0 && above != a.keep; shift -= 2) {
        int (&c)[4][W] = cnt[shift >> 1 & 1];
        int own[3] = {0, 0, 0};
        for (int j = t; j < n; j += T) {
            const uint32_t k = form(j);
#pragma unroll
            for (int x = 0; x < 3; ++x) own[x] += k >= (threshold | (uint32_t)(x + 1) << shift);
        }
#pragma unroll
        for (int x = 0; x < 3; ++x) {
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) own[x] += __shfl_xor(own[x], d);
            if (lane == 0) c[x][wave] = own[x];
        }
        __syncthreads();
        int all[3];
        wave_counts<W>(c, lane, all);
        const int digit = all[2] >= a.keep ? 3 : all[1] >= a.keep ? 2 : all[0] >= a.keep ? 1 : 0;
        if (digit) above = all[digit - 1];
        threshold |= (uint32_t)digit << shift;
    }
    int greater = 0;
    for (int j = t; j < n; j += T) greater += form(j) > threshold;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) greater += __shfl_xor(greater, d);
    __syncthreads();
    if (lane == 0) red[0][wave] = greater;
    __syncthreads();
    int ties = a.keep, holes = 0, movers = 0;  // equal keys still to keep; numbers so far
#pragma unroll
    for (int x = 0; x < W; ++x) ties -= red[0][x];
    int2* moves = a.moves + u * a.max_moves;
    const uint64_t below = (1ull << lane) - 1;
    for (int j0 = 0; j0 < n; j0 += T) {
        const int j = j0 + t;
        const uint32_t k = j < n ? form(j) : 0;
        const uint64_t eq = __ballot(j < n && k == threshold);
        __syncthreads();
        if (lane == 0) red[0][wave] = __builtin_popcountll(eq);
        __syncthreads();
        int before = __builtin_popcountll(eq & below), all = 0;
        for (int x = 0; x < W; ++x) {
            if (x < wave) before += red[0][x];
            all += red[0][x];
        }
        const bool kept = j < n && (k > threshold || (k == threshold && before < ties));
        const bool hole = j < a.keep && !kept, mover = j >= a.keep && kept;
        const uint64_t hb = __ballot(hole), mb = __ballot(mover);
        if (lane == 0) {
            red[1][wave] = __builtin_popcountll(hb);
            red[2][wave] = __builtin_popcountll(mb);
        }
        __syncthreads();
        int h = holes + __builtin_popcountll(hb & below), m = movers + __builtin_popcountll(mb & below);
        for (int x = 0; x < W; ++x) {
            if (x < wave) {
                h += red[1][x];
                m += red[2][x];
            }
            holes += red[1][x];
            movers += red[2][x];
        }
        if (hole) moves[h].x = j;
        if (mover) moves[m].y = j;
        ties -= min(ties, all);
    }
    if (t == 0) a.count[u] = movers;
}

__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    __shared__ MoveLds lds;
    const int unit = blockIdx.y, b = blockIdx.z, m0 = blockIdx.x * kMoveChunk;
    const int64_t u = (int64_t)b * gridDim.y + unit;
    // new_lens may be lens: no other thread of the launch reads either
    if (!a.write_lens && blockIdx.x == 0 && unit == 0 && threadIdx.x == 0)
        a.new_lens[b] = evict_len(a.lens[b], a.keep, a.max_seq);
    const int n = min(kMoveChunk, a.count[u] - m0);
    if (n > 0) evict_move(lds, a, b, unit, n, [&](int i) { return a.moves[u * a.max_moves + m0 + i]; });
}

__global__ __launch_bounds__(256) void evict_lens_kernel(const int32_t* lens, int32_t* new_lens, int batch, int keep,
                                                         int max_seq) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= batch) return;
    new_lens[b] = evict_len(lens[b], keep, max_seq);
}

// Moves that the selecting workgroup makes itself, without the second launch and its chain of loads
// (cuts of at most 64 tokens of 16 requests, 12 layers x 3 KV heads: 22.4 us so, 27.7 + 11.1 with
// moves of their own, before the selection was quicker). More moves are worth more workgroups.
constexpr int kFusedMoves = 128;

template <bool FUSE>
bool launch_select(const EvictArgs& a, dim3 grid, hipStream_t stream) {
#define CRUCIBLE_EVICT(T, R)                                                                              \
    if (a.max_seq <= T * R) {                                                                             \
        hipLaunchKernelGGL((evict_select_kernel<T, R, FUSE>), grid, dim3(T), 0, stream, a);               \
        return true;                                                                                      \
    }
    CRUCIBLE_EVICT(256, 1)
    CRUCIBLE_EVICT(256, 2)
    CRUCIBLE_EVICT(256, 3)
    CRUCIBLE_EVICT(256, 4)
    CRUCIBLE_EVICT(256, 5)
    CRUCIBLE_EVICT(256, 6)
    CRUCIBLE_EVICT(256, 8)
    CRUCIBLE_EVICT(256, 16)
    CRUCIBLE_EVICT(1024, 8)
    CRUCIBLE_EVICT(1024, 12)
    CRUCIBLE_EVICT(1024, 16)
    if constexpr (!FUSE) {
        CRUCIBLE_EVICT(1024, 24)
        CRUCIBLE_EVICT(1024, 32)
        hipLaunchKernelGGL(evict_select_long_kernel, grid, dim3(1024), 0, stream, a);
        return true;
    }
#undef CRUCIBLE_EVICT
    return false;
}

int64_t evict_moves(int64_t max_seq, int64_t keep) {
    const int64_t over = max_seq > keep ? max_seq - keep : 0;
    return over < keep ? over : keep;
}

int check_weights(const char* what, int64_t requests, int64_t n_head, int64_t n_kv_head, int64_t head_dim,
                  int64_t table_stride, int64_t kv_dim) {
    CRUCIBLE_CHECK(requests >= 0 && requests <= 65535 && table_stride > 0 &&
                       table_stride <= kMaxTablePages,
                   CRUCIBLE_ERR_INVALID, "%s: requests=%lld table_stride=%lld", what, (long long)requests,
                   (long long)table_stride);
    CRUCIBLE_CHECK(n_head > 0 && n_kv_head > 0 && n_head <= (1 << 20) && n_head % n_kv_head == 0,
                   CRUCIBLE_ERR_INVALID, "%s: n_head %lld must be a positive multiple of n_kv_head %lld", what,
                   (long long)n_head, (long long)n_kv_head);
    CRUCIBLE_CHECK(generic_head_dim_ok(head_dim), CRUCIBLE_ERR_UNSUPPORTED,
                   "%s: head_dim %lld unsupported (a multiple of 8 up to 256)", what, (long long)head_dim);
    CRUCIBLE_CHECK(kv_dim == n_kv_head * head_dim, CRUCIBLE_ERR_INVALID,
                   "%s: kv_dim %lld != n_kv_head * head_dim", what, (long long)kv_dim);
    return CRUCIBLE_OK;
}

bool misaligned16(const void* p) { return ((uintptr_t)p & 15) != 0; }

}  // namespace
}  // namespace crucible

using namespace crucible;

extern "C" size_t crucible_cache_weigh_workspace_bytes(int64_t requests, int64_t max_chunk, int64_t table_stride,
                                                       int64_t n_head, int64_t n_kv_head, int64_t head_dim,
                                                       int64_t n_observe) {
    if (requests <= 0 || requests > 65535 || max_chunk <= 0 || max_chunk > INT32_MAX || table_stride <= 0 ||
        table_stride > kMaxTablePages || n_head <= 0 || n_head > (1 << 20) || n_kv_head <= 0 ||
        n_head % n_kv_head || !generic_head_dim_ok(head_dim) || n_observe <= 0)
        return 0;
    ObserveShape s;
    if (!observe_shape(s, requests, max_chunk, n_head, n_kv_head, head_dim, table_stride, n_observe)) return 0;
    return observe_bytes(s);
}

extern "C" int crucible_cache_weigh_tiled(const void* q, int q_dtype, const void* k_pool, float* w_pool,
                                          int32_t* pos_pool, const int32_t* tables, const int32_t* segments,
                                          const int32_t* positions, int64_t requests, int64_t max_chunk,
                                          int64_t table_stride, int64_t n_head, int64_t n_kv_head, int64_t head_dim,
                                          int64_t n_layer, int64_t layer, int64_t kv_dim, int64_t n_observe,
                                          void* workspace, size_t workspace_bytes, crucible_stream_t stream) {
    const char* what = "cache_weigh_tiled";
    if (int rc = check_weights(what, requests, n_head, n_kv_head, head_dim, table_stride, kv_dim)) return rc;
    CRUCIBLE_CHECK(dtype_ok(q_dtype), CRUCIBLE_ERR_INVALID, "%s: bad dtype", what);
    CRUCIBLE_CHECK(max_chunk >= 0 && max_chunk <= INT32_MAX && n_observe >= 0 && n_observe <= INT32_MAX,
                   CRUCIBLE_ERR_INVALID, "%s: rows=%lld n_observe=%lld", what, (long long)max_chunk,
                   (long long)n_observe);
    PoolAddr addr;
    CRUCIBLE_CHECK(paged_addr(n_layer, layer, kv_dim, addr), CRUCIBLE_ERR_INVALID, "%s: layer %lld of %lld", what,
                   (long long)layer, (long long)n_layer);
    if (requests == 0 || max_chunk == 0) return CRUCIBLE_OK;
    CRUCIBLE_CHECK(q && k_pool && w_pool && pos_pool && tables && segments && positions, CRUCIBLE_ERR_INVALID,
                   "%s: null buffer", what);
    CRUCIBLE_CHECK(!misaligned16(k_pool), CRUCIBLE_ERR_INVALID, "%s: pools must be 16-byte aligned", what);
    ObserveShape s;
    CRUCIBLE_CHECK(observe_shape(s, requests, max_chunk, n_head, n_kv_head, head_dim, table_stride, n_observe),
                   CRUCIBLE_ERR_INVALID, "%s: %lld requests of %lld rows and %lld heads are past the grid", what,
                   (long long)requests, (long long)max_chunk, (long long)n_head);
    const size_t need = s.columns ? observe_bytes(s) : 0;
    CRUCIBLE_CHECK(need == 0 || (workspace && workspace_bytes >= need), CRUCIBLE_ERR_WORKSPACE,
                   "%s: workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : 0, need);
    CRUCIBLE_CHECK(need == 0 || !misaligned16(workspace), CRUCIBLE_ERR_INVALID,
                   "%s: workspace must be 16-byte aligned", what);
    ObserveArgs a{};
    a.q = q;
    a.k_pool = static_cast<const half_t*>(k_pool);
    a.w_pool = w_pool;
    a.pos_pool = pos_pool;
    a.tables = tables;
    a.segments = segments;
    a.positions = positions;
    a.addr = addr;
    a.addr.kv_dim = (int32_t)kv_dim;
    a.n_head = (int)n_head;
    a.n_kv_head = (int)n_kv_head;
    a.group = (int)(n_head / n_kv_head);
    a.max_chunk = (int)max_chunk;
    a.table_stride = (int)table_stride;
    a.max_seq = (int)(table_stride * kPageTokens);
    a.n_observe = (int)n_observe;
    a.n_layer = (int)n_layer;
    a.layer = (int)layer;
    a.head_dim = (int)head_dim;
    a.n_tiles = s.n_tiles;
    a.split_pages = s.split_pages;
    a.n_splits = s.n_splits;
    a.columns = (int)s.columns;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)head_dim));
    if (need) {
        a.frag = static_cast<half8_t*>(workspace);
        a.norm = reinterpret_cast<float4*>(a.frag + s.frag);
        a.part = reinterpret_cast<float2*>(a.norm + s.norm);
    }
    const bool f32 = q_dtype == CRUCIBLE_F32;
    const int r = (int)requests;
    switch (wide_dim(head_dim)) {
        case 32: launch_observe_hd<32>(a, f32, s, r, stream); break;
        case 64: launch_observe_hd<64>(a, f32, s, r, stream); break;
        case 96: launch_observe_hd<96>(a, f32, s, r, stream); break;
        case 128: launch_observe_hd<128>(a, f32, s, r, stream); break;
        case 160: launch_observe_hd<160>(a, f32, s, r, stream); break;
        case 192: launch_observe_hd<192>(a, f32, s, r, stream); break;
        case 224: launch_observe_hd<224>(a, f32, s, r, stream); break;
        default: launch_observe_hd<256>(a, f32, s, r, stream); break;
    }
    return fail_launch(what);
}

extern "C" size_t crucible_cache_evict_workspace_bytes(int64_t batch, int64_t n_kv_head, int64_t n_layer,
                                                       int64_t max_seq, int64_t keep) {
    const int64_t units = checked_mul(batch, n_kv_head, n_layer);
    if (units < 0 || units > INT64_MAX / 16) return SIZE_MAX;
    if (units == 0 || max_seq <= 0 || max_seq > kMaxTablePages * kPageTokens || keep < 0) return 0;
    const int64_t each = checked_mul(units, evict_moves(max_seq, keep), sizeof(int2));
    const int64_t counts = (units * (int64_t)sizeof(int32_t) + 15) / 16 * 16;
    if (each < 0 || each > INT64_MAX - counts) return SIZE_MAX;
    return (size_t)(each + counts);
}

extern "C" int crucible_cache_evict_paged(void* k_pool, void* v_pool, float* w_pool, int32_t* pos_pool,
                                          const int32_t* page_tables, const int32_t* seq_lens, int32_t* new_lens,
                                          int64_t batch, int64_t n_kv_head, int64_t head_dim, int64_t table_stride,
                                          int64_t n_layer, int64_t kv_dim, int64_t max_seq, int64_t keep,
                                          int64_t n_sink, int64_t n_recent, void* workspace, size_t workspace_bytes,
                                          crucible_stream_t stream) {
    const char* what = "cache_evict_paged";
    if (int rc = check_weights(what, batch, n_kv_head, n_kv_head, head_dim, table_stride, kv_dim)) return rc;
    PoolAddr addr;
    CRUCIBLE_CHECK(paged_addr(n_layer, 0, kv_dim, addr) && n_layer * n_kv_head <= 65535, CRUCIBLE_ERR_INVALID,
                   "%s: n_layer %lld x %lld KV heads", what, (long long)n_layer, (long long)n_kv_head);
    CRUCIBLE_CHECK(max_seq > 0 && max_seq <= table_stride * kPageTokens, CRUCIBLE_ERR_INVALID,
                   "%s: max_seq %lld past the table's %lld pages", what, (long long)max_seq,
                   (long long)table_stride);
    CRUCIBLE_CHECK(keep > 0 && keep <= INT32_MAX && n_sink >= 0 && n_recent >= 0 && n_sink <= keep &&
                       n_recent <= keep - n_sink,
                   CRUCIBLE_ERR_INVALID, "%s: keep %lld must hold %lld first and %lld newest tokens", what,
                   (long long)keep, (long long)n_sink, (long long)n_recent);
    if (batch == 0) return CRUCIBLE_OK;
    CRUCIBLE_CHECK(k_pool && v_pool && w_pool && pos_pool && page_tables && seq_lens && new_lens,
                   CRUCIBLE_ERR_INVALID, "%s: null buffer", what);
    CRUCIBLE_CHECK(!misaligned16(k_pool), CRUCIBLE_ERR_INVALID, "%s: pools must be 16-byte aligned", what);
    EvictArgs a{};
    a.k_pool = static_cast<half_t*>(k_pool);
    a.v_pool = static_cast<half_t*>(v_pool);
    a.w_pool = w_pool;
    a.pos_pool = pos_pool;
    a.tables = page_tables;
    a.lens = seq_lens;
    a.new_lens = new_lens;
    a.n_kv_head = (int)n_kv_head;
    a.head_dim = (int)head_dim;
    a.kv_dim = (int)kv_dim;
    a.table_stride = (int)table_stride;
    a.n_layer = (int)n_layer;
    a.max_seq = (int)max_seq;
    a.keep = (int)keep;
    a.n_sink = (int)n_sink;
    a.n_recent = (int)n_recent;
    a.max_moves = (int)evict_moves(max_seq, keep);
    const int units = (int)(n_layer * n_kv_head);
    if (a.max_moves > 0) {
        const size_t need = crucible_cache_evict_workspace_bytes(batch, n_kv_head, n_layer, max_seq, keep);
        CRUCIBLE_CHECK(workspace && workspace_bytes >= need, CRUCIBLE_ERR_WORKSPACE,
                       "%s: workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : 0, need);
        CRUCIBLE_CHECK(!misaligned16(workspace), CRUCIBLE_ERR_INVALID, "%s: workspace must be 16-byte aligned", what);
        a.count = static_cast<int32_t*>(workspace);
        a.moves = reinterpret_cast<int2*>(static_cast<char*>(workspace) + (batch * units * 4 + 15) / 16 * 16);
        a.write_lens = new_lens != seq_lens;
        const dim3 select((unsigned)units, (unsigned)batch);
        const bool fused = a.max_moves <= kFusedMoves && launch_select<true>(a, select, stream);
        if (!fused) {
            launch_select<false>(a, select, stream);
            const dim3 grid((unsigned)((a.max_moves + kMoveChunk - 1) / kMoveChunk), (unsigned)units, (unsigned)batch);
            hipLaunchKernelGGL(evict_move_kernel, grid, dim3(256), 0, stream, a);
            return fail_launch(what);
        }
        if (a.write_lens) return fail_launch(what);
        // in place: only when every workgroup has read its request's length
    }
    hipLaunchKernelGGL(evict_lens_kernel, dim3((unsigned)((batch + 255) / 256)), dim3(256), 0, stream, seq_lens,
                       new_lens, (int)batch, (int)keep, (int)max_seq);
    return fail_launch(what);
}
