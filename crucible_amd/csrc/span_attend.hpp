// Attention over a span of a paged cache: the first tokens ("sinks") and a window of the newest.
//
// A row at position p sees token j where  j <= p  and  (j < n_sink  or  p - j < window):
//   o = sum_j softmax_j(q . k_j / sqrt(head_dim)) v_j,   0 for a row that sees nothing.
// The pages between the sinks and the window are not read, and neither are their table entries:
// a caller may have given them back.
//
// 16 columns of a 16x16x32 f16 product are 16 (row, query head) pairs of one KV head, rows
// outermost: the heads of a GQA group share each K/V byte, and so do neighbouring rows. A step
// takes two pages, 32 keys, with keys and values in the order that leaves nothing to move between
// lanes: row r of score tile t is key 8 (r / 4) + 4 t + r % 4 of the pair, so lane (col, grp) ends
// with the scores of keys 8 grp .. + 7, which are the k range that it supplies to the V^T . P^T
// product and 16 contiguous bytes of each V^T row. Sums, maxima and the softmax are f32; P and an
// f32 query enter the products as fp16 hi + lo (about 22 bits).
#pragma once

#include "hd_attend.hpp"

namespace crucible {

// Pages of a table, at most: positions, and what is a few pages past them, stay within 31 bits.
constexpr int64_t kMaxTablePages = (int64_t)1 << 26;

// What a row sees.
struct SpanMask {
    int window, n_sink;
    __device__ __forceinline__ bool sees(int p, int j) const {
        return j <= p && (j < n_sink || p - j < window);
    }
};

// The pages that rows at positions p0 .. p1 see: [0, n_head) and [first, last], by index.
struct SpanPages {
    int n_head, first, count;
    int lo;  // the first key of the windows

    __device__ __forceinline__ SpanPages(const SpanMask& m, int p0, int p1) {
        const int last = p1 >> kPageShift;
        lo = p0 >= m.window ? p0 - m.window + 1 : 0;
        n_head = min((m.n_sink + kPageMask) >> kPageShift, last + 1);
        first = max(n_head, lo >> kPageShift);
        count = n_head + max(0, last - first + 1);
    }
    __device__ __forceinline__ int page(int i) const { return i < n_head ? i : first + i - n_head; }
};

// The rows of request b and where they are: segments[b] = {packed row, rows, first position,
// table}, or (no segments) row b at position lens[b] - 1.
struct SpanRows {
    int packed, rows, first;
    const int32_t* table;

    template <class Args>
    __device__ __forceinline__ SpanRows(const Args& a, int b) {
        int t = b;
        if (a.segments) {
            const int32_t* s = a.segments + 4 * (int64_t)b;
            packed = s[0];
            rows = s[1];
            first = s[2];
            t = s[3];
        } else {
            packed = b;
            rows = 1;
            first = a.lens[b] - 1;
        }
        table = a.tables + (int64_t)t * a.table_stride;
        // rows past the table, or past what the grid covers, are none of this call's
        rows = min(rows, a.max_chunk);
        if (first < 0 || packed < 0 || first > a.max_seq - rows) rows = 0;
    }
};

// Upper bound of SpanPages::count for `rows` neighbouring rows of a table of `pages` pages.
inline int64_t span_pages_bound(int64_t window, int64_t n_sink, int64_t rows, int64_t pages) {
    const int64_t n = (n_sink + kPageMask) / kPageTokens + (window + rows + kPageMask) / kPageTokens + 1;
    return n < pages ? n : pages;
}

// The head dimension: HD itself, or (PAD) any multiple of 8 below it, whose operands are 0 from
// there on. Queries and outputs start anywhere (their vector accesses ask for no alignment).
template <int HD, bool PAD>
struct SpanDim {
    int n;
    __device__ __forceinline__ int hd() const { return PAD ? n : HD; }
    __device__ __forceinline__ bool has(int d) const { return !PAD || d < n; }
};

typedef float4_t float4_any_t __attribute__((aligned(4)));
typedef half8_t half8_any_t __attribute__((aligned(2)));
typedef half4_t half4_any_t __attribute__((aligned(2)));

// 8 consecutive values of a query row as f32.
template <bool F32>
__device__ __forceinline__ void span_load8(const void* q, int64_t off, float (&x)[8]) {
    if constexpr (F32) {
        const float* p = static_cast<const float*>(q) + off;
        const float4_t a = *reinterpret_cast<const float4_any_t*>(p);
        const float4_t b = *reinterpret_cast<const float4_any_t*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = a[i];
            x[4 + i] = b[i];
        }
    } else {
        const half8_t a = *reinterpret_cast<const half8_any_t*>(static_cast<const half_t*>(q) + off);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
    }
}

// The query of a column as operands; `off` is its element 0, on: whether the column holds a row.
template <int HD, bool F32, bool PAD>
__device__ __forceinline__ void span_query(HdQuery<HD, F32>& out, const SpanDim<HD, PAD>& dim, const void* q,
                                           int64_t off, bool on, int grp, float scale_log2) {
    float x[HD / 32][8];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
        if (on && dim.has(32 * i + 8 * grp)) span_load8<F32>(q, off + 32 * i + 8 * grp, x[i]);
    }
    out.set(x, scale_log2);
}

// K operands of two pages in the order above.
template <int HD, bool PAD>
struct SpanKeys {
    half8_t k[2][HD / 32];

    // base: element offset of the (page, layer) block that row `col` of the tiles lies in
    __device__ __forceinline__ void load(const SpanDim<HD, PAD>& dim, const half_t* kp, int64_t base, int kv_dim,
                                         int head_off, int col, int grp) {
        const int slot = 8 * ((col >> 2) & 1) + (col & 3);
        const half_t* kb = kp + base + slot * kv_dim + head_off + 8 * grp;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                if (PAD) k[t][i] = half8_t{};
                if (dim.has(32 * i + 8 * grp))
                    k[t][i] = *reinterpret_cast<const half8_t*>(kb + 4 * t * kv_dim + 32 * i);
            }
    }
};

// V^T operands of two pages: 8 slots of the page that the lane group covers.
template <int HD, bool PAD>
struct SpanValues {
    half8_t v[HD / 16];

    __device__ __forceinline__ void load(const SpanDim<HD, PAD>& dim, const half_t* vp, int64_t base, int head_off,
                                         int col, int grp) {
        const half_t* vb = vp + base + (head_off + col) * kPageTokens + 8 * (grp & 1);
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            if (PAD) v[i] = half8_t{};
            if (dim.has(16 * i + col)) v[i] = *reinterpret_cast<const half8_t*>(vb + 16 * kPageTokens * i);
        }
    }
    // Slots that no row sees may hold anything, NaN included, and 0 * NaN is NaN: they become 0.
    // `key`: the first of the lane's 8.
    __device__ __forceinline__ void zero_unseen(const SpanMask& m, const SpanPages& sp, int p1, int key) {
        uint32_t keep[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t bits = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int j = key + 2 * w + e;
                if (j <= p1 && (j < m.n_sink || j >= sp.lo)) bits |= 0xffffu << (16 * e);
            }
            keep[w] = bits;
        }
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            u32x4_t x = __builtin_bit_cast(u32x4_t, v[i]);
#pragma unroll
            for (int w = 0; w < 4; ++w) x[w] &= keep[w];
            v[i] = __builtin_bit_cast(half8_t, x);
        }
    }
};

// The scores of a pair for one column block: s[t][r] is the lane's key 4 t + r.
template <int HD, bool F32, bool PAD>
__device__ __forceinline__ void span_scores(float4_t (&s)[2], const HdQuery<HD, F32>& q,
                                            const SpanKeys<HD, PAD>& kv) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        s[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            s[t] = mfma_16x16x32(kv.k[t][i], q.hi[i], s[t]);
            if constexpr (F32) s[t] = mfma_16x16x32(kv.k[t][i], q.lo[i], s[t]);
        }
    }
}

// Scores of fp16 hi + lo halves are not what f32 sums give where an operand is infinite (an infinity
// times a lo half of 0 is NaN). Where any of a wave's scores is not finite, its lanes sum theirs
// again, plainly. `base`: the block of the lane's 8 keys; `off`: element 0 of its column's query.
template <int HD, bool F32, bool PAD>
__device__ __forceinline__ void span_exact_scores(float4_t (&s)[2], const HdQuery<HD, F32>& q,
                                                  const SpanDim<HD, PAD>& dim, const void* qs, const half_t* kp,
                                                  int64_t base, int kv_dim, int head_off, bool on, int64_t off,
                                                  int grp, float scale_log2, bool q_f32) {
    float z = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) z = __builtin_fmaf(s[t][r], 0.0f, z);
    if (__ballot(!(z == 0.0f)) == 0) return;
    if (!on) return;
    const float up = scale_log2 / q.scale;  // a power of two
    for (int e = 0; e < 8; ++e) {
        const half_t* kr = kp + base + (8 * (grp & 1) + e) * kv_dim + head_off;
        float acc = 0.0f;
        for (int d = 0; d < dim.hd(); ++d) {
            const float x = q_f32 ? static_cast<const float*>(qs)[off + d]
                                  : (float)static_cast<const half_t*>(qs)[off + d];
            acc = __builtin_fmaf(x * up, (float)kr[d], acc);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (e == 4 * t + r) s[t][r] = acc;
    }
}

// In place: masked scores of a row at position p become -inf. `key`: the lane's first.
__device__ __forceinline__ void span_mask(float4_t (&s)[2], const SpanMask& m, int p, int key) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (!m.sees(p, key + 4 * t + r)) s[t][r] = -INFINITY;
}

// One pair of values under scores s (not yet scaled) into a column block's state. s comes back
// in log2 units. State sums are the lane's own until hd_merge_waves.
template <int HD, bool PAD>
__device__ __forceinline__ void span_accumulate(HdState<HD>& st, float4_t (&s)[2], float scale,
                                                const SpanValues<HD, PAD>& kv) {
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma clang fp contract(off)
            s[t][r] = s[t][r] * scale;  // once, so that the largest minus the maximum is exactly 0
            mx = fmaxf(mx, s[t][r]);
        }
    const float mn = fmaxf(st.m, group_max4(mx));
    const float at = mn == -INFINITY ? 0.0f : mn;
    const float alpha = fast_exp2(st.m - at);
    st.m = mn;
    u32x4_t hw, lw;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        float pf[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) pf[r] = fast_exp2(s[t][r] - at);
        sum += (pf[0] + pf[1]) + (pf[2] + pf[3]);
        const uint32_t h01 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(pf[0], pf[1]));
        const uint32_t h23 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(pf[2], pf[3]));
        uint32_t l01, l23;
        split_lo4(pf, h01, h23, l01, l23);
        hw[2 * t] = h01;
        hw[2 * t + 1] = h23;
        lw[2 * t] = l01;
        lw[2 * t + 1] = l23;
    }
    st.l = __builtin_fmaf(st.l, alpha, sum);
    const half8_t ph = __builtin_bit_cast(half8_t, hw), pl = __builtin_bit_cast(half8_t, lw);
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
        st.o[i] = mfma_16x16x32(kv.v[i], ph, st.o[i] * alpha);
        st.o[i] = mfma_16x16x32(kv.v[i], pl, st.o[i]);
    }
}

// ---------------------------------------------------------------- one row, plainly

constexpr int kRowThreads = 256;

struct RowLds {
    alignas(16) float q[256];
    float p[kRowThreads];
    float red[kRowThreads / 64];
};

template <bool MAX>
__device__ __forceinline__ float row_reduce(RowLds& lds, float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float w = __shfl_xor(v, off);
        v = MAX ? fmaxf(v, w) : v + w;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0 && threadIdx.x < kRowThreads) lds.red[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = lds.red[0];
#pragma unroll
    for (int w = 1; w < kRowThreads / 64; ++w) r = MAX ? fmaxf(r, lds.red[w]) : r + lds.red[w];
    return r;
}

// One (row, query head) by the whole workgroup, whose threads past kRowThreads only pass the
// barriers, without a product with a masked value, whatever it holds. `q` is element 0 of the query
// row; the result is o, through store(d, value). Blocks of 16 pages: a thread scores a token, then
// sums a dimension.
template <class Store>
__device__ void span_row(RowLds& lds, const void* q, bool q_f32, const half_t* k_pool, const half_t* v_pool,
                         const PoolAddr& addr, const int32_t* table, int g, int hd, const SpanMask& mask, int p,
                         float scale_log2, Store store) {
    const int t = threadIdx.x;
    __syncthreads();
    for (int d = t; d < hd; d += blockDim.x)
        lds.q[d] = q_f32 ? static_cast<const float*>(q)[d] : (float)static_cast<const half_t*>(q)[d];
    __syncthreads();
    const SpanPages sp(mask, p, p);
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int i0 = 0; i0 < sp.count; i0 += kRowThreads / kPageTokens) {
        const int i = i0 + (t >> kPageShift);
        float s = -INFINITY;
        bool seen = false;
        if (i < sp.count && t < kRowThreads) {
            const int page = sp.page(i), j = page * kPageTokens + (t & kPageMask);
            seen = mask.sees(p, j);
            if (seen) {
                const half_t* kr = k_pool + block_base(addr, table[page]) + (t & kPageMask) * addr.kv_dim + g * hd;
                float acc = 0.0f;
                for (int d = 0; d < hd; d += 8) {
                    const half8_t k8 = *reinterpret_cast<const half8_t*>(kr + d);
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc = __builtin_fmaf(lds.q[d + e], (float)k8[e], acc);
                }
                s = acc * scale_log2;
            }
        }
        const float mn = fmaxf(m, row_reduce<true>(lds, s));
        const float at = mn == -INFINITY ? 0.0f : mn;
        const float w = seen ? fast_exp2(s - at) : 0.0f;
        const float alpha = fast_exp2(m - at);
        l = l * alpha + row_reduce<false>(lds, w);
        m = mn;
        if (t < kRowThreads) lds.p[t] = seen ? w : -1.0f;  // -1: not seen (a weight is never below 0)
        __syncthreads();
        if (t < hd) {
            o *= alpha;
            for (int pp = 0; pp < kRowThreads / kPageTokens && i0 + pp < sp.count; ++pp) {
                const half_t* vr = v_pool + block_base(addr, table[sp.page(i0 + pp)]) +
                                   (int64_t)(g * hd + t) * kPageTokens;
                const half8_t v0 = *reinterpret_cast<const half8_t*>(vr);
                const half8_t v1 = *reinterpret_cast<const half8_t*>(vr + 8);
#pragma unroll
                for (int e = 0; e < kPageTokens; ++e) {
                    const float w = lds.p[pp * kPageTokens + e];
                    if (!(w < 0.0f)) o = __builtin_fmaf(w, (float)(e < 8 ? v0[e] : v1[e - 8]), o);
                }
            }
        }
        __syncthreads();
    }
    if (t < hd) store(t, l == 0.0f ? 0.0f : o / l);
    __syncthreads();
}

}  // namespace crucible
