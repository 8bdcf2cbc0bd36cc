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

// Upper bound of SpanPages::count for `rows` neighbouring rows of a table of `pages` pages.
inline int64_t span_pages_bound(int64_t window, int64_t n_sink, int64_t rows, int64_t pages) {
    const int64_t n = (n_sink + kPageMask) / kPageTokens + (window + rows + kPageMask) / kPageTokens + 1;
    return n < pages ? n : pages;
}

// K operands of two pages in the order above.
template <int HD>
struct SpanKeys {
    half8_t k[2][HD / 32];

    // base: element offset of the (page, layer) block that row `col` of the tiles lies in
    __device__ __forceinline__ void load(const half_t* kp, int64_t base, int kv_dim, int head_off, int col,
                                         int grp) {
        const int slot = 8 * ((col >> 2) & 1) + (col & 3);
        const half_t* kb = kp + base + slot * kv_dim + head_off + 8 * grp;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < HD / 32; ++i)
                k[t][i] = *reinterpret_cast<const half8_t*>(kb + 4 * t * kv_dim + 32 * i);
    }
};

// V^T operands of two pages: 8 slots of the page that the lane group covers.
template <int HD>
struct SpanValues {
    half8_t v[HD / 16];

    __device__ __forceinline__ void load(const half_t* vp, int64_t base, int head_off, int col, int grp) {
        const half_t* vb = vp + base + (head_off + col) * kPageTokens + 8 * (grp & 1);
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
            v[i] = *reinterpret_cast<const half8_t*>(vb + 16 * kPageTokens * i);
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
template <int HD, bool F32>
__device__ __forceinline__ void span_scores(float4_t (&s)[2], const HdQuery<HD, F32>& q, const SpanKeys<HD>& kv) {
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
template <int HD>
__device__ __forceinline__ void span_accumulate(HdState<HD>& st, float4_t (&s)[2], float scale,
                                                const SpanValues<HD>& kv) {
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
// barriers: any multiple of 8 up to 256 as head_dim, any alignment of q and out, and no product
// with a masked value, whatever it holds. `q` is element 0 of the query row. score(j, s) is called
// with each seen token's score in log2 units; the result is (m, l) and, through store(d, value), o.
// Blocks of 16 pages: a thread scores a token, then sums a dimension.
template <class Score, class Store>
__device__ void span_row(RowLds& lds, const void* q, bool q_f32, const half_t* k_pool, const half_t* v_pool,
                         const PoolAddr& addr, const int32_t* table, int g, int hd, const SpanMask& mask, int p,
                         float scale_log2, float& m_out, float& l_out, Score score, Store store) {
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
                score(j, s);
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
    m_out = m;
    l_out = l;
    if (t < hd) store(t, sp.count == 0 || l == 0.0f ? 0.0f : o / l);
    __syncthreads();
}

}  // namespace crucible
