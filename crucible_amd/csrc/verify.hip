// Drafted tokens against the target's probabilities, from given random numbers.
//
// With p_i = softmax(target_i / T) and q_i = softmax(draft_i / T) (or, without draft logits, all of
// q_i on the drafted token), draft t_i is taken while  u_i q_i(t_i) < p_i(t_i). At the first refusal
// the next token comes from max(p_i - q_i, 0), and past the last draft from p_n: the lowest t whose
// running sum of that mass exceeds u * total. A token so drawn has the target's distribution.
// No counterpart in the reference, whose selection is greedy (argmax.hip).
//
// Every probability and sum is f64: the running sum passes 50,000 borders that are 2e-5 apart on
// average, and a border moved by f32 rounding (6e-8 a term) would change the token of one draw in
// a few hundred. A NaN logit counts as -inf; an infinite one takes all.
//
// Two launches. verify_sums_kernel: maximum and sum of exponentials of each row's chunks of
// columns. verify_pick_kernel: every workgroup joins its request's rows and finds what is taken;
// after a refusal each sums max(p - q, 0) over one chunk, and the last of a request to do so finds
// the chunk in which the running sum passes the border, then the token in it. (After none, the
// chunks' sums of p_n are known and the first workgroup does.)
//
// Bound: 96 MB of logits (32 requests of up to 7 drafts, 50,257 columns) are 20 us at the rate of a
// copy, their 24 million exponentials in f64 about 10 us of the vector units.
#include "common.hpp"

namespace crucible {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxDrafts = 64;
constexpr int kTable = 64;  // entries of exp64's table

constexpr int kChunk = kThreads * 4;  // columns

struct Part {
    double sum;
    double top;  // a float's value
};

struct VerifyArgs {
    const void* target;  // [batch][drafts + 1][vocab]
    const void* draft;   // [batch][drafts][vocab], or null
    const int32_t* drafts;
    const int32_t* n_draft;
    const float* u_accept;
    const float* u_sample;
    int32_t* tokens;
    int32_t* accepted;
    int32_t k, vocab, chunks, f16;
    double inv_t;
    Part* parts;      // [batch][target rows, then draft rows][chunk]
    double* mass;     // [batch][chunk]
    uint32_t* count;  // [batch] chunks summed: cleared by the first launch
    float* drafted;   // [batch][target rows, then draft rows] the drafted token's logit
};

__device__ __forceinline__ float logit(const VerifyArgs& a, const void* x, int64_t i) {
    const float v = a.f16 ? (float)static_cast<const half_t*>(x)[i] : static_cast<const float*>(x)[i];
    return v == v ? v : -INFINITY;
}

// exp(x), x <= 0, in f64: x = (64 e + j) ln 2 / 64 + r, |r| <= ln 2 / 128, so that
// exp(x) = 2^e 2^(j / 64) exp(r) with six terms of the series, the first left out r^6 / 720 < 4e-17.
// 12 f64 operations where the library's exp is some 35; the sums' kernel is bound by them.
struct Exp64 {
    const double* table;  // 2^(j / 64), in LDS

    static __device__ __forceinline__ void fill(double (&t)[kTable]) {
        if (threadIdx.x < kTable) t[threadIdx.x] = exp2((double)threadIdx.x / kTable);
    }
    __device__ __forceinline__ double operator()(double x) const {
        x = fmax(x, -800.0);  // 0 from -746 on, whatever the temperature
        const double n = __builtin_rint(x * (kTable * 1.4426950408889634));
        double r = __builtin_fma(n, -0x1.62e42fefap-1 / kTable, x);  // 36 bits: n times it is exact
        r = __builtin_fma(n, -0x1.cf79abc9e3b39p-40 / kTable, r);
        const int i = (int)n;
        double p = __builtin_fma(r, 1.0 / 120, 1.0 / 24);
        p = __builtin_fma(r, p, 1.0 / 6);
        p = __builtin_fma(r, p, 0.5);
        p = __builtin_fma(r, p, 1.0);
        const double t = table[i & (kTable - 1)];
        return __builtin_amdgcn_ldexp(__builtin_fma(t * r, p, t), i >> 6);
    }
};

// exp((x - top) / T) of a logit x <= top; the top itself is 1 and -inf is 0, also where they are infinite
__device__ __forceinline__ double weight(const Exp64& e, float x, float top, double inv_t) {
    if (x == -INFINITY) return 0.0;
    if (x == top) return 1.0;
    return e(((double)x - (double)top) * inv_t);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) { return min(a.n_draft[b], a.k); }

// Four logits of a row from column c on (none past the row), -inf for NaN.
__device__ __forceinline__ void load4(const VerifyArgs& a, const void* x, int64_t base, int c, float (&v)[4]) {
    if (c + 4 <= a.vocab) {
        if (a.f16) {
            typedef half4_t half4_any_t __attribute__((aligned(2)));
            const half4_t y = *reinterpret_cast<const half4_any_t*>(static_cast<const half_t*>(x) + base + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)y[e];
        } else {
            typedef float4_t float4_any_t __attribute__((aligned(4)));
            const float4_t y = *reinterpret_cast<const float4_any_t*>(static_cast<const float*>(x) + base + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = y[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = v[e] == v[e] ? v[e] : -INFINITY;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < a.vocab ? logit(a, x, base + c + e) : -INFINITY;
    }
}

// grid (U chunks, row of 2 k + 1, request): with U = 4 a workgroup, which starts with a chain of
// loads, reads four times as much behind it
template <int U>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a) {
    __shared__ float top_red[kWaves];
    __shared__ double red[U][kWaves], table[kTable];
    const int row = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
    const int n = drafts_of(a, b);
    if (blockIdx.x == 0 && row == 0 && t == 0) a.count[b] = 0;
    const bool is_draft = row > a.k;
    const int i = is_draft ? row - a.k - 1 : row;
    if (n < 0 || (is_draft ? i >= n : i > n)) return;
    const int token = i < n ? a.drafts[(int64_t)b * a.k + i] : -1;
    const void* x = is_draft ? a.draft : a.target;
    const int64_t base = (is_draft ? (int64_t)b * a.k + i : (int64_t)b * (a.k + 1) + i) * a.vocab;
    float v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
        load4(a, x, base, (blockIdx.x * U + u) * kChunk + 4 * t, v[u]);
    Exp64::fill(table);
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            top = fmaxf(top, v[u][e]);
            const int c = (blockIdx.x * U + u) * kChunk + 4 * t + e;
            if (c == token && c < a.vocab) a.drafted[(int64_t)b * (2 * a.k + 1) + row] = v[u][e];
        }
    top = wave_max(top);
    if ((t & 63) == 0) top_red[t >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, top_red[w]);
    const Exp64 ex{table};
#pragma unroll
    for (int u = 0; u < U; ++u) {
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) s += weight(ex, v[u][e], top, a.inv_t);
        s = wave_sum(s);
        if ((t & 63) == 0) red[u][t >> 6] = s;
    }
    __syncthreads();
    const int chunk = blockIdx.x * U + t;
    if (t < U && chunk < a.chunks) {
        double s = red[t][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) s += red[t][w];
        a.parts[((int64_t)b * (2 * a.k + 1) + row) * a.chunks + chunk] = Part{s, (double)top};
    }
}

struct RowSum {
    double inv;  // 1 / sum, 0 for a row without mass
    float top;
};

struct VerifyLds {
    RowSum row[2 * kMaxDrafts + 1];
    double red[kWaves], table[kTable];
    int drafts[kMaxDrafts];
    int n;
};

// The rows' maxima and sums, and how many drafts are taken, in lds; false for an inactive request.
// Every thread calls it.
__device__ __forceinline__ bool decide(VerifyLds& lds, const VerifyArgs& a, int b, int n) {
    const int lane = threadIdx.x & 63, half = threadIdx.x >> 5, l32 = threadIdx.x & 31;
    const Exp64 ex{lds.table};
    // Half a wave a row, a lane a chunk. Every load is under way before the first wait, n's too: rows
    // past it hold anything and are not used.
    const int rows = a.draft ? 2 * a.k + 1 : a.k + 1;
    const Part none{0.0, -INFINITY};
    const Part* parts = a.parts + (int64_t)b * (2 * a.k + 1) * a.chunks;
    Part mine = none;
    if (half < rows && l32 < a.chunks) mine = parts[(int64_t)half * a.chunks + l32];
    float lp = -INFINITY, lq = -INFINITY, u = 0.0f;
    int token = -1;
    if ((int)threadIdx.x < a.k) {  // lane i of the first wave: draft i
        token = a.drafts[(int64_t)b * a.k + lane];
        u = a.u_accept[(int64_t)b * a.k + lane];
        lp = a.drafted[(int64_t)b * (2 * a.k + 1) + lane];
        if (a.draft) lq = a.drafted[(int64_t)b * (2 * a.k + 1) + a.k + 1 + lane];
        lds.drafts[lane] = token;
    }
    Exp64::fill(lds.table);
    if (n < 0) return false;
    const bool inside = (int)threadIdx.x < n && token >= 0 && token < a.vocab;
    __syncthreads();
    for (int j = half; j < rows; j += kThreads / 32) {
        if (j <= a.k ? j > n : j - a.k - 1 >= n) continue;
        const Part* p = parts + (int64_t)j * a.chunks;
        if (j != half) mine = l32 < a.chunks ? p[l32] : none;
        float top = (float)mine.top;
        for (int c = l32 + 32; c < a.chunks; c += 32) top = fmaxf(top, (float)p[c].top);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        double s = mine.sum * weight(ex, (float)mine.top, top, a.inv_t);
        for (int c = l32 + 32; c < a.chunks; c += 32) s += p[c].sum * weight(ex, (float)p[c].top, top, a.inv_t);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor(s, d);
        if (l32 == 0) lds.row[j] = RowSum{s > 0.0 ? 1.0 / s : 0.0, top};
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        bool taken = false;
        if (inside) {
            const RowSum& p = lds.row[lane];
            const double pt = weight(ex, lp, p.top, a.inv_t) * p.inv;
            double qt = 1.0;
            if (a.draft) {
                const RowSum& q = lds.row[a.k + 1 + lane];
                qt = weight(ex, lq, q.top, a.inv_t) * q.inv;
            }
            taken = (double)u * qt < pt;
        }
        const uint64_t no = ~__ballot(taken);
        if (lane == 0) lds.n = no ? min(n, (int)__builtin_ctzll(no)) : n;
    }
    __syncthreads();
    return true;
}

// The masses of four columns of the row at which the drafts end: p, or (less) max(p - q, 0).
__device__ __forceinline__ void mass4(const VerifyLds& lds, const VerifyArgs& a, int b, int row, bool less, int c,
                                      double (&m)[4]) {
// p and q are rounded before they meet: fused, the difference of equal ones would be a rounding
// error in place of 0
#pragma clang fp contract(off)
    const Exp64 ex{lds.table};
    float x[4], y[4];
    load4(a, a.target, ((int64_t)b * (a.k + 1) + row) * a.vocab, c, x);
    const RowSum p = lds.row[row];
    const bool q_row = less && a.draft;
    if (q_row) load4(a, a.draft, ((int64_t)b * a.k + row) * a.vocab, c, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = weight(ex, x[e], p.top, a.inv_t) * p.inv;
    if (q_row) {
        const RowSum q = lds.row[a.k + 1 + row];
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = fmax(m[e] - weight(ex, y[e], q.top, a.inv_t) * q.inv, 0.0);
    } else if (less) {
        const int t = lds.drafts[row];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e == t) m[e] = 0.0;
    }
}

struct PickLds {
    int chunk, token, last;
    double before, border;
    bool less, mine;
};

// The chunk in which the running sum passes the border, by the first wave. `less`: of the sums of
// max(p - q, 0), which other workgroups wrote; p's own where nothing is left over, or not less.
__device__ __forceinline__ void find_chunk(PickLds& s, const VerifyLds& lds, const VerifyArgs& a, int b, int row,
                                           bool less, float u) {
    const int lane = threadIdx.x & 63;
    const Exp64 ex{lds.table};
    const Part* parts = a.parts + ((int64_t)b * (2 * a.k + 1) + row) * a.chunks;
    const double* mass = a.mass + (int64_t)b * a.chunks;
    const RowSum p = lds.row[row];
    double first = 0.0, total = 0.0, run = 0.0, before = 0.0;  // first: the lane's of the first 64 chunks
    int at = -1, last = -1;
    for (int pass = 0; pass < 2; ++pass) {  // the total, then the place of the border
        for (int c0 = 0; c0 < a.chunks && at < 0; c0 += 64) {
            const int c = c0 + lane;
            double m = first;
            if (pass == 0 || c0 > 0) {
                m = 0.0;
                if (c < a.chunks)
                    m = less ? __hip_atomic_load(&mass[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                             : parts[c].sum * weight(ex, (float)parts[c].top, p.top, a.inv_t) * p.inv;
                if (c0 == 0) first = m;
            }
            double sum = m;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double x = __shfl_up(sum, d);
                if (lane >= d) sum += x;
            }
            if (pass == 1) {
                const uint64_t some = __ballot(m > 0.0);
                const uint64_t past = __ballot(m > 0.0 && run + sum > (double)u * total);
                if (some) last = c0 + 63 - __builtin_clzll(some);
                if (past) {
                    at = c0 + __builtin_ctzll(past);
                    before = run + __shfl(sum - m, at - c0);
                }
            }
            run += __shfl(sum, 63);
        }
        if (pass == 0) {
            total = run;
            run = 0.0;
            if (less && !(total > 0.0)) {  // nothing is left over: p decides
                less = false;
                pass = -1;
            }
        }
    }
    if (lane == 0) {
        // a border at or past the total (u near 1): the last token with any mass
        s.chunk = at >= 0 ? at : last;
        s.before = at >= 0 ? before : -INFINITY;
        s.border = (double)u * total;
        s.less = less;
        s.token = INT32_MAX;
        s.last = -1;
    }
}

// grid (chunk, request). The first pass sums a workgroup's chunk of max(p - q, 0); the second, by
// the workgroup that counts last, looks for the token in the border's chunk. A chain of waits: of
// 4 drafts' 9 us, 2.2 until the decision, 3.4 for the chunk's sum and its count, 1.5 for the chunk of
// the border, 1.9 for the token.
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a) {
    __shared__ VerifyLds lds;
    __shared__ PickLds s;
    const int b = blockIdx.y, t = threadIdx.x, lane = t & 63;
    const int n = drafts_of(a, b);
    const float u = a.u_sample[b];  // now: not after the sums
    if (!decide(lds, a, b, n)) return;
    const int row = lds.n;
    const bool refused = row < n;
    if (!refused && blockIdx.x > 0) return;  // p itself: its chunks' sums are known
    bool less = refused;
    int chunk = blockIdx.x;
    for (int pass = refused ? 0 : 1; pass < 2; ++pass) {
        if (pass == 1) {
            if (t < 64) find_chunk(s, lds, a, b, row, refused, u);
            __syncthreads();
            less = s.less;
            chunk = s.chunk;
            if (chunk < 0) break;
        }
        // the chunk's columns in order, four a thread
        const int c0 = chunk * kChunk + 4 * t;
        double m[4];
        mass4(lds, a, b, row, less, c0, m);
        const double own = (m[0] + m[1]) + (m[2] + m[3]);
        double sum = own;  // up to and with this thread, of its wave
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double x = __shfl_up(sum, d);
            if (lane >= d) sum += x;
        }
        if (lane == 63) lds.red[t >> 6] = sum;
        __syncthreads();
        if (pass == 0) {
            // The sums go out and come in past the XCDs' L2 (agent scope), and each has been
            // acknowledged before its workgroup counts: the one that counts last finds all of them.
            if (t == 0) {
                double all = 0.0;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) all += lds.red[w];
                __hip_atomic_store(&a.mass[(int64_t)b * a.chunks + chunk], all, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                s.mine = __hip_atomic_fetch_add(&a.count[b], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                         (uint32_t)a.chunks - 1;
            }
            __syncthreads();
            if (!s.mine) return;
            continue;
        }
        double run = s.before + (sum - own);
        for (int w = 0; w < t >> 6; ++w) run += lds.red[w];
        int token = INT32_MAX, last = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            run += m[e];
            if (m[e] > 0.0) {
                last = c0 + e;
                if (run > s.border) token = min(token, last);
            }
        }
        // columns rise with the lane: one atomic a wave (one a thread, 512 in a row on the same
        // word, took 5 us)
        const uint64_t found = __ballot(token != INT32_MAX), some = __ballot(last >= 0);
        if (found && lane == __builtin_ctzll(found)) atomicMin(&s.token, token);
        if (some && lane == 63 - __builtin_clzll(some)) atomicMax(&s.last, last);
    }
    __syncthreads();
    // rounding inside the chunk may leave the border unpassed: its last token then. No mass: token 0.
    const int token = s.token != INT32_MAX ? s.token : max(s.last, 0);
    for (int i = t; i <= a.k; i += kThreads)
        a.tokens[(int64_t)b * (a.k + 1) + i] = i < row ? lds.drafts[i] : i == row ? token : -1;
    if (t == 0) a.accepted[b] = row;
}

struct VerifySizes {
    int u;
    int64_t chunks, parts, mass, count, drafted;  // bytes from parts on
};

bool verify_sizes(VerifySizes& s, int64_t batch, int64_t k, int64_t vocab) {
    s.chunks = (vocab + kChunk - 1) / kChunk;
    s.u = batch * (2 * k + 1) * s.chunks > 8 * (int64_t)device_cu_count() ? 4 : 1;
    s.parts = checked_mul(batch * (2 * k + 1), s.chunks, sizeof(Part));
    s.mass = checked_mul(batch, s.chunks, sizeof(double));
    s.count = batch * (int64_t)sizeof(uint32_t);
    s.drafted = batch * (2 * k + 1) * (int64_t)sizeof(float);
    return s.parts >= 0 && s.mass >= 0 && s.parts < INT64_MAX / 4 && s.mass < INT64_MAX / 4;
}

size_t verify_bytes(const VerifySizes& s) { return (size_t)(s.parts + s.mass + s.count + s.drafted); }

template <int U>
void launch_verify(const VerifyArgs& a, unsigned rows, unsigned batch, hipStream_t stream) {
    hipLaunchKernelGGL((verify_sums_kernel<U>), dim3((unsigned)((a.chunks + U - 1) / U), rows, batch), dim3(kThreads), 0,
                       stream, a);
    hipLaunchKernelGGL(verify_pick_kernel, dim3((unsigned)a.chunks, batch), dim3(kThreads), 0, stream, a);
}

}  // namespace
}  // namespace crucible

using namespace crucible;

extern "C" size_t crucible_verify_drafts_workspace_bytes(int64_t batch, int64_t max_draft, int64_t vocab) {
    VerifySizes s;
    if (batch <= 0 || batch > 65535 || max_draft < 0 || max_draft > kMaxDrafts || vocab <= 0 ||
        vocab >= INT32_MAX - (1 << 20) || !verify_sizes(s, batch, max_draft, vocab))
        return 0;
    return verify_bytes(s);
}

extern "C" int crucible_verify_drafts(const void* target, const void* draft, int dtype, const int32_t* drafts,
                                      const int32_t* n_draft, const float* u_accept, const float* u_sample,
                                      int32_t* tokens, int32_t* accepted, int64_t batch, int64_t max_draft,
                                      int64_t vocab, double temperature, void* workspace, size_t workspace_bytes,
                                      crucible_stream_t stream) {
    const char* what = "verify_drafts";
    CRUCIBLE_CHECK(dtype_ok(dtype), CRUCIBLE_ERR_INVALID, "%s: bad dtype", what);
    CRUCIBLE_CHECK(batch >= 0 && batch <= 65535 && max_draft >= 0 && max_draft <= kMaxDrafts && vocab > 0 &&
                       vocab < INT32_MAX - (1 << 20),
                   CRUCIBLE_ERR_INVALID, "%s: batch=%lld drafts=%lld (at most %d) vocab=%lld", what, (long long)batch,
                   (long long)max_draft, kMaxDrafts, (long long)vocab);
    CRUCIBLE_CHECK(temperature > 0.0 && temperature <= 3.4e38 && temperature >= 1e-30, CRUCIBLE_ERR_INVALID,
                   "%s: temperature must be positive and finite", what);
    if (batch == 0) return CRUCIBLE_OK;
    CRUCIBLE_CHECK(target && n_draft && u_sample && tokens && accepted && (max_draft == 0 || (drafts && u_accept)),
                   CRUCIBLE_ERR_INVALID, "%s: null buffer", what);
    VerifySizes s;
    CRUCIBLE_CHECK(verify_sizes(s, batch, max_draft, vocab), CRUCIBLE_ERR_INVALID, "%s: too large", what);
    const size_t need = verify_bytes(s);
    CRUCIBLE_CHECK(workspace && workspace_bytes >= need, CRUCIBLE_ERR_WORKSPACE,
                   "%s: workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : 0, need);
    CRUCIBLE_CHECK(((uintptr_t)workspace & 15) == 0, CRUCIBLE_ERR_INVALID, "%s: workspace must be 16-byte aligned",
                   what);
    VerifyArgs a{};
    a.target = target;
    a.draft = draft;
    a.drafts = drafts;
    a.n_draft = n_draft;
    a.u_accept = u_accept;
    a.u_sample = u_sample;
    a.tokens = tokens;
    a.accepted = accepted;
    a.k = (int)max_draft;
    a.vocab = (int)vocab;
    a.chunks = (int)s.chunks;
    a.f16 = dtype == CRUCIBLE_F16;
    a.inv_t = 1.0 / temperature;
    a.parts = static_cast<Part*>(workspace);
    a.mass = reinterpret_cast<double*>(static_cast<char*>(workspace) + s.parts);
    const unsigned rows = (unsigned)(draft ? 2 * max_draft + 1 : max_draft + 1);
    a.count = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + s.parts + s.mass);
    a.drafted = reinterpret_cast<float*>(a.count + batch);
    s.u == 4 ? launch_verify<4>(a, rows, (unsigned)batch, stream) : launch_verify<1>(a, rows, (unsigned)batch, stream);
    return fail_launch(what);
}
