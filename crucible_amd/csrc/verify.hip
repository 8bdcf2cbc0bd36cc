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
// Three launches. verify_sums_kernel: maximum and sum of exponentials of each row's chunks of
// kChunk columns. verify_mass_kernel: a workgroup joins its request's rows, finds what is taken,
// and after a refusal sums max(p - q, 0) over one chunk. verify_pick_kernel: finds the chunk in
// which the running sum passes the border, then the token in it.
#include "common.hpp"

namespace crucible {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kPer = 8;  // columns of a chunk a thread
constexpr int kChunk = kThreads * kPer;
constexpr int kMaxDrafts = 64;

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
    Part* parts;   // [batch][target rows, then draft rows][chunk]
    double* mass;  // [batch][chunk]
};

__device__ __forceinline__ float logit(const VerifyArgs& a, const void* x, int64_t i) {
    const float v = a.f16 ? (float)static_cast<const half_t*>(x)[i] : static_cast<const float*>(x)[i];
    return v == v ? v : -INFINITY;
}

// exp((x - top) / T) of a logit x <= top; the top itself is 1 and -inf is 0, also where they are infinite
__device__ __forceinline__ double weight(float x, float top, double inv_t) {
    if (x == -INFINITY) return 0.0;
    if (x == top) return 1.0;
    return exp(((double)x - (double)top) * inv_t);
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

__device__ __forceinline__ double block_sum(double v, double (&red)[kWaves]) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = red[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) s += red[w];
    return s;
}

__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) { return min(a.n_draft[b], a.k); }

// grid (chunk, row of 2 k + 1, request)
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a) {
    __shared__ float top_red[kWaves];
    __shared__ double red[kWaves];
    const int row = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
    const int n = drafts_of(a, b);
    const bool is_draft = row > a.k;
    const int i = is_draft ? row - a.k - 1 : row;
    if (n < 0 || (is_draft ? i >= n : i > n)) return;
    const void* x = is_draft ? a.draft : a.target;
    const int64_t base = (is_draft ? (int64_t)b * a.k + i : (int64_t)b * (a.k + 1) + i) * a.vocab;
    const int c0 = blockIdx.x * kChunk;
    float v[kPer];
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int c = c0 + j * kThreads + t;
        v[j] = c < a.vocab ? logit(a, x, base + c) : -INFINITY;
        top = fmaxf(top, v[j]);
    }
    top = wave_max(top);
    if ((t & 63) == 0) top_red[t >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, top_red[w]);
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) s += weight(v[j], top, a.inv_t);
    s = block_sum(s, red);
    if (t == 0) a.parts[((int64_t)b * (2 * a.k + 1) + row) * a.chunks + blockIdx.x] = Part{s, (double)top};
}

struct RowSum {
    double inv;  // 1 / sum, 0 for a row without mass
    float top;
};

struct VerifyLds {
    RowSum row[2 * kMaxDrafts + 1];
    double red[kWaves];
    int n;
};

// The rows' maxima and sums, and how many drafts are taken, in lds. Every thread calls it.
__device__ __forceinline__ void decide(VerifyLds& lds, const VerifyArgs& a, int b, int n) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int row = wave; row < 2 * a.k + 1; row += kWaves) {
        const bool is_draft = row > a.k;
        if (is_draft ? !a.draft || row - a.k - 1 >= n : row > n) continue;
        const Part* p = a.parts + ((int64_t)b * (2 * a.k + 1) + row) * a.chunks;
        float top = -INFINITY;
        for (int c = lane; c < a.chunks; c += 64) top = fmaxf(top, (float)p[c].top);
        top = wave_max(top);
        double s = 0.0;
        for (int c = lane; c < a.chunks; c += 64) s += p[c].sum * weight((float)p[c].top, top, a.inv_t);
        s = wave_sum(s);
        if (lane == 0) lds.row[row] = RowSum{s > 0.0 ? 1.0 / s : 0.0, top};
    }
    __syncthreads();
    if (wave == 0) {
        // lane i: draft i
        bool taken = false;
        if (lane < n) {
            const int t = a.drafts[(int64_t)b * a.k + lane];
            if (t >= 0 && t < a.vocab) {
                const RowSum& p = lds.row[lane];
                const double pt =
                    weight(logit(a, a.target, ((int64_t)b * (a.k + 1) + lane) * a.vocab + t), p.top, a.inv_t) * p.inv;
                double qt = 1.0;
                if (a.draft) {
                    const RowSum& q = lds.row[a.k + 1 + lane];
                    qt = weight(logit(a, a.draft, ((int64_t)b * a.k + lane) * a.vocab + t), q.top, a.inv_t) * q.inv;
                }
                taken = (double)a.u_accept[(int64_t)b * a.k + lane] * qt < pt;
            }
        }
        const uint64_t no = ~__ballot(taken);
        if (lane == 0) lds.n = no ? min(n, (int)__builtin_ctzll(no)) : n;
    }
    __syncthreads();
}

// max(p - q, 0) of column c of the row at which the drafts were refused
__device__ __forceinline__ double left_over(const VerifyLds& lds, const VerifyArgs& a, int b, int row, int c) {
    const RowSum& p = lds.row[row];
    const double pc = weight(logit(a, a.target, ((int64_t)b * (a.k + 1) + row) * a.vocab + c), p.top, a.inv_t) * p.inv;
    if (!a.draft) return c == a.drafts[(int64_t)b * a.k + row] ? 0.0 : pc;
    const RowSum& q = lds.row[a.k + 1 + row];
    const double qc = weight(logit(a, a.draft, ((int64_t)b * a.k + row) * a.vocab + c), q.top, a.inv_t) * q.inv;
    return pc > qc ? pc - qc : 0.0;
}

// grid (chunk, request)
__global__ __launch_bounds__(kThreads) void verify_mass_kernel(VerifyArgs a) {
    __shared__ VerifyLds lds;
    const int b = blockIdx.y, t = threadIdx.x;
    const int n = drafts_of(a, b);
    if (n < 0) return;
    decide(lds, a, b, n);
    const int row = lds.n;
    if (row == n) return;  // p itself: its chunks' sums are known
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int c = blockIdx.x * kChunk + j * kThreads + t;
        if (c < a.vocab) s += left_over(lds, a, b, row, c);
    }
    s = block_sum(s, lds.red);
    if (t == 0) a.mass[(int64_t)b * a.chunks + blockIdx.x] = s;
}

// grid (request)
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a) {
    __shared__ VerifyLds lds;
    __shared__ int s_chunk, s_last;
    __shared__ double s_before, s_border;
    __shared__ bool s_p;
    __shared__ int s_token;
    const int b = blockIdx.x, t = threadIdx.x;
    const int n = drafts_of(a, b);
    if (n < 0) return;
    decide(lds, a, b, n);
    const int row = lds.n;
    const Part* parts = a.parts + ((int64_t)b * (2 * a.k + 1) + row) * a.chunks;
    const RowSum p = lds.row[row];
    if (t == 0) {
        const double* mass = a.mass + (int64_t)b * a.chunks;
        double total = 0.0;
        if (row < n)
            for (int c = 0; c < a.chunks; ++c) total += mass[c];
        s_p = !(total > 0.0);  // also where nothing is left over
        const auto chunk = [&](int c) {
            return s_p ? parts[c].sum * weight((float)parts[c].top, p.top, a.inv_t) * p.inv : mass[c];
        };
        if (s_p) {
            total = 0.0;
            for (int c = 0; c < a.chunks; ++c) total += chunk(c);
        }
        const double border = (double)a.u_sample[b] * total;
        double run = 0.0, before = 0.0;
        int at = -1, last = -1;
        for (int c = 0; c < a.chunks; ++c) {
            const double m = chunk(c);
            if (m > 0.0) last = c;
            if (at < 0 && run + m > border) {
                at = c;
                before = run;
            }
            run += m;
        }
        // a border at or past the total (u near 1): the last token with any mass
        s_chunk = at >= 0 ? at : last;
        s_before = at >= 0 ? before : -INFINITY;
        s_border = at >= 0 ? border : INFINITY;
        s_token = INT32_MAX;
        s_last = -1;
    }
    __syncthreads();
    if (s_chunk >= 0) {
        // the chunk's columns in order: kPer a thread, side by side
        const int c0 = s_chunk * kChunk + t * kPer;
        double m[kPer], own = 0.0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int c = c0 + j;
            m[j] = 0.0;
            if (c < a.vocab)
                m[j] = s_p ? weight(logit(a, a.target, ((int64_t)b * (a.k + 1) + row) * a.vocab + c), p.top, a.inv_t) *
                                 p.inv
                           : left_over(lds, a, b, row, c);
            own += m[j];
        }
        double sum = own;  // up to and with this thread, of its wave
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double x = __shfl_up(sum, d);
            if ((t & 63) >= d) sum += x;
        }
        if ((t & 63) == 63) lds.red[t >> 6] = sum;
        __syncthreads();
        double run = s_before + (sum - own);
        for (int w = 0; w < t >> 6; ++w) run += lds.red[w];
        int token = INT32_MAX, last = -1;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            run += m[j];
            if (m[j] > 0.0) {
                last = c0 + j;
                if (run > s_border) token = min(token, c0 + j);
            }
        }
        if (token != INT32_MAX) atomicMin(&s_token, token);
        if (last >= 0) atomicMax(&s_last, last);
    }
    __syncthreads();
    // rounding inside the chunk may leave the border unpassed: its last token then. No mass: token 0.
    const int token = s_token != INT32_MAX ? s_token : max(s_last, 0);
    for (int i = t; i <= a.k; i += kThreads)
        a.tokens[(int64_t)b * (a.k + 1) + i] =
            i < row ? a.drafts[(int64_t)b * a.k + i] : i == row ? token : -1;
    if (t == 0) a.accepted[b] = row;
}

struct VerifySizes {
    int64_t chunks, parts, mass;  // count, bytes, bytes
};

bool verify_sizes(VerifySizes& s, int64_t batch, int64_t k, int64_t vocab) {
    s.chunks = (vocab + kChunk - 1) / kChunk;
    s.parts = checked_mul(batch * (2 * k + 1), s.chunks, sizeof(Part));
    s.mass = checked_mul(batch, s.chunks, sizeof(double));
    return s.parts >= 0 && s.mass >= 0 && s.parts < INT64_MAX / 4 && s.mass < INT64_MAX / 4;
}

}  // namespace
}  // namespace crucible

using namespace crucible;

extern "C" size_t crucible_verify_drafts_workspace_bytes(int64_t batch, int64_t max_draft, int64_t vocab) {
    VerifySizes s;
    if (batch <= 0 || batch > 65535 || max_draft < 0 || max_draft > kMaxDrafts || vocab <= 0 ||
        vocab >= INT32_MAX - kChunk || !verify_sizes(s, batch, max_draft, vocab))
        return 0;
    return (size_t)(s.parts + s.mass);
}

extern "C" int crucible_verify_drafts(const void* target, const void* draft, int dtype, const int32_t* drafts,
                                      const int32_t* n_draft, const float* u_accept, const float* u_sample,
                                      int32_t* tokens, int32_t* accepted, int64_t batch, int64_t max_draft,
                                      int64_t vocab, double temperature, void* workspace, size_t workspace_bytes,
                                      crucible_stream_t stream) {
    const char* what = "verify_drafts";
    CRUCIBLE_CHECK(dtype_ok(dtype), CRUCIBLE_ERR_INVALID, "%s: bad dtype", what);
    CRUCIBLE_CHECK(batch >= 0 && batch <= 65535 && max_draft >= 0 && max_draft <= kMaxDrafts && vocab > 0 &&
                       vocab < INT32_MAX - kChunk,
                   CRUCIBLE_ERR_INVALID, "%s: batch=%lld drafts=%lld (at most %d) vocab=%lld", what, (long long)batch,
                   (long long)max_draft, kMaxDrafts, (long long)vocab);
    CRUCIBLE_CHECK(temperature > 0.0 && temperature <= 3.4e38 && temperature >= 1e-30, CRUCIBLE_ERR_INVALID,
                   "%s: temperature must be positive and finite", what);
    if (batch == 0) return CRUCIBLE_OK;
    CRUCIBLE_CHECK(target && n_draft && u_sample && tokens && accepted && (max_draft == 0 || (drafts && u_accept)),
                   CRUCIBLE_ERR_INVALID, "%s: null buffer", what);
    VerifySizes s;
    CRUCIBLE_CHECK(verify_sizes(s, batch, max_draft, vocab), CRUCIBLE_ERR_INVALID, "%s: too large", what);
    const size_t need = (size_t)(s.parts + s.mass);
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
    hipLaunchKernelGGL(verify_sums_kernel, dim3((unsigned)s.chunks, rows, (unsigned)batch), dim3(kThreads), 0, stream,
                       a);
    hipLaunchKernelGGL(verify_mass_kernel, dim3((unsigned)s.chunks, (unsigned)batch), dim3(kThreads), 0, stream, a);
    hipLaunchKernelGGL(verify_pick_kernel, dim3((unsigned)batch), dim3(kThreads), 0, stream, a);
    return fail_launch(what);
}
