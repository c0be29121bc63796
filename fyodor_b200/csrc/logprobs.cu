// logprobs.cu - log probability and rank of a given token, entropy and the most
// probable alternatives of rows of logits, in one pass over them.
//
//   m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m)
//   ln p(t) = x_t - m - ln S        H = ln S - T / S
//
// Bound by HBM: each logit is read once. The rows lie on a line of chunks (a
// chunk: 64 bytes for each of 256 threads) that is shared out evenly over the
// CTAs, whatever rows and vocabulary are; a row that crosses CTAs leaves a partial
// for each, which the last CTA to finish joins in order (no CTA waits for
// another, results do not depend on timing).
//
// A thread sums against a reference of its own that moves only when a logit is more
// than 8 above it, so sums are not rescaled at every new maximum (their terms are
// at most e^8); pairs of terms go through the packed F32 instructions. A warp
// keeps the best 32 logits sorted over its lanes; a logit is looked at only if it
// is above the last of them that counts, so alternatives cost a comparison for
// 16 logits but for some K ln(n) insertions. The first batch of a row bounds the
// list from below by the K-th largest of the lanes' maxima.
#include "common.cuh"
#include "kernels.h"
#include "fyodor_b200.h"
#include <climits>

namespace fyb {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_LOADS = 4, LP_GRID = 4 * 148;
constexpr float LP_LOWEST = -3.402823466e38f, LP_FAR = -1e4f;  // e^LP_FAR is 0

struct LpSums {
    float top, m, s, t;  // largest logit; reference, S and T relative to it
};
struct LpBest {
    float v;
    int i;
};
struct Logprobs {
    const void *x;
    size_t stride, rows;
    unsigned n, top, chunks;  // chunks of a row
    const int *tokens;
    float *logprob, *entropy, *top_logprobs;
    int *rank, *top_tokens;
    unsigned *counters;   // [grid] arrivals at the row that begins in CTA c and ends beyond it; zero between calls
    LpSums *part;         // [2 grid]
    unsigned *part_rank;  // [2 grid]
    LpBest *part_best;    // [2 grid][32]
    unsigned *error;
};
constexpr size_t LP_COUNTER_BYTES = (LP_GRID * 4 + 255) / 256 * 256;
constexpr size_t LP_PART_BYTES = 2 * LP_GRID * (sizeof(LpSums) + 4);

FYB_DEV float lp_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float LP_LOG2E = 1.44269504f;

// Sums relative to m taken to the reference M >= m (or to any M where s is 0).
FYB_DEV void lp_move(float &m, float &s, float &t, float M)
{
    const float d = fmaxf(m - M, LP_FAR), f = lp_exp2(d * LP_LOG2E);
    t = fmaf(s, d, t) * f;
    s *= f;
    m = M;
}
FYB_DEV LpSums lp_join(LpSums a, const LpSums &b)
{
    // the new reference is the larger of the two largest logits, at least the lowest number
    LpSums c = b;
    const float top = fmaxf(a.top, b.top), M = fmaxf(top, LP_LOWEST);
    lp_move(a.m, a.s, a.t, M);
    lp_move(c.m, c.s, c.t, M);
    return LpSums{top, M, a.s + c.s, a.t + c.t};
}
FYB_DEV LpSums lp_shuffle(const LpSums &a, int o)
{
    return LpSums{__shfl_xor_sync(0xffffffffu, a.top, o), __shfl_xor_sync(0xffffffffu, a.m, o),
                  __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o)};
}

// ---- the best, sorted over a warp's lanes -----------------------------------------
FYB_DEV bool lp_before(const LpBest &a, const LpBest &b) { return a.v > b.v || (a.v == b.v && (unsigned)a.i < (unsigned)b.i); }
FYB_DEV LpBest lp_none() { return LpBest{-INFINITY, -1}; }
// One more (the same on all lanes).
FYB_DEV void lp_insert(LpBest &mine, const LpBest &x, unsigned lane)
{
    const unsigned at = __popc(__ballot_sync(0xffffffffu, lp_before(mine, x)));
    const float v = __shfl_up_sync(0xffffffffu, mine.v, 1);
    const int i = __shfl_up_sync(0xffffffffu, mine.i, 1);
    if (lane == at) mine = x;
    else if (lane > at) mine = LpBest{v, i};
}
// The best 32 of two sorted lists.
FYB_DEV LpBest lp_merge(const LpBest &a, const LpBest &b, unsigned lane)
{
    const LpBest r{__shfl_sync(0xffffffffu, b.v, 31 - lane), __shfl_sync(0xffffffffu, b.i, 31 - lane)};
    LpBest x = lp_before(a, r) ? a : r;  // the best 32, rising and falling once
#pragma unroll
    for (unsigned o = 16; o; o >>= 1) {
        const LpBest y{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)};
        if (lp_before(y, x) == !(lane & o)) x = y;
    }
    return x;
}
// The k-th largest (from 0) of the lanes' values.
FYB_DEV float lp_kth(float v, unsigned k, unsigned lane)
{
#pragma unroll
    for (unsigned size = 2; size <= 32; size *= 2)
#pragma unroll
        for (unsigned o = size / 2; o; o >>= 1) {
            const float y = __shfl_xor_sync(0xffffffffu, v, o);
            v = ((lane & o) == 0) == ((lane & size) == 0) ? fmaxf(v, y) : fminf(v, y);
        }
    return __shfl_sync(0xffffffffu, v, (int)k);
}

template <typename T> struct LpVec;  // the values of a 16-byte access
template <> struct LpVec<float> {
    static constexpr int V = 4;
    static FYB_DEV void get(const uint4 &u, float *x)
    {
        x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
    }
};
template <> struct LpVec<__half> {
    static constexpr int V = 8;
    static FYB_DEV void get(const uint4 &u, float *x)
    {
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
};
template <> struct LpVec<__nv_bfloat16> {
    static constexpr int V = 8;
    static FYB_DEV void get(const uint4 &u, float *x)
    {
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

// What a thread (and its warp) carries along a row.
template <bool TOP> struct LpState {
    float top, m;
    F2 s, t;
    unsigned before;
    LpBest best;  // lane's place of the warp's list
    float last;   // the top-th of it
    bool first;
    FYB_DEV void begin()
    {
        top = -INFINITY;
        m = LP_LOWEST;
        s = t = f2(0.f, 0.f);
        before = 0;
        best = lp_none();
        last = -INFINITY;
        first = true;
    }
    // N logits, the j-th of index(j); all lanes of the warp call it, with -inf of index INT_MAX for what they do not have
    template <int N, typename Index>
    FYB_DEV void take(const float (&x)[N], float given, int token, int lo, int hi, unsigned k, volatile unsigned *bound, unsigned lane, Index index)
    {
        float high = x[0];
#pragma unroll
        for (int j = 1; j < N; ++j) high = fmaxf(high, x[j]);
        top = fmaxf(top, high);
        if (high - m > 8.f) {
            float2 a = f2_get(s), b = f2_get(t);
            float sum = a.x + a.y, weighted = b.x + b.y;
            lp_move(m, sum, weighted, high);
            s = f2(sum, 0.f);
            t = f2(weighted, 0.f);
        }
        const F2 minus = f2(-m, -m), unit = f2(LP_LOG2E, LP_LOG2E);
        static_assert(N == 1 || N % 2 == 0, "");
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const F2 d = f2_add(f2(x[j], N > 1 ? x[j + 1 < N ? j + 1 : j] : -INFINITY), minus);
            const float2 q = f2_get(f2_mul(d, unit)), dd = f2_get(d);
            const F2 e = f2(lp_exp2(q.x), lp_exp2(q.y));
            s = f2_add(s, e);  // NaN stays here
            t = f2_fma(e, f2(fmaxf(dd.x, LP_FAR), fmaxf(dd.y, LP_FAR)), t);
        }
        // logits from index lo to hi: before the token equal ones count too
        if (hi < token && given > -INFINITY) {
#pragma unroll
            for (int j = 0; j < N; ++j) before += x[j] >= given;
        } else if (lo > token) {
#pragma unroll
            for (int j = 0; j < N; ++j) before += x[j] > given;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) before += x[j] > given || (x[j] == given && index(j) < token);
        }
        if constexpr (TOP) {
            // A warp's batches ascend: of equal logits those in the list come first, so the next has to be above its last.
            // Another warp's last is a bound too; logits that equal it may come first.
            const float other = float_from_order_key(*bound);
            if (!__any_sync(0xffffffffu, high > last && high >= other)) return;
            float least = other;
            if (N > 1 && first) {
                least = fmaxf(least, lp_kth(high, k - 1, lane));
                first = false;
            }
            const float was = last;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                unsigned left = __ballot_sync(0xffffffffu, x[j] > was && x[j] >= least);
                while (left) {
                    const int from = __ffs((int)left) - 1;
                    left &= left - 1;
                    lp_insert(best, LpBest{__shfl_sync(0xffffffffu, x[j], from), __shfl_sync(0xffffffffu, index(j), from)}, lane);
                    least = fmaxf(least, __shfl_sync(0xffffffffu, best.v, (int)k - 1));
                    left &= __ballot_sync(0xffffffffu, x[j] >= least);
                }
            }
            last = __shfl_sync(0xffffffffu, best.v, (int)k - 1);
            if (lane == 0 && last > other) atomicMax(const_cast<unsigned *>(bound), float_order_key(last));
        }
    }
};

FYB_DEV unsigned lp_begin(unsigned long long U, unsigned C, unsigned c) { return (unsigned)(U * c / C); }
FYB_DEV unsigned lp_cta_of(unsigned long long U, unsigned C, unsigned u) { return (unsigned)(((u + 1ull) * C - 1) / U); }

// Lists of all warps into warp 0's; every thread of the CTA, behind a barrier.
FYB_DEV void lp_merge_warps(LpBest (&best)[LP_WARPS][32])
{
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (unsigned o = LP_WARPS / 2; o; o >>= 1) {
        if (warp < o) best[warp][lane] = lp_merge(best[warp][lane], best[warp + o][lane], lane);
        __syncthreads();
    }
}

template <typename T, bool TOP> __global__ void __launch_bounds__(LP_THREADS, 4) logprobs_kernel(const __grid_constant__ Logprobs A)
{
    constexpr int V = LpVec<T>::V, CHUNK = LP_LOADS * LP_THREADS;  // 16-byte accesses of a chunk
    constexpr int N = 16, PER = N / V;                              // logits that are taken at once, accesses of them
    __shared__ LpSums sums_s[LP_WARPS];
    __shared__ unsigned rank_s[LP_WARPS], bound_s, flag_s;
    __shared__ LpBest best_s[LP_WARPS][32];
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, C = gridDim.x;
    const unsigned long long U = (unsigned long long)A.rows * A.chunks;
    unsigned at = lp_begin(U, C, blockIdx.x);
    const unsigned end = lp_begin(U, C, blockIdx.x + 1);
    LpState<TOP> st;
    while (at < end) {
        const unsigned row = at / A.chunks, c0 = at % A.chunks, c1 = min(A.chunks, c0 + (end - at));
        const T *x = static_cast<const T *>(A.x) + row * A.stride;
        // elements before the first 16-byte boundary, whole accesses, elements behind them
        const unsigned head = min(A.n, (unsigned)((16 - ((uintptr_t)x & 15)) & 15) / (unsigned)sizeof(T));
        const unsigned vectors = (A.n - head) / V, tail = head + vectors * V;
        const uint4 *body = reinterpret_cast<const uint4 *>(x + head);
        int token = A.tokens ? A.tokens[row] : -1;
        if (token >= (int)A.n) {
            if (tid == 0 && c0 == 0) raise_error(A.error, ERR_BOUNDS);
            token = -1;
        }
        const float given = token >= 0 ? row_value(x[token]) : INFINITY;
        if (TOP) {
            __syncthreads();
            if (tid == 0) bound_s = float_order_key(-INFINITY);
            __syncthreads();
        }
        st.begin();
        auto edge = [&](unsigned from, unsigned to) {  // fewer than V elements, warp 0
            const unsigned i = from + lane;
            const float y[1] = {i < to ? row_value(x[i]) : -INFINITY};
            st.take(y, given, token, 0, (int)A.n, A.top, &bound_s, lane, [&](int) { return i < to ? (int)i : INT_MAX; });
        };
        if (c0 == 0 && warp == 0 && head) edge(0, head);
        for (unsigned c = c0; c < c1; ++c) {
            const unsigned v0 = c * CHUNK + warp * LP_LOADS * 32 + lane;
            uint4 raw[LP_LOADS];
#pragma unroll
            for (int u = 0; u < LP_LOADS; ++u)
                if (v0 + u * 32 < vectors) raw[u] = ldg_stream_u4(body + v0 + u * 32);
            if (v0 - lane >= vectors) break;  // the warp has none
#pragma unroll
            for (int u = 0; u < LP_LOADS; u += PER) {
                float y[N];
#pragma unroll
                for (int w = 0; w < PER; ++w) {
                    LpVec<T>::get(raw[u + w], y + w * V);
                    if (v0 + (u + w) * 32 >= vectors) {
#pragma unroll
                        for (int j = 0; j < V; ++j) y[w * V + j] = -INFINITY;
                    }
                }
                const unsigned first = head + (v0 + u * 32) * V;
                st.take(y, given, token, (int)first, (int)(first + ((PER - 1) * 32 + 1) * V - 1), A.top, &bound_s, lane,
                        [&](int j) { return v0 + (u + j / V) * 32 < vectors ? (int)(first + (j / V) * 32 * V + j % V) : INT_MAX; });
            }
        }
        if (c1 == A.chunks && warp == 0 && tail < A.n) edge(tail, A.n);

        // ---- the CTA's part of the row
        const float2 s2 = f2_get(st.s), t2 = f2_get(st.t);
        LpSums sums{st.top, st.m, s2.x + s2.y, t2.x + t2.y};
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            sums = lp_join(sums, lp_shuffle(sums, o));
            st.before += __shfl_xor_sync(0xffffffffu, st.before, o);
        }
        if (lane == 0) { sums_s[warp] = sums; rank_s[warp] = st.before; }
        if (TOP) best_s[warp][lane] = st.best;
        __syncthreads();
        if (TOP) lp_merge_warps(best_s);
        unsigned before = 0;
        if (warp == 0) {
            sums = lane < LP_WARPS ? sums_s[lane] : LpSums{-INFINITY, LP_LOWEST, 0.f, 0.f};
            before = lane < LP_WARPS ? rank_s[lane] : 0;
#pragma unroll
            for (int o = 16; o; o >>= 1) {  // every lane writes an alternative: all need them
                sums = lp_join(sums, lp_shuffle(sums, o));
                before += __shfl_xor_sync(0xffffffffu, before, o);
            }
        }
        bool write = true;
        if (c0 || c1 < A.chunks) {
            // ---- a part: the last CTA of the row joins them all in order
            const unsigned first = row * A.chunks, f = lp_cta_of(U, C, first), l = lp_cta_of(U, C, first + A.chunks - 1);
            const unsigned slot = 2 * blockIdx.x + (blockIdx.x == f ? 1 : 0);
            if (warp == 0) {
                if (lane == 0) { A.part[slot] = sums; A.part_rank[slot] = before; }
                if (TOP) A.part_best[slot * 32 + lane] = best_s[0][lane];
                __threadfence();
                __syncwarp();
                if (lane == 0) flag_s = atomicAdd(&A.counters[f], 1u) == l - f;
            }
            __syncthreads();
            write = flag_s;
            if (write) {
                __threadfence();
                if (tid == 0) A.counters[f] = 0;
                auto slot_of = [&](unsigned p) { return 2 * (f + p) + (p == 0 ? 1 : 0); };
                const unsigned parts = l - f + 1;
                if (warp == 0) {
                    sums = LpSums{-INFINITY, LP_LOWEST, 0.f, 0.f};
                    before = 0;
                    for (unsigned p = lane; p < parts; p += 32) {
                        const float4 y = __ldcg(reinterpret_cast<const float4 *>(A.part) + slot_of(p));
                        sums = lp_join(sums, LpSums{y.x, y.y, y.z, y.w});
                        before += __ldcg(A.part_rank + slot_of(p));
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) {
                        sums = lp_join(sums, lp_shuffle(sums, o));
                        before += __shfl_xor_sync(0xffffffffu, before, o);
                    }
                }
                if (TOP) {
                    LpBest mine = lp_none();
                    for (unsigned p = warp; p < parts; p += LP_WARPS) {
                        const float2 y = __ldcg(reinterpret_cast<const float2 *>(A.part_best) + slot_of(p) * 32 + lane);
                        mine = lp_merge(mine, LpBest{y.x, __float_as_int(y.y)}, lane);
                    }
                    best_s[warp][lane] = mine;
                    __syncthreads();
                    lp_merge_warps(best_s);
                }
            }
        }
        if (write && warp == 0) {
            const bool bad = isnan(sums.s), none = sums.top == -INFINITY && !bad;
            const float log_sum = logf(sums.s);
            if (lane == 0) {
                if (bad) raise_error(A.error, ERR_NONFINITE);
                if (A.logprob) A.logprob[row] = token < 0 ? 0.f : bad ? NAN : none ? -INFINITY : given - sums.m - log_sum;
                if (A.rank) A.rank[row] = token < 0 ? -1 : (int)before;
                if (A.entropy) A.entropy[row] = bad ? NAN : none ? 0.f : log_sum - sums.t / sums.s;
            }
            if (TOP && lane < A.top) {
                const LpBest b = best_s[0][lane];
                A.top_tokens[(size_t)row * A.top + lane] = b.i;
                A.top_logprobs[(size_t)row * A.top + lane] = bad ? NAN : b.i < 0 ? -INFINITY : b.v - sums.m - log_sum;
            }
        }
        __syncthreads();
        at += c1 - c0;
    }
}

template <typename T> static int logprobs_launch(const Logprobs &A, unsigned grid, cudaStream_t s)
{
    if (A.top) logprobs_kernel<T, true><<<grid, LP_THREADS, 0, s>>>(A);
    else logprobs_kernel<T, false><<<grid, LP_THREADS, 0, s>>>(A);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace fyb

using namespace fyb;

extern "C" size_t fyb_logprobs_workspace(size_t rows, uint32_t vocabulary, uint32_t top)
{
    if (rows > 0x7fffffffu || !vocabulary || vocabulary > 0x7fffffffu || top > FYB_LOGPROBS_TOP) return 0;
    return LP_COUNTER_BYTES + LP_PART_BYTES + (top ? 2 * LP_GRID * 32 * sizeof(LpBest) : 0);
}

extern "C" int fyb_logprobs(uint32_t type, const void *logits, size_t stride, size_t rows, uint32_t vocabulary,
    const int32_t *tokens, float *logprob, int32_t *rank, float *entropy, uint32_t top, int32_t *top_tokens,
    float *top_logprobs, void *workspace, size_t workspace_bytes, uint32_t *error, void *stream)
{
    const size_t need = fyb_logprobs_workspace(rows, vocabulary, top);
    const size_t width = type == T_F32 ? 4 : 2;
    if ((type != T_F32 && type != T_F16 && type != T_BF16) || !need || stride < vocabulary || !workspace ||
        (uintptr_t)workspace % 16 || workspace_bytes < need || (uintptr_t)logits % width)
        return -1;
    if (rows && (!logits || !tokens != !logprob || (rank && !tokens) || (top && (!top_tokens || !top_logprobs)))) return -1;
    if (!rows) return 0;
    Logprobs A{};
    A.x = logits; A.stride = stride; A.rows = rows; A.n = vocabulary; A.top = top;
    A.tokens = tokens; A.logprob = logprob; A.entropy = entropy; A.rank = rank;
    A.top_tokens = top_tokens; A.top_logprobs = top_logprobs; A.error = error;
    const size_t chunk = (size_t)LP_LOADS * LP_THREADS * (16 / width);
    A.chunks = (unsigned)((vocabulary + chunk - 1) / chunk);
    const unsigned long long units = (unsigned long long)rows * A.chunks;
    if (units > 0xffffffffull - LP_GRID) return -1;
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    A.counters = reinterpret_cast<unsigned *>(ws);
    A.part = reinterpret_cast<LpSums *>(ws + LP_COUNTER_BYTES);
    A.part_rank = reinterpret_cast<unsigned *>(A.part + 2 * LP_GRID);
    A.part_best = reinterpret_cast<LpBest *>(ws + LP_COUNTER_BYTES + LP_PART_BYTES);
    const unsigned grid = (unsigned)std::min<unsigned long long>(LP_GRID, units);
    cudaStream_t s = (cudaStream_t)stream;
    if (type == T_F32) return logprobs_launch<float>(A, grid, s);
    if (type == T_F16) return logprobs_launch<__half>(A, grid, s);
    return logprobs_launch<__nv_bfloat16>(A, grid, s);
}
