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
// at most e^8); pairs of terms go through the packed F32 instructions.
//
// Alternatives: a warp keeps the best 32 logits sorted over its lanes, and looks at
// one only if it is above the last of them that counts and not below a bound that
// the CTA's warps share. The bound: of the largest logits that the 256 threads have
// seen, taken together by lane, the K-th of 32 largest has K logits at or above it.
// It is found before the first chunk is looked at and again as chunks pass, so some
// 30 logits of a chunk, then of each doubling of them, are looked at by all warps
// together (with the lists' own last ones alone each warp looked at K ln(n) of its
// own: a prompt of 400 rows with 20 alternatives 83 us, so 67).
#include "common.cuh"
#include "kernels.h"
#include "fyodor_b200.h"
#include <climits>

namespace fyb {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_LOADS = 4, LP_CTAS = 3, LP_GRID = LP_CTAS * 148;
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

// The values of a 16-byte access, -inf taken as the type's lowest number (its exponential is 0 all the same, and the
// product with it too, where -inf would leave NaN): `far` says whether that holds against a reference m. Largest and
// count of those above (or at) a value, NaN being neither.
template <typename T> struct LpVec;
template <> struct LpVec<float> {
    static constexpr int V = 4;
    static FYB_DEV uint4 none() { const unsigned x = 0xff800000u; return make_uint4(x, x, x, x); }
    static FYB_DEV void get(const uint4 &u, float *x)
    {
        x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
    }
    static FYB_DEV void finite(const uint4 &u, float *x)
    {
        get(u, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("max.NaN.f32 %0, %1, %2;" : "=f"(x[i]) : "f"(x[i]), "f"(LP_LOWEST));
    }
    static FYB_DEV bool far(float m) { return m > -1e30f && m < 1e30f; }
    template <int N> static FYB_DEV float largest(const uint4 (&u)[N])
    {
        float h = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float x[4];
            get(u[i], x);
            h = fmaxf(fmaxf(h, fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
        }
        return h;
    }
    template <bool EQUAL, int N> static FYB_DEV unsigned above(const uint4 (&u)[N], float than)
    {
        unsigned c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float x[4];
            get(u[i], x);
#pragma unroll
            for (int j = 0; j < 4; ++j) c += EQUAL ? x[j] >= than : x[j] > than;
        }
        return c;
    }
};
template <typename H2> struct LpPairs {  // two values a word
    static constexpr int V = 8;
    static FYB_DEV H2 pair(unsigned w) { return *reinterpret_cast<const H2 *>(&w); }
    static FYB_DEV unsigned word(H2 p) { return *reinterpret_cast<const unsigned *>(&p); }
};
template <> struct LpVec<__half> : LpPairs<__half2> {
    static FYB_DEV uint4 none() { const unsigned x = 0xfc00fc00u; return make_uint4(x, x, x, x); }
    static FYB_DEV float2 two(unsigned w) { return __half22float2(pair(w)); }
    static FYB_DEV unsigned finite(unsigned w) { return word(__hmax2_nan(pair(w), pair(0xfbfffbffu))); }
    static FYB_DEV bool far(float m) { return m > -65000.f; }
    static FYB_DEV __half2 one(float x) { return __float2half2_rn(x); }
};
template <> struct LpVec<__nv_bfloat16> : LpPairs<__nv_bfloat162> {
    static FYB_DEV uint4 none() { const unsigned x = 0xff80ff80u; return make_uint4(x, x, x, x); }
    static FYB_DEV float2 two(unsigned w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static FYB_DEV unsigned finite(unsigned w) { return word(__hmax2_nan(pair(w), pair(0xff7fff7fu))); }
    static FYB_DEV bool far(float m) { return m > -1e30f && m < 1e30f; }
    static FYB_DEV __nv_bfloat162 one(float x) { return __float2bfloat162_rn(x); }
};
template <typename T> struct LpRow : LpVec<T> {  // what both 16-bit types do alike
    using B = LpVec<T>;
    static FYB_DEV void get(const uint4 &u, float *x)
    {
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = B::two(w[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
    }
    static FYB_DEV void finite(const uint4 &u, float *x)
    {
        get(make_uint4(B::finite(u.x), B::finite(u.y), B::finite(u.z), B::finite(u.w)), x);
    }
    template <int N> static FYB_DEV float largest(const uint4 (&u)[N])
    {
        auto h = B::pair(B::none().x);
#pragma unroll
        for (int i = 0; i < N; ++i)
            h = __hmax2(h, __hmax2(__hmax2(B::pair(u[i].x), B::pair(u[i].y)), __hmax2(B::pair(u[i].z), B::pair(u[i].w))));
        const float2 f = B::two(B::word(h));
        return fmaxf(f.x, f.y);
    }
    template <bool EQUAL, int N> static FYB_DEV unsigned above(const uint4 (&u)[N], float than)
    {
        const auto t = B::one(than);  // of this type, so exactly itself
        auto c = B::one(0.f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) c = __hadd2(c, EQUAL ? __hge2(B::pair(w[j]), t) : __hgt2(B::pair(w[j]), t));  // 1 or 0 each
        }
        const float2 f = B::two(B::word(c));
        return (unsigned)(f.x + f.y);
    }
};
template <> struct LpRow<float> : LpVec<float> {};

// What a thread (and its warp) carries along a row.
template <typename T, bool TOP> struct LpState {
    using Row = LpRow<T>;
    float top, m;
    F2 s, t;
    unsigned before;
    LpBest best;  // lane's place of the warp's list
    float last;   // the top-th of it
    FYB_DEV void begin()
    {
        top = -INFINITY;
        m = LP_LOWEST;
        s = t = f2(0.f, 0.f);
        before = 0;
        best = lp_none();
        last = -INFINITY;
    }
    FYB_DEV void reach(float high)
    {
        top = fmaxf(top, high);
        if (high - m > 8.f) {
            float2 a = f2_get(s), b = f2_get(t);
            float sum = a.x + a.y, weighted = b.x + b.y;
            lp_move(m, sum, weighted, high);
            s = f2(sum, 0.f);
            t = f2(weighted, 0.f);
        }
    }
    template <bool FAR> FYB_DEV void add(float x, float y)
    {
        const F2 d = f2_add(f2(x, y), f2(-m, -m));
        const float2 q = f2_get(f2_mul(d, f2(LP_LOG2E, LP_LOG2E))), dd = f2_get(d);
        const F2 e = f2(lp_exp2(q.x), lp_exp2(q.y));
        s = f2_add(s, e);  // NaN stays here
        t = f2_fma(e, FAR ? d : f2(fmaxf(dd.x, LP_FAR), fmaxf(dd.y, LP_FAR)), t);
    }
    // Candidates for the list: N logits of a lane, of which high is the largest; index(l, j) is that of lane l's j-th. A
    // warp's batches ascend: of equal logits those in the list come first, so the next has to be above its last; logits
    // that equal the bound may come first. stage: [32][20] of the warp.
    template <int N, typename Get, typename Index>
    FYB_DEV void choose(float high, unsigned k, volatile unsigned *bound, float *stage, unsigned lane, Get get, Index index)
    {
        float least = float_from_order_key(*bound);
        if (!__any_sync(0xffffffffu, high > last && high >= least)) return;
        float x[N];
        get(x);
        unsigned mask = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) mask |= (x[j] > last && x[j] >= least ? 1u : 0u) << j;
        __syncwarp();
        if constexpr (N == 1) {
            stage[lane * 20] = x[0];
        } else {
#pragma unroll
            for (int j = 0; j < N; j += 4) *reinterpret_cast<float4 *>(stage + lane * 20 + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        }
        __syncwarp();
#pragma unroll 1
        for (unsigned left; (left = __ballot_sync(0xffffffffu, mask != 0)) != 0;) {
            const int from = __ffs((int)left) - 1, j = __ffs((int)__shfl_sync(0xffffffffu, mask, from)) - 1;
            if ((int)lane == from) mask &= mask - 1;
            const float v = stage[from * 20 + j];
            if (v < least) continue;
            lp_insert(best, LpBest{v, index(from, j)}, lane);
            least = fmaxf(least, __shfl_sync(0xffffffffu, best.v, (int)k - 1));
        }
        last = __shfl_sync(0xffffffffu, best.v, (int)k - 1);
    }
    // PER accesses, index(l, j) that of lane l's j-th logit (INT_MAX for what is not the row's, which is -inf), from lo to hi; all
    // lanes of the warp call it
    template <int PER, typename Index>
    FYB_DEV void take(const uint4 (&u)[PER], float given, int token, int lo, int hi, unsigned k, volatile unsigned *bound, float *stage, unsigned lane, Index index)
    {
        constexpr int N = PER * Row::V;
        const float high = Row::largest(u);
        reach(high);
        if (__builtin_expect(Row::far(m), 1)) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                float x[Row::V];
                Row::finite(u[i], x);
#pragma unroll
                for (int j = 0; j < Row::V; j += 2) add<true>(x[j], x[j + 1]);
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < PER; ++i) {
                uint4 w = u[0];
#pragma unroll
                for (int j = 1; j < PER; ++j) if (i == j) w = u[j];
                float x[Row::V];
                Row::get(w, x);
#pragma unroll
                for (int j = 0; j < Row::V; j += 2) add<false>(x[j], x[j + 1]);
            }
        }
        // rank: before the token equal ones count too
        if (__any_sync(0xffffffffu, high >= given)) {
            if (lo > token) {
                before += Row::template above<false>(u, given);
            } else if (hi < token && given > -INFINITY) {
                before += Row::template above<true>(u, given);
            } else {
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    float x[Row::V];
                    Row::get(u[i], x);
#pragma unroll
                    for (int j = 0; j < Row::V; ++j) before += x[j] > given || (x[j] == given && index((int)lane, i * Row::V + j) < token);
                }
            }
        }
        if constexpr (TOP)
            choose<N>(high, k, bound, stage, lane, [&](float (&x)[N]) {
#pragma unroll
                for (int i = 0; i < PER; ++i) Row::get(u[i], x + i * Row::V);
            }, index);
    }
    // One logit a lane, the l-th of index i0 + l; -inf of index INT_MAX for none.
    FYB_DEV void take(float x, int i, float given, int token, unsigned k, volatile unsigned *bound, float *stage, unsigned lane, int i0)
    {
        reach(x);
        add<false>(x, -INFINITY);
        before += x > given || (x == given && i < token);
        if constexpr (TOP) choose<1>(x, k, bound, stage, lane, [&](float (&y)[1]) { y[0] = x; }, [&](int l, int) { return i0 + l; });
    }
};

FYB_DEV unsigned lp_begin(unsigned long long U, unsigned C, unsigned c) { return (unsigned)(U * c / C); }
FYB_DEV unsigned lp_cta_of(unsigned long long U, unsigned C, unsigned u) { return (unsigned)(((u + 1ull) * C - 1) / U); }

// The best k of up to 32 sorted lists (lane l's: lists[l * stride ..], k entries) by one warp, the best of the lists' heads
// at a time. Up to LP_FEW of them this is quicker than merging sorted lists in pairs (16 rows with 5 alternatives 11.4
// us, merged 13.4; 400 rows with 9, merged, 58.3, with 8 so 54.3).
constexpr unsigned LP_FEW = 8;
FYB_DEV LpBest lp_heads(const LpBest *lists, unsigned count, unsigned stride, unsigned k, unsigned lane)
{
    const LpBest *mine = lists + lane * stride, *end = mine + k;
    LpBest head = lane < count ? *mine : lp_none(), out = lp_none();
    for (unsigned j = 0; j < k; ++j) {
        const unsigned key = float_order_key(head.v + 0.f), top = __reduce_max_sync(0xffffffffu, key);  // -0 counts as 0
        const unsigned first = __reduce_min_sync(0xffffffffu, key == top ? (unsigned)head.i : 0xffffffffu);
        const bool won = key == top && (unsigned)head.i == first;
        const float v = __shfl_sync(0xffffffffu, head.v, __ffs((int)__ballot_sync(0xffffffffu, won)) - 1);
        if (lane == j) out = LpBest{v, (int)first};
        if (won && lane < count) head = ++mine < end ? *mine : lp_none();
    }
    return out;
}
// Lists of all warps into warp 0's; every thread of the CTA, behind a barrier.
FYB_DEV void lp_merge_warps(LpBest (&best)[LP_WARPS][32])
{
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (unsigned o = LP_WARPS / 2; o; o >>= 1) {
        if (warp < o) best[warp][lane] = lp_merge(best[warp][lane], best[warp + o][lane], lane);
        __syncthreads();
    }
}

template <typename T, bool TOP> __global__ void __launch_bounds__(LP_THREADS, LP_CTAS) logprobs_kernel(const __grid_constant__ Logprobs A)
{
    using Row = LpRow<T>;
    constexpr int V = Row::V, CHUNK = LP_LOADS * LP_THREADS;  // 16-byte accesses of a chunk
    constexpr int PER = 16 / V;                                // accesses that are taken at once
    // what the warps hold of a row, of two rows in turn: one warp joins them while the others go on
    __shared__ LpSums sums_s[2][LP_WARPS];
    __shared__ unsigned rank_s[2][LP_WARPS], bound_s[2], flag_s;
    __shared__ LpBest best_s[2][LP_WARPS][32];
    __shared__ float seen_s[TOP ? LP_WARPS : 1][32];                 // largest logit that each thread has seen of the row
    __shared__ __align__(16) float stage_s[TOP ? LP_WARPS : 1][32 * 20];
    static_assert(sizeof(LpBest) * 32 * LP_FEW <= sizeof(float) * 32 * 20, "a warp's place holds the lists of 32 parts");
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, C = gridDim.x;
    const unsigned long long U = (unsigned long long)A.rows * A.chunks;
    unsigned at = lp_begin(U, C, blockIdx.x);
    const unsigned end = lp_begin(U, C, blockIdx.x + 1);
    LpState<T, TOP> st;
    unsigned turn = 0;
    if (tid == 0) bound_s[0] = float_order_key(-INFINITY);
    __syncthreads();
    for (; at < end; ++turn) {
        const unsigned use = turn & 1;
        const unsigned row = at / A.chunks, c0 = at % A.chunks, c1 = min(A.chunks, c0 + (end - at));
        const T *x = static_cast<const T *>(A.x) + row * A.stride;
        // elements before the first 16-byte boundary, whole accesses, elements behind them
        const unsigned head = min(A.n, (unsigned)((16 - ((uintptr_t)x & 15)) & 15) / (unsigned)sizeof(T));
        const unsigned vectors = (A.n - head) / V, tail = head + vectors * V;
        const uint4 *body = reinterpret_cast<const uint4 *>(x + head);
        // a chunk is asked for while the one before is taken, the first before all else
        uint4 raw[LP_LOADS];
        unsigned v0 = c0 * CHUNK + warp * LP_LOADS * 32 + lane;
        auto ask = [&] {
#pragma unroll
            for (int u = 0; u < LP_LOADS; ++u) {
                raw[u] = Row::none();
                if (v0 + u * 32 < vectors) raw[u] = ldg_stream_u4(body + v0 + u * 32);
            }
        };
        ask();
        const bool begins = c0 == 0 && warp == 0 && head, ends = c1 == A.chunks && warp == 0 && tail < A.n;
        const float early = begins && lane < head ? row_value(x[lane]) : -INFINITY;
        const float late = ends && tail + lane < A.n ? row_value(x[tail + lane]) : -INFINITY;
        int token = A.tokens ? A.tokens[row] : -1;
        if (token >= (int)A.n) {
            if (tid == 0 && c0 == 0) raise_error(A.error, ERR_BOUNDS);
            token = -1;
        }
        const float given = token >= 0 ? row_value(x[token]) : INFINITY;
        st.begin();
        float *stage = stage_s[TOP ? warp : 0];
        // the K-th largest of the lanes' largest logits, all warps': K logits of the row are at or above it
        auto bound = [&] {
            float h = seen_s[0][lane];
#pragma unroll
            for (int w = 1; w < (TOP ? LP_WARPS : 1); ++w) h = fmaxf(h, *(volatile float *)&seen_s[w][lane]);
            h = lp_kth(h, A.top - 1, lane);
            if (lane == 0) atomicMax(&bound_s[use], float_order_key(h));
        };
        if constexpr (TOP) {
            seen_s[warp][lane] = Row::largest(raw);
            __syncthreads();
            if (warp == 0) bound();
            __syncthreads();
        }
        if (begins) st.take(early, lane < head ? (int)lane : INT_MAX, given, token, A.top, &bound_s[use], stage, lane, 0);
#pragma unroll 1
        for (unsigned c = c0; c < c1 && v0 - lane < vectors; ++c) {
            uint4 now[LP_LOADS];
#pragma unroll
            for (int u = 0; u < LP_LOADS; ++u) now[u] = raw[u];
            const unsigned v = v0;
            v0 += CHUNK;
            if (c + 1 < c1) ask();
#pragma unroll
            for (int u = 0; u < LP_LOADS; u += PER) {
                uint4 part[PER];
#pragma unroll
                for (int w = 0; w < PER; ++w) part[w] = now[u + w];
                const unsigned first = head + (v + u * 32) * V;
                st.take(part, given, token, (int)first, (int)(first + ((PER - 1) * 32 + 1) * V - 1), A.top, &bound_s[use], stage, lane,
                        [&](int l, int j) {
                            const unsigned at = v - lane + (unsigned)l + (u + j / V) * 32;
                            return at < vectors ? (int)(head + at * V + j % V) : INT_MAX;
                        });
            }
            if constexpr (TOP) {
                const unsigned i = c - c0;
                if (i) {
                    seen_s[warp][lane] = st.top;
                    __syncwarp();
                    if (((i & (i - 1)) == 0 || i % 4 == 0) && warp == i % LP_WARPS) bound();
                }
            }
        }
        if (ends) st.take(late, tail + lane < A.n ? (int)(tail + lane) : INT_MAX, given, token, A.top, &bound_s[use], stage, lane, (int)tail);

        // ---- the CTA's part of the row
        const float2 s2 = f2_get(st.s), t2 = f2_get(st.t);
        LpSums sums{st.top, st.m, s2.x + s2.y, t2.x + t2.y};
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            sums = lp_join(sums, lp_shuffle(sums, o));
            st.before += __shfl_xor_sync(0xffffffffu, st.before, o);
        }
        if (lane == 0) { sums_s[use][warp] = sums; rank_s[use][warp] = st.before; }
        if (TOP) best_s[use][warp][lane] = st.best;
        if (tid == 0) bound_s[use ^ 1] = float_order_key(-INFINITY);
        __syncthreads();
        at += c1 - c0;
        const bool last = at >= end;  // nothing to go on with: all warps help
        if (!last && warp != turn % LP_WARPS) continue;
        const bool lead = !last || warp == 0;
        unsigned before = 0;
        LpBest best = lp_none();
        auto whole = [&] {  // sums over the lanes: every lane writes an alternative and needs them
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                sums = lp_join(sums, lp_shuffle(sums, o));
                before += __shfl_xor_sync(0xffffffffu, before, o);
            }
        };
        const bool few = A.top <= LP_FEW;
        auto merge = [&] {  // the warps' lists
            if constexpr (TOP) {
                if (few) {
                    if (lead) best = lp_heads(best_s[use][0], LP_WARPS, 32, A.top, lane);
                } else if (last) {
                    lp_merge_warps(best_s[use]);
                    best = best_s[use][0][lane];
                } else {
                    best = best_s[use][0][lane];
#pragma unroll 1
                    for (int w = 1; w < LP_WARPS; ++w) best = lp_merge(best, best_s[use][w][lane], lane);
                }
            }
        };
        if (lead) {
            sums = lane < LP_WARPS ? sums_s[use][lane] : LpSums{-INFINITY, LP_LOWEST, 0.f, 0.f};
            before = lane < LP_WARPS ? rank_s[use][lane] : 0;
            whole();
        }
        merge();
        if (c0 || c1 < A.chunks) {
            // ---- a part: the last CTA of the row joins them all in order
            const unsigned first = row * A.chunks, f = lp_cta_of(U, C, first), l = lp_cta_of(U, C, first + A.chunks - 1);
            const unsigned slot = 2 * blockIdx.x + (blockIdx.x == f ? 1 : 0);
            unsigned all = 0;
            if (lead) {
                if (lane == 0) { A.part[slot] = sums; A.part_rank[slot] = before; }
                if (TOP) A.part_best[slot * 32 + lane] = best;
                __threadfence();
                __syncwarp();
                if (lane == 0) all = atomicAdd(&A.counters[f], 1u) == l - f;
                all = __shfl_sync(0xffffffffu, all, 0);
            }
            if (last) {
                if (tid == 0) flag_s = all;
                __syncthreads();
                all = flag_s;
            }
            if (!all) continue;
            __threadfence();
            if (lead && lane == 0) A.counters[f] = 0;
            auto slot_of = [&](unsigned p) { return 2 * (f + p) + (p == 0 ? 1 : 0); };
            const unsigned parts = l - f + 1, step = last ? LP_WARPS : 1;
            if (lead) {
                sums = LpSums{-INFINITY, LP_LOWEST, 0.f, 0.f};
                before = 0;
                for (unsigned p = lane; p < parts; p += 32) {
                    const float4 y = __ldcg(reinterpret_cast<const float4 *>(A.part) + slot_of(p));
                    sums = lp_join(sums, LpSums{y.x, y.y, y.z, y.w});
                    before += __ldcg(A.part_rank + slot_of(p));
                }
                whole();
            }
            if (TOP && few && parts <= 32) {
                // all parts' lists at once into this warp's place
                LpBest *lists = reinterpret_cast<LpBest *>(stage_s[warp]);
                if (lead) {
                    for (unsigned i = lane; i < parts * A.top; i += 32) {
                        const float2 y = __ldcg(reinterpret_cast<const float2 *>(A.part_best) + slot_of(i / A.top) * 32 + i % A.top);
                        lists[i] = LpBest{y.x, __float_as_int(y.y)};
                    }
                    __syncwarp();
                    best = lp_heads(lists, parts, A.top, A.top, lane);
                }
            } else if constexpr (TOP) {
                best = lp_none();
#pragma unroll 1
                for (unsigned p = last ? warp : 0; p < parts; p += 4 * step) {
                    float2 y[4];
#pragma unroll
                    for (unsigned u = 0; u < 4; ++u)
                        if (p + u * step < parts) y[u] = __ldcg(reinterpret_cast<const float2 *>(A.part_best) + slot_of(p + u * step) * 32 + lane);
#pragma unroll
                    for (unsigned u = 0; u < 4; ++u)
                        if (p + u * step < parts) best = lp_merge(best, LpBest{y[u].x, __float_as_int(y[u].y)}, lane);
                }
                if (last) {
                    best_s[use][warp][lane] = best;
                    __syncthreads();
                    merge();
                }
            }
        }
        if (lead) {
            const bool bad = isnan(sums.s), none = sums.top == -INFINITY && !bad;
            const float log_sum = logf(sums.s);
            if (lane == 0) {
                if (bad) raise_error(A.error, ERR_NONFINITE);
                if (A.logprob) A.logprob[row] = token < 0 ? 0.f : bad ? NAN : none ? -INFINITY : given - sums.m - log_sum;
                if (A.rank) A.rank[row] = token < 0 ? -1 : (int)before;
                if (A.entropy) A.entropy[row] = bad ? NAN : none ? 0.f : log_sum - sums.t / sums.s;
            }
            if (TOP && lane < A.top) {
                A.top_tokens[(size_t)row * A.top + lane] = best.i;
                A.top_logprobs[(size_t)row * A.top + lane] = bad ? NAN : best.i < 0 ? -INFINITY : best.v - sums.m - log_sum;
            }
        }
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
