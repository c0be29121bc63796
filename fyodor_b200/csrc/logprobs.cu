// logprobs.cu - log probability and rank of a given token, entropy and the most
// probable alternatives of rows of logits.
//
//   m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m)
//   ln p(t) = x_t - m - ln S        H = ln S - T / S
//
// One CTA a row: the maximum, then the sums and the rank, then one pass for each
// alternative (the greatest logit after the one before it in their order).
#include "common.cuh"
#include "kernels.h"
#include "fyodor_b200.h"

namespace fyb {

constexpr int LP_THREADS = 512;

struct Logprobs {
    const void *x;
    size_t stride, rows;
    unsigned n, top;
    const int *tokens;
    float *logprob, *entropy, *top_logprobs;
    int *rank, *top_tokens;
    unsigned *error;
};

template <typename V, typename Op> FYB_DEV V lp_reduce(V v, V *part, Op op)
{
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = part[0];
    for (int w = 1; w < LP_THREADS / 32; ++w) v = op(v, part[w]);
    return v;
}

template <typename T> __global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(Logprobs A)
{
    __shared__ float part_f[LP_THREADS / 32];
    __shared__ unsigned part_u[LP_THREADS / 32];
    __shared__ unsigned long long part_k[LP_THREADS / 32];
    auto fmax_ = [](float a, float b) { return fmaxf(a, b); };
    auto add = [](float a, float b) { return a + b; };
    auto addu = [](unsigned a, unsigned b) { return a + b; };
    const size_t row = blockIdx.x;
    const T *x = static_cast<const T *>(A.x) + row * A.stride;
    float m = -INFINITY;
    unsigned bad = 0;
    for (unsigned i = threadIdx.x; i < A.n; i += LP_THREADS) {
        const float v = row_value(x[i]);
        bad |= !(v < INFINITY);
        m = fmaxf(m, v);
    }
    m = lp_reduce(m, part_f, fmax_);
    bad = lp_reduce(bad, part_u, [](unsigned a, unsigned b) { return a | b; });
    int token = A.tokens ? A.tokens[row] : -1;
    if (token >= (int)A.n) {
        if (threadIdx.x == 0) raise_error(A.error, ERR_BOUNDS);
        token = -1;
    }
    const float given = token >= 0 ? row_value(x[token]) : 0.f;
    float sum = 0.f, weighted = 0.f;
    unsigned before = 0;
    for (unsigned i = threadIdx.x; i < A.n; i += LP_THREADS) {
        const float v = row_value(x[i]), d = v - m, e = expf(d);
        if (v > -INFINITY) { sum += e; weighted = fmaf(e, d, weighted); }
        before += v > given || (v == given && (int)i < token);
    }
    sum = lp_reduce(sum, part_f, add);
    weighted = lp_reduce(weighted, part_f, add);
    before = lp_reduce(before, part_u, addu);
    const float log_sum = logf(sum);
    const bool none = m == -INFINITY && !bad;
    if (threadIdx.x == 0) {
        if (bad) raise_error(A.error, ERR_NONFINITE);
        if (A.logprob) A.logprob[row] = token < 0 ? 0.f : bad ? NAN : none ? -INFINITY : given - m - log_sum;
        if (A.rank) A.rank[row] = token < 0 ? -1 : (int)before;
        if (A.entropy) A.entropy[row] = bad ? NAN : none ? 0.f : log_sum - weighted / sum;
    }
    unsigned long long last = ~0ull;
    for (unsigned t = 0; t < A.top; ++t) {
        // key: the logit's order above the index's, so that the first of equal ones is the greatest
        unsigned long long best = 0;
        for (unsigned i = threadIdx.x; i < A.n; i += LP_THREADS) {
            const float v = row_value(x[i]) + 0.f;  // -0 counts as 0
            if (!(v > -INFINITY)) continue;
            const unsigned long long key = (unsigned long long)float_order_key(v) << 32 | (0xffffffffu - i);
            if (key < last) best = max(best, key);
        }
        best = lp_reduce(best, part_k, [](unsigned long long a, unsigned long long b) { return max(a, b); });
        last = best;
        if (threadIdx.x == 0) {
            A.top_tokens[row * A.top + t] = best ? (int)(0xffffffffu - (unsigned)best) : -1;
            A.top_logprobs[row * A.top + t] = bad ? NAN : best ? float_from_order_key((unsigned)(best >> 32)) - m - log_sum : -INFINITY;
        }
    }
}

}  // namespace fyb

using namespace fyb;

extern "C" size_t fyb_logprobs_workspace(size_t rows, uint32_t vocabulary, uint32_t top)
{
    return rows > 0x7fffffffu || !vocabulary || vocabulary > 0x7fffffffu || top > FYB_LOGPROBS_TOP ? 0 : 256;
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
    const Logprobs A{logits, stride, rows, vocabulary, top, tokens, logprob, entropy, top_logprobs, rank, top_tokens, error};
    cudaStream_t s = (cudaStream_t)stream;
    if (type == T_F32) logprobs_kernel<float><<<(unsigned)rows, LP_THREADS, 0, s>>>(A);
    else if (type == T_F16) logprobs_kernel<__half><<<(unsigned)rows, LP_THREADS, 0, s>>>(A);
    else logprobs_kernel<__nv_bfloat16><<<(unsigned)rows, LP_THREADS, 0, s>>>(A);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
