// kv8_attention.cu - causal attention of requests' newest rows over the paged
// 8-bit KV cache.
//
// S = (q . k_q) k_scale scale, p = exp(S - max), out = sum p v_scale v_q / sum p,
// the maximum and the sum kept while the cache passes by once.
#include "kv8_attention.cuh"

namespace fyb {

constexpr unsigned KA_THREADS = 128;

// One CTA per (row, head): thread = position for the scores, thread = head
// dimension for the value sums.
template <typename T, int HD, unsigned FMT>
__global__ void __launch_bounds__(KA_THREADS) kv8_attention_kernel(Kv8Attention A)
{
    __shared__ float q_s[HD], p_s[KA_THREADS], red[KA_THREADS / 32];
    __shared__ float part[KA_THREADS];
    const unsigned tid = threadIdx.x, head = blockIdx.y, kv = A.c.kv_heads, kvh = head / (A.heads / kv);
    const unsigned size = 1u << A.shift;
    const size_t row = blockIdx.x;
    unsigned r = (unsigned)row;
    int start = (int)row, n = 1;
    if (A.row_start) {
        unsigned lo = 0, hi = A.requests;
        while (hi - lo > 1) {
            const unsigned mid = (lo + hi) / 2;
            if (A.row_start[mid] <= (int)row) lo = mid; else hi = mid;
        }
        r = lo;
        start = A.row_start[r];
        n = A.row_start[r + 1] - start;
    }
    const int j = (int)row - start;
    if (r >= A.requests || j < 0 || j >= n) return;
    if ((unsigned)j >= A.max_rows) { if (tid == 0) raise_error(A.error, ERR_BOUNDS); return; }
    int len = A.lengths[r];
    if (len > (long long)A.table_stride * size) { len = 0; if (tid == 0) raise_error(A.error, ERR_BOUNDS); }
    const int end = len - n + j + 1;
    const T *q = static_cast<const T *>(A.q) + row * A.q_stride + (size_t)head * HD;
    for (unsigned i = tid; i < HD; i += KA_THREADS) q_s[i] = row_value(q[i]);
    float m = -INFINITY, l = 0.f, acc = 0.f;
    constexpr unsigned GROUPS = KA_THREADS / HD;
    const unsigned d = tid % HD, g = tid / HD;
    const int *table = A.table + (size_t)r * A.table_stride;
    const unsigned char *kc = static_cast<const unsigned char *>(A.c.k), *vc = static_cast<const unsigned char *>(A.c.v);
    __syncthreads();
    for (int base = 0; base < end; base += KA_THREADS) {
        const int p = base + (int)tid;
        float s = -INFINITY;
        if (p < end) {
            const int id = table[p >> A.shift];
            if (id >= 0 && (unsigned)id < A.c.blocks) {
                const size_t at = (size_t)id * kv + kvh;
                const uint4 *kr = reinterpret_cast<const uint4 *>(kc + ((at << A.shift) + (p & (size - 1))) * HD);
                float dot = 0.f;
                for (unsigned w = 0; w < HD / 16; ++w) {
                    const uint4 u = kr[w];
                    const unsigned x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e = 0; e < 16; ++e) dot = fmaf(q_s[w * 16 + e], kv8_number<FMT>((x[e / 4] >> 8 * (e % 4)) & 0xffu), dot);
                }
                s = dot * A.c.k_scale[at] * (A.scale * 0.69314718f);
            } else {
                raise_error(A.error, ERR_BOUNDS);
            }
        }
        float top = warp_max(s);
        if (tid % 32 == 0) red[tid / 32] = top;
        __syncthreads();
        top = red[0];
        for (unsigned w = 1; w < KA_THREADS / 32; ++w) top = fmaxf(top, red[w]);
        const float m2 = fmaxf(m, top), ref = m2 == -INFINITY ? 0.f : m2;
        const float alpha = expf(m - ref), pr = expf(s - ref);
        m = m2;
        float sum = warp_sum(pr);
        __syncthreads();
        if (tid % 32 == 0) red[tid / 32] = sum;
        p_s[tid] = pr;
        __syncthreads();
        sum = 0.f;
        for (unsigned w = 0; w < KA_THREADS / 32; ++w) sum += red[w];
        l = l * alpha + sum;
        acc *= alpha;
        for (unsigned i = g; i < KA_THREADS && base + (int)i < end; i += GROUPS) {
            const int pp = base + (int)i, id = table[pp >> A.shift];
            if (id < 0 || (unsigned)id >= A.c.blocks) continue;
            const size_t at = (size_t)id * kv + kvh;
            acc = fmaf(p_s[i] * A.c.v_scale[at], kv8_number<FMT>(vc[((at << A.shift) + (pp & (size - 1))) * HD + d]), acc);
        }
        __syncthreads();
    }
    part[tid] = acc;
    __syncthreads();
    if (tid < HD) {
        for (unsigned k = 1; k < GROUPS; ++k) acc += part[tid + k * HD];
        T *out = static_cast<T *>(A.out) + row * A.out_stride + (size_t)head * HD;
        out[tid] = row_round<T>(l > 0.f || isnan(l) ? acc / l : 0.f);
    }
}

template <typename T> static void attention_launch(const Kv8Attention &A, dim3 grid, cudaStream_t s)
{
    if (A.c.head_dim == 128) {
        if (A.c.format == FYB_KV8_INT8) kv8_attention_kernel<T, 128, FYB_KV8_INT8><<<grid, KA_THREADS, 0, s>>>(A);
        else kv8_attention_kernel<T, 128, FYB_KV8_E4M3><<<grid, KA_THREADS, 0, s>>>(A);
    } else {
        if (A.c.format == FYB_KV8_INT8) kv8_attention_kernel<T, 64, FYB_KV8_INT8><<<grid, KA_THREADS, 0, s>>>(A);
        else kv8_attention_kernel<T, 64, FYB_KV8_E4M3><<<grid, KA_THREADS, 0, s>>>(A);
    }
}

}  // namespace fyb

using namespace fyb;

extern "C" size_t fyb_kv8_attention_workspace(uint32_t requests, uint32_t max_rows, uint32_t heads, uint32_t kv_heads,
    uint32_t head_dim)
{
    if (!requests || !max_rows || !kv_heads || heads < kv_heads || heads % kv_heads || heads / kv_heads > 64 ||
        (head_dim != 64 && head_dim != 128))
        return 0;
    return KA_COUNTER_BYTES + kv8_decode_part_bytes(head_dim);
}

extern "C" int fyb_kv8_attention(const fyb_kv8_cache *cache, const int32_t *lengths, const int32_t *row_start,
    uint32_t requests, uint32_t max_rows, size_t rows, const int32_t *table, size_t table_stride, uint32_t type,
    const void *q, size_t q_stride, void *out, size_t out_stride, uint32_t heads, float scale, void *workspace,
    size_t workspace_bytes, uint32_t *error, void *stream)
{
    if (kv8_check(cache) || (type != T_F32 && type != T_F16 && type != T_BF16) || table_stride == 0 ||
        table_stride > 0x7fffffffu || rows > 0x7fffffffu)
        return -1;
    const size_t need = fyb_kv8_attention_workspace(requests, max_rows, heads, cache->kv_heads, cache->head_dim);
    const size_t row = (size_t)heads * cache->head_dim;
    if (!need || !lengths || !table || !q || !out || q_stride < row || out_stride < row || !workspace || (uintptr_t)workspace % 16 ||
        workspace_bytes < need || (!row_start && rows != requests))
        return -1;
    if (!rows) return 0;
    Kv8Attention A{};
    A.c = *cache;
    A.lengths = lengths; A.row_start = row_start; A.table = table; A.table_stride = table_stride;
    A.rows = (unsigned)rows; A.q = q; A.q_stride = q_stride; A.out = out; A.out_stride = out_stride;
    A.requests = requests; A.max_rows = max_rows; A.heads = heads; A.shift = kv8_shift(cache);
    A.scale = scale * 1.44269504f; A.error = error;
    A.type = type; A.group = heads / cache->kv_heads; A.row_tile = max_rows;
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    A.counters = reinterpret_cast<unsigned *>(ws);
    A.part_ml = reinterpret_cast<float2 *>(ws + KA_COUNTER_BYTES);
    A.part_o = reinterpret_cast<float *>(A.part_ml + 2 * KA_GRID * KV8_DECODE_ROWS);
    if ((unsigned long long)max_rows * A.group <= KV8_DECODE_ROWS) return launch_kv8_decode(A, (cudaStream_t)stream);
    const dim3 grid((unsigned)rows, heads);
    cudaStream_t s = (cudaStream_t)stream;
    if (type == T_F32) attention_launch<float>(A, grid, s);
    else if (type == T_F16) attention_launch<__half>(A, grid, s);
    else attention_launch<__nv_bfloat16>(A, grid, s);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
