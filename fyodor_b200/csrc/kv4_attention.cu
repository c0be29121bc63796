// kv4_attention.cu - the entry point of attention over the paged 4-bit cache:
// argument checks, the workspace, and which kernel runs. Up to eight query rows
// per KV head run on kv4_decode.cu.
//
// Many rows: a warp takes one query row of one head and walks the positions it attends:
// lanes share out the head's dimensions, and of a group the score is scale (q . n)
// + low sum(q), so the held numbers are used as they lie.
#include "kv4_attention.cuh"

namespace fyb {

constexpr int K4_WARPS = 8;

// K or V as token rows of head_dim / 2 bytes, boxes of one block (128 rows at most), rows of 64 bytes in the swizzle of
// 64 bytes: 16-byte chunk c of token row t lies at chunk c ^ (t >> 1 & 3).
static int kv4_tensor_map(CUtensorMap *map, const fyb_kv8_cache &c, const void *pool)
{
    return kv8_tensor_map(map, pool, c.head_dim / 2, (size_t)c.blocks * c.kv_heads * c.block_size,
                          std::min(c.block_size, (unsigned)K4_TILE), c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Lane's 16 bits of a token's row (HD 128: four values, HD 64: two, 8 bits) from its first dimension.
template <typename T, int HD> __global__ void __launch_bounds__(32 * K4_WARPS) kv4_rows_kernel(const __grid_constant__ Kv4Attention A)
{
    constexpr int E = HD / 32, GROUPS = HD / 64;
    const unsigned lane = threadIdx.x & 31, kv = A.c.kv_heads, size = 1u << A.shift;
    const size_t item = (size_t)blockIdx.x * K4_WARPS + (threadIdx.x >> 5);
    if (item >= (size_t)A.rows * A.heads) return;
    const unsigned row = (unsigned)(item / A.heads), head = (unsigned)(item % A.heads), kvh = head / A.group;
    // the request of the row
    unsigned r = row;
    Kv8Request q = kv8_request(A, 0, item == 0);
    if (A.row_start) {
        for (r = 0; r < A.requests; ++r) {
            q = kv8_request(A, r, lane == 0 && head == 0 && (int)row == max(0, A.row_start[r]));
            if ((int)row >= q.first && (int)row < q.first + q.n) break;
        }
        if (r == A.requests || (int)row >= q.first + q.rows) return;
    } else {
        q = kv8_request(A, r, lane == 0 && head == 0);
    }
    const int last = q.len - q.n + ((int)row - q.first) + 1;
    const unsigned e = lane * E, group = e / 64, word = HD == 64 ? e / 8 : (e % 64 / 8) * 2 + group;
    const T *qp = static_cast<const T *>(A.q) + row * A.q_stride + (size_t)head * HD + e;
    float x[E], sum = 0.f, o[E] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) { x[i] = row_value(qp[i]); sum += x[i]; }
    for (int t = 0; t < last; ++t) {
        const int id = A.table[(size_t)r * A.table_stride + (t >> A.shift)];
        if ((unsigned)id >= A.c.blocks) {
            if (lane == 0 && kvh * A.group == head) raise_error(A.error, ERR_BOUNDS);
            t |= (int)size - 1;
            continue;
        }
        const size_t at = ((size_t)id * kv + kvh) * size + ((unsigned)t & (size - 1));
        const unsigned kw = static_cast<const unsigned *>(A.c.k)[at * (HD / 8) + word] >> (e % 8 * 4);
        const unsigned vw = static_cast<const unsigned *>(A.c.v)[at * (HD / 8) + word] >> (e % 8 * 4);
        const float2 ks = __half22float2(A.ks[at * GROUPS + group]), vs = __half22float2(A.vs[at * GROUPS + group]);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) dot = fmaf(x[i], (float)(kw >> (4 * i) & 15u), dot);
        const float score = warp_sum(fmaf(dot, ks.x, sum * ks.y)) * A.scale;
        const float top = fmaxf(m, score), keep = m == top ? 1.f : exp2f(m - top), p = exp2f(score - top);
        m = top;
        l = fmaf(l, keep, p);
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = fmaf(o[i], keep, p * fmaf((float)(vw >> (4 * i) & 15u), vs.x, vs.y));
    }
    const float n = l > 0.f || isnan(l) ? 1.f / l : 0.f;
    T *out = static_cast<T *>(A.out) + row * A.out_stride + (size_t)head * HD + e;
#pragma unroll
    for (int i = 0; i < E; ++i) out[i] = row_round<T>(o[i] * n);
}

template <typename T> static void rows_launch(const Kv4Attention &A, unsigned grid, cudaStream_t s)
{
    if (A.c.head_dim == 128) kv4_rows_kernel<T, 128><<<grid, 32 * K4_WARPS, 0, s>>>(A);
    else kv4_rows_kernel<T, 64><<<grid, 32 * K4_WARPS, 0, s>>>(A);
}

}  // namespace fyb

using namespace fyb;

extern "C" size_t fyb_kv4_attention_workspace(uint32_t requests, uint32_t max_rows, uint32_t heads, uint32_t kv_heads,
    uint32_t head_dim)
{
    return fyb_kv8_attention_workspace(requests, max_rows, heads, kv_heads, head_dim);
}

extern "C" int fyb_kv4_attention(const fyb_kv4_cache *cache, const int32_t *lengths, const int32_t *row_start,
    uint32_t requests, uint32_t max_rows, size_t rows, const int32_t *table, size_t table_stride, uint32_t type,
    const void *q, size_t q_stride, void *out, size_t out_stride, uint32_t heads, float scale, void *workspace,
    size_t workspace_bytes, uint32_t *error, void *stream)
{
    if (kv4_check(cache) || (type != T_F32 && type != T_F16 && type != T_BF16) || table_stride == 0 ||
        table_stride > 0x7fffffffu || rows > 0x7fffffffu || max_rows > 0x7fffffffu)
        return -1;
    const size_t need = fyb_kv4_attention_workspace(requests, max_rows, heads, cache->kv_heads, cache->head_dim);
    const size_t row = (size_t)heads * cache->head_dim;
    if (!need || !lengths || !table || (rows && (!q || !out)) || q_stride < row || out_stride < row || !workspace ||
        (uintptr_t)workspace % 16 || workspace_bytes < need || (!row_start && rows != requests))
        return -1;
    if (!rows) return 0;
    Kv4Attention A{};
    A.c.k = cache->k; A.c.v = cache->v;
    A.c.blocks = cache->blocks; A.c.kv_heads = cache->kv_heads; A.c.block_size = cache->block_size;
    A.c.head_dim = cache->head_dim;
    A.ks = static_cast<const __half2 *>(cache->k_scale); A.vs = static_cast<const __half2 *>(cache->v_scale);
    A.lengths = lengths; A.row_start = row_start; A.table = table; A.table_stride = table_stride;
    A.rows = (unsigned)rows; A.q = q; A.q_stride = q_stride; A.out = out; A.out_stride = out_stride;
    A.requests = requests; A.max_rows = max_rows; A.heads = heads; A.group = heads / cache->kv_heads;
    A.shift = kv4_shift(cache); A.type = type; A.scale = scale * 1.44269504f; A.error = error;
    cudaStream_t s = (cudaStream_t)stream;
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    A.counters = reinterpret_cast<unsigned *>(ws);
    A.part_ml = reinterpret_cast<float2 *>(ws + KA_COUNTER_BYTES);
    A.part_o = reinterpret_cast<float *>(A.part_ml + 2 * KA_GRID * KV8_DECODE_ROWS);
    if ((unsigned long long)max_rows * A.group <= KV8_DECODE_ROWS) {
        CUtensorMap k, v;
        if (kv4_tensor_map(&k, A.c, A.c.k) || kv4_tensor_map(&v, A.c, A.c.v)) return -2;
        A.row_tile = max_rows;
        // no more CTAs than the most units the tables can hold
        const unsigned long long holds = (unsigned long long)table_stride << A.shift;
        const unsigned long long units = (holds + K4_TILE - 1) / K4_TILE * requests * cache->kv_heads;
        return launch_kv4_decode(A, k, v, (unsigned)std::min<unsigned long long>(KA_GRID, units), s);
    }
    const size_t grid = (rows * heads + K4_WARPS - 1) / K4_WARPS;
    if (grid > 0x7fffffffu) return -1;
    if (type == T_F32) rows_launch<float>(A, (unsigned)grid, s);
    else if (type == T_F16) rows_launch<__half>(A, (unsigned)grid, s);
    else rows_launch<__nv_bfloat16>(A, (unsigned)grid, s);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
