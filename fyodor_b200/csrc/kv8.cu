// kv8.cu - rows into and out of the paged 8-bit KV cache.
//
// Append: a block's scale is s' = max(s, max|x| (1 / top)) over the values it
// was ever given (top 127 or 448, its reciprocal rounded to F32); a new value
// is stored as round(x / s'), and where s' > s the block's older tokens are
// stored anew as round(q (s / s')). Every product and quotient is the IEEE one
// in F32, so the stored bytes are defined to the bit. Bound by memory: each row is read once and written in a byte a
// value.
//
// The rows of one block are adjacent in the slot list, so the first of them
// (the row whose predecessor lies in another block) speaks for the block: one
// CTA takes its whole run for one KV head of K or of V, and no two CTAs touch
// the same block of a head.
#include "rope.cuh"
#include "kv8.cuh"

namespace fyb {

constexpr unsigned KV8_THREADS = 256;

struct Kv8Append {
    fyb_kv8_cache c;
    const int *slots, *positions;
    const void *k, *v;
    size_t k_stride, v_stride, rows;
    RopeTable rope;   // rope.cos null: K is stored as it comes
    RopeRows q;       // rotated in the same launch (heads 0: none)
    unsigned shift, window, items;
    bool vec;
    unsigned *error;
};

// E consecutive values of one head's row at e, rotated when `turn`.
template <typename T, int HD, int E>
FYB_DEV void kv8_row(const Kv8Append &A, const T *row, unsigned e, bool turn, size_t tab, float (&x)[E])
{
    if (A.vec) row_load<T, E, true>(row + e, x); else row_load<T, E, false>(row + e, x);
    if (!turn) return;
    const float *c = A.rope.cos + tab, *s = A.rope.sin + tab;
    if (A.rope.layout == 0) {
#pragma unroll
        for (int i = 0; i < E; i += 2)
            if (e + i < A.rope.dims) rope_turn(x[i], x[i + 1], c[(e + i) / 2], s[(e + i) / 2]);
    } else {
        const unsigned pairs = A.rope.dims / 2;
        if (e >= A.rope.dims) return;
        const bool low = e < pairs;  // dims / 2 is a multiple of E: a run lies in one half
        float y[E];
        const unsigned other = low ? e + pairs : e - pairs, p = low ? e : e - pairs;
        if (A.vec) row_load<T, E, true>(row + other, y); else row_load<T, E, false>(row + other, y);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (low) rope_turn(x[i], y[i], c[p + i], s[p + i]);
            else { rope_turn(y[i], x[i], c[p + i], s[p + i]); }
        }
    }
}

// Grid (windows of rows, 2 * kv_heads + CTAs for q).
template <typename T, int HD, unsigned FMT>
__global__ void __launch_bounds__(KV8_THREADS) kv8_append_kernel(Kv8Append A)
{
    constexpr int E = HD / 32;
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t row0 = (size_t)blockIdx.x * A.window, row1 = min(row0 + A.window, A.rows);
    const unsigned part = blockIdx.y, kv = A.c.kv_heads;
    if (part >= 2 * kv) {
        const unsigned i = (part - 2 * kv) * KV8_THREADS + tid, head = i / A.items, item = i % A.items;
        if (head >= A.q.heads) return;
        for (size_t r = row0; r < row1; ++r) {
            const int pos = A.positions[r];
            if (pos < 0 || (unsigned)pos >= A.rope.rows) { if (i == 0) raise_error(A.error, ERR_BOUNDS); continue; }
            const T *in = static_cast<const T *>(A.q.in) + r * A.q.in_stride + (size_t)head * HD;
            T *out = static_cast<T *>(A.q.out) + r * A.q.out_stride + (size_t)head * HD;
            const size_t t = (size_t)pos * (A.rope.dims / 2);
            if (A.vec) rope_item<T, 16 / sizeof(T), true>(in, out, A.rope.cos + t, A.rope.sin + t, A.rope.dims, A.rope.layout, item);
            else if (A.rope.layout == 0) rope_item<T, 2, false>(in, out, A.rope.cos + t, A.rope.sin + t, A.rope.dims, 0, item);
            else rope_item<T, 1, false>(in, out, A.rope.cos + t, A.rope.sin + t, A.rope.dims, 1, item);
        }
        return;
    }
    __shared__ unsigned run_s, first_s, peak_s;
    const bool is_k = part < kv, turn = is_k && A.rope.cos;
    const unsigned head = is_k ? part : part - kv, size = 1u << A.shift;
    const T *src = static_cast<const T *>(is_k ? A.k : A.v) + (size_t)head * HD;
    const size_t stride = is_k ? A.k_stride : A.v_stride;
    unsigned char *pool = static_cast<unsigned char *>(is_k ? A.c.k : A.c.v);
    float *scales = is_k ? A.c.k_scale : A.c.v_scale;
    const int limit = (int)(A.c.blocks << A.shift);
    // the block of row r, or -1 for a row that is not stored
    auto block_of = [&](size_t r) {
        const int slot = A.slots[r];
        if (slot < 0 || slot >= limit) return -1;
        if (turn) {
            const int pos = A.positions[r];
            if (pos < 0 || (unsigned)pos >= A.rope.rows) return -1;
        }
        return slot >> A.shift;
    };
    for (size_t r0 = row0; r0 < row1; ++r0) {
        const int b = block_of(r0);
        if (b < 0) {
            if (tid == 0 && A.slots[r0] >= 0) raise_error(A.error, ERR_BOUNDS);
            continue;
        }
        if (r0 > 0 && block_of(r0 - 1) == b) continue;
        // the run of rows in block b (at most one per slot) and its lowest offset
        __syncthreads();
        if (tid == 0) { run_s = size; first_s = size; peak_s = 0u; }
        __syncthreads();
        const bool in = tid < size && r0 + tid < A.rows && block_of(r0 + tid) == b;
        if (!in && tid < size) atomicMin(&run_s, tid);
        __syncthreads();
        const unsigned run = run_s;
        if (tid < run) atomicMin(&first_s, (unsigned)A.slots[r0 + tid] & (size - 1));
        float peak = 0.f;
        bool bad = false;
        for (unsigned i = warp; i < run; i += KV8_THREADS / 32) {
            float x[E];
            const size_t tab = turn ? (size_t)A.positions[r0 + i] * (A.rope.dims / 2) : 0;
            kv8_row<T, HD, E>(A, src + (r0 + i) * stride, lane * E, turn, tab, x);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (isfinite(x[e])) peak = fmaxf(peak, fabsf(x[e])); else bad = true;
            }
        }
        if (bad) raise_error(A.error, ERR_NONFINITE);
        peak = warp_max(peak);
        if (lane == 0) atomicMax(&peak_s, __float_as_uint(peak));  // non-negative: ordered as integers
        __syncthreads();
        const unsigned first = first_s;
        const size_t at = (size_t)b * kv + head;
        const float was = first ? scales[at] : 0.f;
        const float now = fmaxf(was, kv8_scale(FMT, __uint_as_float(peak_s)));
        unsigned char *blk = pool + at * size * HD;
        if (now > was && first) {
            const float keep = __fdiv_rn(was, now);
            unsigned *w = reinterpret_cast<unsigned *>(blk);
            for (unsigned i = tid; i < first * HD / 4; i += KV8_THREADS) {
                const unsigned old = w[i];
                unsigned q = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    q |= kv8_store<FMT>(__fmul_rn(kv8_number<FMT>((old >> 8 * e) & 0xffu), keep)) << 8 * e;
                w[i] = q;
            }
        }
        for (unsigned i = warp; i < run; i += KV8_THREADS / 32) {
            float x[E];
            const size_t tab = turn ? (size_t)A.positions[r0 + i] * (A.rope.dims / 2) : 0;
            kv8_row<T, HD, E>(A, src + (r0 + i) * stride, lane * E, turn, tab, x);
            unsigned q = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float y = now > 0.f ? __fdiv_rn(x[e], now) : 0.f;
                if (!isfinite(x[e])) y = isnan(x[e]) ? 0.f : copysignf(kv8_top(FMT), x[e]);
                q |= kv8_store<FMT>(y) << 8 * e;
            }
            unsigned char *dst = blk + ((unsigned)A.slots[r0 + i] & (size - 1)) * HD + lane * E;
            if constexpr (E == 4) *reinterpret_cast<unsigned *>(dst) = q;
            else *reinterpret_cast<unsigned short *>(dst) = (unsigned short)q;
        }
        __syncthreads();
        if (tid == 0) scales[at] = now;
    }
}

// Values at slots: thread = 4 consecutive values of K and of V.
template <unsigned FMT>
__global__ void __launch_bounds__(256) kv8_read_kernel(fyb_kv8_cache c, const int *slots, size_t rows, float *k, float *v,
    unsigned shift, unsigned *error)
{
    const unsigned per_head = c.head_dim / 4, per_row = c.kv_heads * per_head;
    const size_t n = rows * per_row;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t r = i / per_row;
        const unsigned j = (unsigned)(i % per_row), head = j / per_head, e = j % per_head;
        const int slot = slots[r];
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
        if (slot >= 0 && slot < (int)(c.blocks << shift)) {
            const size_t at = (size_t)(slot >> shift) * c.kv_heads + head;
            const size_t off = ((at << shift) + ((unsigned)slot & ((1u << shift) - 1))) * per_head + e;
            const unsigned kw = static_cast<const unsigned *>(c.k)[off], vw = static_cast<const unsigned *>(c.v)[off];
            const float ks = c.k_scale[at], vs = c.v_scale[at];
            auto four = [](unsigned w, float s) {
                return make_float4(kv8_number<FMT>(w & 0xffu) * s, kv8_number<FMT>((w >> 8) & 0xffu) * s,
                                   kv8_number<FMT>((w >> 16) & 0xffu) * s, kv8_number<FMT>(w >> 24) * s);
            };
            a = four(kw, ks);
            b = four(vw, vs);
        } else if (slot >= 0) {
            raise_error(error, ERR_BOUNDS);
        }
        reinterpret_cast<float4 *>(k)[i] = a;
        reinterpret_cast<float4 *>(v)[i] = b;
    }
}

template <typename T> static void append_launch(const Kv8Append &A, dim3 grid, cudaStream_t s)
{
    if (A.c.head_dim == 128) {
        if (A.c.format == FYB_KV8_INT8) kv8_append_kernel<T, 128, FYB_KV8_INT8><<<grid, KV8_THREADS, 0, s>>>(A);
        else kv8_append_kernel<T, 128, FYB_KV8_E4M3><<<grid, KV8_THREADS, 0, s>>>(A);
    } else {
        if (A.c.format == FYB_KV8_INT8) kv8_append_kernel<T, 64, FYB_KV8_INT8><<<grid, KV8_THREADS, 0, s>>>(A);
        else kv8_append_kernel<T, 64, FYB_KV8_E4M3><<<grid, KV8_THREADS, 0, s>>>(A);
    }
}

}  // namespace fyb

using namespace fyb;

extern "C" int fyb_kv8_append(const fyb_kv8_cache *cache, const int32_t *slots, size_t rows, uint32_t type, const void *k,
    size_t k_stride, const void *v, size_t v_stride, const fyb_rope_desc *rope, const int32_t *positions, const void *q,
    size_t q_stride, void *q_out, size_t q_out_stride, uint32_t heads, uint32_t *error, void *stream)
{
    if (kv8_check(cache) || rows > 0x7fffffffu || (type != T_F32 && type != T_F16 && type != T_BF16)) return -1;
    const unsigned hd = cache->head_dim, kv = cache->kv_heads;
    const size_t width = type == T_F32 ? 4 : 2;
    Kv8Append A{};
    if (!k || !v || k_stride < (size_t)kv * hd || v_stride < (size_t)kv * hd || (heads && !rope) || heads > 65536)
        return -1;
    if (rope && (rope_table_of(rope, &A.rope) || A.rope.dims > hd || (A.rope.layout != 0 && A.rope.dims % 8)))
        return -1;
    if (heads && (!q || !q_out || q_stride < (size_t)heads * hd || q_out_stride < (size_t)heads * hd ||
                  (q == q_out && q_stride != q_out_stride)))
        return -1;
    if (!rows) return 0;
    if (!slots || (rope && !positions)) return -1;
    A.c = *cache;
    A.slots = slots; A.positions = positions;
    A.k = k; A.v = v; A.k_stride = k_stride; A.v_stride = v_stride; A.rows = rows;
    A.q = RopeRows{q, q_out, q_stride, q_out_stride, heads};
    A.shift = kv8_shift(cache);
    A.error = error;
    const size_t el = 16 / width;  // elements of a 16-byte access
    A.vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && k_stride % el == 0 && v_stride % el == 0;
    if (rope) A.vec = A.vec && rope_vectors(A.rope, hd, width, A.q);
    unsigned q_parts = 0;
    if (heads) {
        A.items = rope_items(hd, A.rope.dims, A.rope.layout, A.vec ? (unsigned)el : A.rope.layout == 0 ? 2u : 1u);
        q_parts = (unsigned)(((size_t)heads * A.items + KV8_THREADS - 1) / KV8_THREADS);
    }
    if (2 * (size_t)kv + q_parts > 65535) return -1;
    // a CTA looks at one row while that makes at most 16 CTAs per SM, at up to
    // a block of rows beyond: a prompt's rows mostly follow one another
    A.window = 1;
    while (A.window < cache->block_size && rows / A.window * 2 * kv > 16 * 148) A.window *= 2;
    const dim3 grid((unsigned)((rows + A.window - 1) / A.window), 2 * kv + q_parts);
    cudaStream_t s = (cudaStream_t)stream;
    if (type == T_F32) append_launch<float>(A, grid, s);
    else if (type == T_F16) append_launch<__half>(A, grid, s);
    else append_launch<__nv_bfloat16>(A, grid, s);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int fyb_kv8_read(const fyb_kv8_cache *cache, const int32_t *slots, size_t rows, float *k, float *v,
    uint32_t *error, void *stream)
{
    if (kv8_check(cache) || !k || !v || ((uintptr_t)k | (uintptr_t)v) % 16 || rows > 0x7fffffffu) return -1;
    if (!rows) return 0;
    if (!slots) return -1;
    const size_t n = rows * cache->kv_heads * (cache->head_dim / 4);
    const unsigned grid = (unsigned)std::min<size_t>((n + 255) / 256, 148 * 16);
    if (cache->format == FYB_KV8_INT8)
        kv8_read_kernel<FYB_KV8_INT8><<<grid, 256, 0, (cudaStream_t)stream>>>(*cache, slots, rows, k, v, kv8_shift(cache), error);
    else
        kv8_read_kernel<FYB_KV8_E4M3><<<grid, 256, 0, (cudaStream_t)stream>>>(*cache, slots, rows, k, v, kv8_shift(cache), error);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
