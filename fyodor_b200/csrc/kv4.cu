// kv4.cu - rows into and out of the paged 4-bit KV cache.
//
// Append: of a group's finite values, clamped to +-KV4_MOST, low and high are
// the least and the greatest rounded to F16, scale = F16((high - low) / 15); a
// value is held as the whole number nearest to (x - low) / scale, ties to even,
// in 0..15. Every rounding is defined (quotients and borders as real numbers),
// so the stored bits are. A token's groups need nothing of its neighbours: a
// thread takes eight values (one word), eight lanes a group, whose bounds they
// find by shuffles.
#include "rope.cuh"
#include "kv4.cuh"

namespace fyb {

constexpr unsigned KV4_THREADS = 256;

struct Kv4Append {
    fyb_kv4_cache c;
    const int *slots, *positions;
    const void *k, *v;
    size_t k_stride, v_stride, rows;
    RopeTable rope;   // rope.cos null: K is stored as it comes
    RopeRows q;       // rotated in the same launch where rows are few (heads 0: none)
    RopeWork work;
    unsigned shift, ctas, q_rows;  // ctas: of K and V; q_rows: CTAs of a row of q
    bool vec, many;
    unsigned *error;
};

// Eight values from e of a row's head in F32, rotated when `turn`; row: the head's first value.
template <typename T> FYB_DEV void kv4_load(const Kv4Append &A, const T *row, unsigned e, bool turn, size_t tab, float (&x)[8])
{
    const float *c = A.rope.cos + tab, *s = A.rope.sin + tab;
    const unsigned dims = A.rope.dims, pairs = dims / 2;
    if (A.vec) {
        constexpr int V = 16 / sizeof(T);
        auto eight = [](const T *p, float (&y)[8]) {
#pragma unroll
            for (int i = 0; i < 8; i += V) {
                const RopePack<T, V> u = rope_get<T, V, true>(p + i);
#pragma unroll
                for (int j = 0; j < V; ++j) y[i + j] = row_value(u.t[j]);
            }
        };
        eight(row + e, x);
        if (!turn || e >= dims) return;
        if (A.rope.layout == 0) {
            float cv[4], sv[4];
            rope_row<4, true>(c + e / 2, cv);
            rope_row<4, true>(s + e / 2, sv);
#pragma unroll
            for (int i = 0; i < 4; ++i) rope_turn(x[2 * i], x[2 * i + 1], cv[i], sv[i]);
        } else {
            const bool low = e < pairs;  // pairs is a multiple of 8: the eight lie in one half
            const unsigned p = low ? e : e - pairs;
            float o[8], cv[8], sv[8];
            eight(row + (low ? e + pairs : p), o);
            rope_row<8, true>(c + p, cv);
            rope_row<8, true>(s + p, sv);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (low) rope_turn(x[i], o[i], cv[i], sv[i]); else rope_turn(o[i], x[i], cv[i], sv[i]);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = row_value(row[e + i]);
    if (!turn) return;
    if (A.rope.layout == 0) {
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            if (e + i < dims) rope_turn(x[i], x[i + 1], c[(e + i) / 2], s[(e + i) / 2]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned d = e + i;
            if (d >= dims) continue;
            const bool low = d < pairs;
            const unsigned p = low ? d : d - pairs;
            float o = row_value(row[low ? d + pairs : p]);
            if (low) rope_turn(x[i], o, c[p], s[p]); else rope_turn(o, x[i], c[p], s[p]);
        }
    }
}

// The number nearest to (x - low) / scale, 0..15, ties to even. `inv` is the F32 reciprocal of scale: the F32 quotient
// y is within 4e-6 of the real one where it matters (0 <= y <= 15.1), so only next to a border between two numbers is
// more needed: there x and the border, exact in 64 bits, are compared.
FYB_DEV unsigned kv4_number(float x, float low, float scale, float inv)
{
    const float y = fminf(fmaxf(__fmul_rn(__fsub_rn(x, low), inv), 0.f), 15.f);  // NaN to 0
    const float n = rintf(y);
    if (fabsf(fabsf(y - n) - 0.5f) > 1e-5f) return (unsigned)n;
    const unsigned k = (unsigned)y;
    const double border = (double)low + ((double)k + 0.5) * (double)scale;
    return x > border || (x == border && (k & 1)) ? k + 1 : k;
}

// CTAs of K and V: thread = word w of one head of one row of K or V; then those of q.
template <typename T, int HD> __global__ void __launch_bounds__(KV4_THREADS) kv4_append_kernel(Kv4Append A)
{
    constexpr unsigned WORDS = HD / 8, GROUPS = HD / KV4_GROUP;
    if (blockIdx.x >= A.ctas) {
        rope_row_of_q<T, HD, KV4_THREADS>(A, blockIdx.x - A.ctas);
        return;
    }
    const unsigned per_row = 2 * A.c.kv_heads * WORDS;
    const size_t i = (size_t)blockIdx.x * KV4_THREADS + threadIdx.x;
    const size_t row = i / per_row;
    const unsigned j = (unsigned)(i % per_row);
    const bool is_k = j < per_row / 2;
    const unsigned head = (is_k ? j : j - per_row / 2) / WORDS, lane = j % WORDS;
    const unsigned group = lane / 8, word = (lane % 8) * GROUPS + group, e = kv4_first<HD>(word);
    const bool turn = is_k && A.rope.cos;
    // the eight lanes of a group take the same way
    int slot = -1, pos = 0;
    if (row < A.rows) {
        slot = A.slots[row];
        if (turn) pos = A.positions[row];
        if (slot >= (int)(A.c.blocks << A.shift) || (slot >= 0 && turn && (unsigned)pos >= A.rope.rows)) {
            if (lane == 0) raise_error(A.error, ERR_BOUNDS);
            slot = -1;
        }
    }
    float x[8];
    float low = INFINITY, high = -INFINITY;
    bool bad = false;
    if (slot >= 0) {
        const T *src = static_cast<const T *>(is_k ? A.k : A.v) + row * (is_k ? A.k_stride : A.v_stride) + (size_t)head * HD;
        kv4_load<T>(A, src, e, turn, turn ? (size_t)pos * (A.rope.dims / 2) : 0, x);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const bool finite = fabsf(x[t]) <= 3.4028235e38f;
            bad = bad || !finite;
            low = fminf(low, finite ? x[t] : INFINITY);
            high = fmaxf(high, finite ? x[t] : -INFINITY);
        }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    if (slot < 0) return;
    if (bad) raise_error(A.error, ERR_NONFINITE);
    if (low > high) low = high = 0.f;  // nothing finite
    const __half lo = __float2half_rn(fminf(fmaxf(low, -KV4_MOST), KV4_MOST));
    const __half hi = __float2half_rn(fminf(fmaxf(high, -KV4_MOST), KV4_MOST));
    const float lf = __half2float(lo);
    const __half sc = __float2half_rn(__fdiv_rn(__fsub_rn(__half2float(hi), lf), 15.f));
    const float sf = __half2float(sc), inv = sf > 0.f ? __frcp_rn(sf) : 0.f;
    unsigned bits = 0;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        float y = x[t];
        if (bad && isnan(y)) y = 0.f;   // held as near to 0 as the group's values are
        if (sf > 0.f) bits |= kv4_number(y, lf, sf, inv) << (4 * t);
    }
    const size_t at = (((size_t)(slot >> A.shift) * A.c.kv_heads + head) << A.shift) + ((unsigned)slot & ((1u << A.shift) - 1));
    static_cast<unsigned *>(is_k ? A.c.k : A.c.v)[at * WORDS + word] = bits;
    if (lane % 8 == 0) static_cast<__half2 *>(is_k ? A.c.k_scale : A.c.v_scale)[at * GROUPS + group] = __halves2half2(sc, lo);
}

// Values at slots: thread = word w of K and of V of one head of a row.
template <int HD>
__global__ void __launch_bounds__(256) kv4_read_kernel(fyb_kv4_cache c, const int *slots, size_t rows, float *k, float *v,
    unsigned shift, unsigned *error)
{
    constexpr unsigned WORDS = HD / 8, GROUPS = HD / KV4_GROUP;
    const unsigned per_row = c.kv_heads * WORDS;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, row = i / per_row;
    const unsigned j = (unsigned)(i % per_row), head = j / WORDS, lane = j % WORDS;
    if (row >= rows) return;
    const unsigned group = lane / 8, word = (lane % 8) * GROUPS + group;
    int slot = slots[row];
    if (slot >= (int)(c.blocks << shift)) {
        if (lane == 0) raise_error(error, ERR_BOUNDS);
        slot = -1;
    }
    unsigned kw = 0, vw = 0;
    float2 ks = make_float2(0.f, 0.f), vs = ks;
    if (slot >= 0) {
        const size_t at = (((size_t)(slot >> shift) * c.kv_heads + head) << shift) + ((unsigned)slot & ((1u << shift) - 1));
        kw = static_cast<const unsigned *>(c.k)[at * WORDS + word];
        vw = static_cast<const unsigned *>(c.v)[at * WORDS + word];
        ks = __half22float2(static_cast<const __half2 *>(c.k_scale)[at * GROUPS + group]);
        vs = __half22float2(static_cast<const __half2 *>(c.v_scale)[at * GROUPS + group]);
    }
    const size_t out = (row * c.kv_heads + head) * HD + kv4_first<HD>(word);
    auto eight = [&](float *p, unsigned w, float2 s) {
        float4 *o = reinterpret_cast<float4 *>(p + out);
        o[0] = make_float4(kv4_value(w, 0, s), kv4_value(w, 1, s), kv4_value(w, 2, s), kv4_value(w, 3, s));
        o[1] = make_float4(kv4_value(w, 4, s), kv4_value(w, 5, s), kv4_value(w, 6, s), kv4_value(w, 7, s));
    };
    eight(k, kw, ks);
    eight(v, vw, vs);
}

template <typename T> static void append_launch(const Kv4Append &A, unsigned grid, cudaStream_t s)
{
    if (A.c.head_dim == 128) kv4_append_kernel<T, 128><<<grid, KV4_THREADS, 0, s>>>(A);
    else kv4_append_kernel<T, 64><<<grid, KV4_THREADS, 0, s>>>(A);
}

}  // namespace fyb

using namespace fyb;

extern "C" int fyb_kv4_append(const fyb_kv4_cache *cache, const int32_t *slots, size_t rows, uint32_t type, const void *k,
    size_t k_stride, const void *v, size_t v_stride, const fyb_rope_desc *rope, const int32_t *positions, const void *q,
    size_t q_stride, void *q_out, size_t q_out_stride, uint32_t heads, uint32_t *error, void *stream)
{
    if (kv4_check(cache) || rows > 0x7fffffffu || (type != T_F32 && type != T_F16 && type != T_BF16)) return -1;
    const unsigned hd = cache->head_dim, kv = cache->kv_heads;
    const size_t width = type == T_F32 ? 4 : 2, el = 16 / width;  // el: elements of a 16-byte access
    Kv4Append A{};
    if ((rows && (!k || !v)) || k_stride < (size_t)kv * hd || v_stride < (size_t)kv * hd || (heads && !rope) || heads > 65536)
        return -1;
    if (rope && (rope_table_of(rope, &A.rope) || A.rope.dims > hd)) return -1;
    if (heads && ((rows && (!q || !q_out)) || q_stride < (size_t)heads * hd || q_out_stride < (size_t)heads * hd ||
                  (q == q_out && q_stride != q_out_stride)))
        return -1;
    if (!rows) return 0;
    if (!slots || (rope && !positions)) return -1;
    A.c = *cache;
    A.slots = slots; A.positions = positions;
    A.k = k; A.v = v; A.k_stride = k_stride; A.v_stride = v_stride; A.rows = rows;
    A.q = RopeRows{q, q_out, q_stride, q_out_stride, heads};
    A.shift = kv4_shift(cache);
    A.error = error;
    // 16-byte accesses to rows and tables: eight values of a thread rotate alike, their tables' rows are aligned
    A.vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && k_stride % el == 0 && v_stride % el == 0;
    if (rope) A.vec = A.vec && rope_vectors(A.rope, hd, width, A.q) && A.rope.dims % (A.rope.layout == 0 ? 8 : 16) == 0 &&
                    ((uintptr_t)A.rope.cos | (uintptr_t)A.rope.sin) % 16 == 0;
    cudaStream_t s = (cudaStream_t)stream;
    const size_t ctas = (rows * 2 * kv * (hd / 8) + KV4_THREADS - 1) / KV4_THREADS;
    if (heads && rows > 148) {  // a launch more is little beside a prompt
        const int r = rope_run(type, A.rope, positions, rows, hd, A.q, RopeRows{}, error, s);
        if (r) return r;
    } else if (heads) {
        A.work = rope_work(hd, A.rope.dims, A.rope.layout, A.vec ? (unsigned)el : A.rope.layout == 0 ? 2u : 1u, q == q_out);
        A.many = A.vec && rope_many(rows, heads, A.work);
        const unsigned groups = A.many ? (heads + ROPE_HEADS - 1) / ROPE_HEADS : heads;
        A.q_rows = (unsigned)(((size_t)groups * (A.work.turned + A.work.copied) + KV4_THREADS - 1) / KV4_THREADS);
    }
    const size_t grid = ctas + rows * A.q_rows;
    if (grid > 0x7fffffffu) return -1;
    A.ctas = (unsigned)ctas;
    if (type == T_F32) append_launch<float>(A, (unsigned)grid, s);
    else if (type == T_F16) append_launch<__half>(A, (unsigned)grid, s);
    else append_launch<__nv_bfloat16>(A, (unsigned)grid, s);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int fyb_kv4_read(const fyb_kv4_cache *cache, const int32_t *slots, size_t rows, float *k, float *v,
    uint32_t *error, void *stream)
{
    if (kv4_check(cache) || (rows && (!k || !v)) || ((uintptr_t)k | (uintptr_t)v) % 16 || rows > 0x7fffffffu) return -1;
    if (!rows) return 0;
    if (!slots) return -1;
    const size_t ctas = (rows * cache->kv_heads * (cache->head_dim / 8) + 255) / 256;
    if (ctas > 0x7fffffffu) return -1;
    cudaStream_t s = (cudaStream_t)stream;
    if (cache->head_dim == 128) kv4_read_kernel<128><<<(unsigned)ctas, 256, 0, s>>>(*cache, slots, rows, k, v, kv4_shift(cache), error);
    else kv4_read_kernel<64><<<(unsigned)ctas, 256, 0, s>>>(*cache, slots, rows, k, v, kv4_shift(cache), error);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
