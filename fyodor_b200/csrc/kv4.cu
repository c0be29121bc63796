// kv4.cu - rows into and out of the paged 4-bit KV cache.
//
// Append: of a group's finite values, clamped to +-KV4_MOST, low and high are
// the least and the greatest rounded to F16, scale = F16((high - low) / 15); a
// value is held as the whole number nearest to (x - low) / scale, ties to even,
// in 0..15. Every rounding is defined (quotients and borders as real numbers),
// so the stored bits are. A token's groups need nothing of its neighbours: a
// thread takes 16 values (two words), four lanes a group, whose bounds they
// find by shuffles.
//
// A step's append is one launch, 4 us. Prompts: 6093 rows of 32 / 8 heads of 128, bf16,
// take 17 us for K and V (31 MB: instructions, some 440 a warp for 512 values), 23 for
// q's rotation (0.67 of the measured copy; in one launch with K and V 55 us together
// when one after the other took 39, so q goes along only with few rows, where a launch
// more would count) and 12 to be read back in F32 (0.79). Of the 17, 0.6 are the tests
// whether a group's numbers can leave 0..15 and its scale lies next to a border.
#include "rope.cuh"
#include "kv4.cuh"

namespace fyb {

constexpr unsigned KV4_THREADS = 256;
constexpr int KV4_EACH = 16;  // values of a thread: with 8 an append of 6093 rows of 8 heads took 307 instructions a warp, 17.9 us

// Where a CTA's threads stand among rows of `per_row` items: rows of a CTA, or CTAs of a row.
struct Kv4Grid {
    unsigned per_row, rows, parts;  // rows of a CTA (1 where a row has parts)
};
inline Kv4Grid kv4_grid(unsigned per_row)
{
    return Kv4Grid{per_row, per_row < KV4_THREADS ? KV4_THREADS / per_row : 1, (per_row + KV4_THREADS - 1) / KV4_THREADS};
}
// Thread's row and item of it; false for a thread that has none.
FYB_DEV bool kv4_place(const Kv4Grid &g, unsigned cta, size_t rows, size_t &row, unsigned &j)
{
    if (g.rows == 1) {
        row = cta;
        j = threadIdx.x;
        if (g.parts > 1) {
            row = cta / g.parts;
            j += cta % g.parts * KV4_THREADS;
        }
        return j < g.per_row;
    }
    const unsigned r = threadIdx.x / g.per_row;
    row = (size_t)cta * g.rows + r;
    j = threadIdx.x % g.per_row;
    return r < g.rows && row < rows;
}

struct Kv4Append {
    fyb_kv4_cache c;
    const int *slots, *positions;
    const void *k, *v;
    size_t k_stride, v_stride, rows;
    RopeTable rope;   // rope.cos null: K is stored as it comes
    RopeRows q;       // rotated in the same launch where rows are few (heads 0: none)
    RopeWork work;
    unsigned shift, ctas, q_rows;  // ctas: of K and V; q_rows: CTAs of a row of q
    Kv4Grid grid;
    bool vec, many;
    unsigned *error;
};

// A thread's values of a row's head as they lie there, and of the other half where half pairs are turned.
template <typename T> struct Kv4Raw {
    static constexpr int V = 16 / sizeof(T);
    RopePack<T, V> own[KV4_EACH / V], other[KV4_EACH / V];
};
// Those from e (aligned accesses): asked for before slot and position have come.
template <typename T> FYB_DEV void kv4_ask(const Kv4Append &A, const T *row, unsigned e, bool turn, Kv4Raw<T> &r)
{
    constexpr int V = Kv4Raw<T>::V;
    const unsigned pairs = A.rope.dims / 2;
#pragma unroll
    for (int i = 0; i < KV4_EACH / V; ++i) r.own[i] = rope_get<T, V, true>(row + e + i * V);
    if (turn && A.rope.layout != 0 && e < A.rope.dims) {
        const unsigned o = e < pairs ? e + pairs : e - pairs;
#pragma unroll
        for (int i = 0; i < KV4_EACH / V; ++i) r.other[i] = rope_get<T, V, true>(row + o + i * V);
    }
}
// The same in F32, rotated when `turn`; tab: the position's place in the tables.
template <typename T> FYB_DEV void kv4_turn(const Kv4Append &A, const Kv4Raw<T> &r, unsigned e, bool turn, size_t tab, float (&x)[KV4_EACH])
{
    constexpr int V = Kv4Raw<T>::V;
    const unsigned dims = A.rope.dims, pairs = dims / 2;
#pragma unroll
    for (int i = 0; i < KV4_EACH; ++i) x[i] = row_value(r.own[i / V].t[i % V]);
    if (!turn || e >= dims) return;
    if (A.rope.layout == 0) {
        float cv[KV4_EACH / 2], sv[KV4_EACH / 2];
        rope_row<KV4_EACH / 2, true>(A.rope.cos + tab + e / 2, cv);
        rope_row<KV4_EACH / 2, true>(A.rope.sin + tab + e / 2, sv);
#pragma unroll
        for (int i = 0; i < KV4_EACH / 2; ++i) rope_turn(x[2 * i], x[2 * i + 1], cv[i], sv[i]);
    } else {
        const bool low = e < pairs;  // pairs is a multiple of KV4_EACH: the values lie in one half
        const unsigned p = low ? e : e - pairs;
#pragma unroll
        for (int i = 0; i < KV4_EACH; i += 4) {
            float cv[4], sv[4];
            rope_row<4, true>(A.rope.cos + tab + p + i, cv);
            rope_row<4, true>(A.rope.sin + tab + p + i, sv);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float o = row_value(r.other[(i + j) / V].t[(i + j) % V]);
                if (low) rope_turn(x[i + j], o, cv[j], sv[j]); else rope_turn(o, x[i + j], cv[j], sv[j]);
            }
        }
    }
}
// Both, one value at a time, for rows and tables that begin anywhere.
template <typename T> __device__ __noinline__ void kv4_load(const Kv4Append &A, const T *row, unsigned e, bool turn, size_t tab, float *x)
{
    const float *c = A.rope.cos + tab, *s = A.rope.sin + tab;
    const unsigned dims = A.rope.dims, pairs = dims / 2;
    for (int i = 0; i < KV4_EACH; ++i) {
        const unsigned d = e + i;
        x[i] = row_value(row[d]);
        if (!turn || d >= dims) continue;
        if (A.rope.layout == 0) {
            float o = row_value(row[d ^ 1]);
            if (d & 1) rope_turn(o, x[i], c[d / 2], s[d / 2]); else rope_turn(x[i], o, c[d / 2], s[d / 2]);
        } else {
            const bool low = d < pairs;
            const unsigned p = low ? d : d - pairs;
            float o = row_value(row[low ? d + pairs : p]);
            if (low) rope_turn(x[i], o, c[p], s[p]); else rope_turn(o, x[i], c[p], s[p]);
        }
    }
}

FYB_DEV float max_nan(float a, float b)  // NaN where one is
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// x / 15, correctly rounded: a quotient from the rounded reciprocal, and its remainder's (Markstein 1990).
FYB_DEV float fifteenth(float x)
{
    constexpr float r = 1.f / 15.f;
    const float q = x * r;
    return fmaf(fmaf(-15.f, q, x), r, q);
}
// (high - low) / 15 of two halves as a real number, rounded to F16 once. In F32 the difference and the quotient are off by
// 2^-23 of it together, which matters only next to a border between two normal halves (of subnormal ones differences are
// exact, and quotients no nearer to a border than a thirtieth of a step): there 15 borders and the difference, exact in 64
// bits, are compared.
static __device__ __noinline__ __half kv4_scale_at(float q, float low, float high)
{
    const __half a = __float2half_rd(q), b = __float2half_ru(q);
    const double border = 7.5 * ((double)__half2float(a) + (double)__half2float(b)), d = (double)high - (double)low;
    return d > border || (d == border && (__half_as_ushort(a) & 1)) ? b : a;
}
FYB_DEV __half kv4_scale(float low, float high)
{
    const float q = fifteenth(__fsub_rn(high, low));
    if (__builtin_expect((__float_as_uint(q) & 0x1fffu) - 0xffeu <= 4u, 0)) return kv4_scale_at(q, low, high);
    return __float2half_rn(q);
}
FYB_DEV float rcp_approx(float x)  // within 2^-23 of it
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Eight numbers one by one: nearest to (x - low) / scale, 0..15, ties to even. `inv` is the reciprocal of scale within 2^-23:
// the F32 quotient y is within 4e-6 of the real one where it matters (0 <= y <= 15.1), so only next to a border between two
// numbers is more needed: there x and the border, exact in 64 bits, are compared. NaN is held as 0 would be.
static __device__ __noinline__ unsigned kv4_numbers(const float *x, float low, float scale, float inv)
{
    unsigned bits = 0;
    if (!(scale > 0.f)) return 0;
#pragma unroll 1
    for (int t = 0; t < 8; ++t) {
        const float v = isnan(x[t]) ? 0.f : x[t], y = fminf(fmaxf(__fmul_rn(__fsub_rn(v, low), inv), 0.f), 15.f), n = rintf(y);
        unsigned k = (unsigned)n;
        if (fabsf(fabsf(y - n) - 0.5f) <= 1e-5f) {
            k = (unsigned)y;
            const double border = (double)low + ((double)k + 0.5) * (double)scale;
            if (v > border || (v == border && (k & 1))) ++k;
        }
        bits |= k << (4 * t);
    }
    return bits;
}

// CTAs of K and V: thread = KV4_EACH values of one head of one row of K or V; with Q then those of q.
template <typename T, int HD, bool Q> __global__ void __launch_bounds__(KV4_THREADS) kv4_append_kernel(const __grid_constant__ Kv4Append A)
{
    constexpr unsigned LANES = HD / KV4_EACH, GROUPS = HD / KV4_GROUP, PART = KV4_GROUP / KV4_EACH;  // threads of a head, of a group
    constexpr unsigned WORDS = HD / 8;
    if (Q && blockIdx.x >= A.ctas) {
        rope_row_of_q<T, HD, KV4_THREADS>(A, blockIdx.x - A.ctas);
        return;
    }
    size_t row;
    unsigned j;
    const bool real = kv4_place(A.grid, blockIdx.x, A.rows, row, j);
    const bool is_k = j < A.grid.per_row / 2;
    const unsigned head = (is_k ? j : j - A.grid.per_row / 2) / LANES, lane = j % LANES, group = lane / PART, e = lane * KV4_EACH;
    const bool turn = is_k && A.rope.cos;
    const T *src = static_cast<const T *>(is_k ? A.k : A.v) + row * (is_k ? A.k_stride : A.v_stride) + (size_t)head * HD;
    int slot = -1, pos = 0;  // the lanes of a group take the same way
    Kv4Raw<T> raw;
    if (real) {
        if (A.vec) kv4_ask<T>(A, src, e, turn, raw);
        slot = A.slots[row];
        if (turn) pos = A.positions[row];
        if (slot >= (int)(A.c.blocks << A.shift) || (slot >= 0 && turn && (unsigned)pos >= A.rope.rows)) {
            if (lane == 0) raise_error(A.error, ERR_BOUNDS);
            slot = -1;
        }
    }
    float x[KV4_EACH];
    float low = INFINITY, high = -INFINITY;
    bool bad = false;
    if (slot >= 0) {
        const size_t tab = turn ? (size_t)pos * (A.rope.dims / 2) : 0;
        if (A.vec) {
            kv4_turn<T>(A, raw, e, turn, tab, x);
        } else {
            float y[KV4_EACH];
            kv4_load<T>(A, src, e, turn, tab, y);
#pragma unroll
            for (int t = 0; t < KV4_EACH; ++t) x[t] = y[t];
        }
        F2 nothing = f2(0.f, 0.f);  // NaN where a value is none or infinite
#pragma unroll
        for (int t = 0; t < KV4_EACH; t += 2) {
            low = fminf(fminf(low, x[t]), x[t + 1]);
            high = fmaxf(fmaxf(high, x[t]), x[t + 1]);
            nothing = f2_fma(f2(x[t], x[t + 1]), f2(0.f, 0.f), nothing);
        }
        const float2 zero = f2_get(nothing);
        bad = isnan(zero.x + zero.y);
        if (__builtin_expect(bad, 0)) {  // infinities and NaN do not count
            low = INFINITY;
            high = -INFINITY;
#pragma unroll
            for (int t = 0; t < KV4_EACH; ++t)
                if (fabsf(x[t]) <= 3.4028235e38f) {
                    low = fminf(low, x[t]);
                    high = fmaxf(high, x[t]);
                }
        }
    }
#pragma unroll
    for (unsigned o = 1; o < PART; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    if (slot < 0) return;
    if (bad) raise_error(A.error, ERR_NONFINITE);
    if (low > high) low = high = 0.f;  // nothing finite
    const __half lo = __float2half_rn(fminf(fmaxf(low, -KV4_MOST), KV4_MOST));
    const __half hi = __float2half_rn(fminf(fmaxf(high, -KV4_MOST), KV4_MOST));
    const float lf = __half2float(lo);
    const __half sc = kv4_scale(lf, __half2float(hi));
    const float sf = __half2float(sc), inv = rcp_approx(sf);  // scale 0: no number is certain
    // Low and high as F16, and scale, need not enclose the group (a range of a few steps of F16, a scale below its normal
    // numbers, values beyond KV4_MOST): where a quotient can leave 0..15 the values go one by one, which clamps (6093 F32 rows of
    // nothing else 23 us instead of 13).
    const bool wide = bad || !(__fmul_rn(__fsub_rn(low, lf), inv) >= -0.49f && __fmul_rn(__fsub_rn(high, lf), inv) <= 15.49f);
    const size_t at = (((size_t)(slot >> A.shift) * A.c.kv_heads + head) << A.shift) + ((unsigned)slot & ((1u << A.shift) - 1));
    unsigned *words = static_cast<unsigned *>(is_k ? A.c.k : A.c.v) + at * WORDS + lane % PART * (KV4_EACH / 8) * GROUPS + group;
    // Four numbers at a time as one of 16 bits. A quotient that is no nearer than 1e-5 to a border is certain; the others
    // are few, and eight values with one go one by one.
    constexpr float WHOLE = 12582912.f;  // 1.5 x 2^23: added, a number's fraction is rounded away, ties to even
#pragma unroll
    for (int w = 0; w < KV4_EACH / 8; ++w) {
        unsigned bits = 0;
        float off = 0.f;
#pragma unroll
        for (int t = 0; t < 8; t += 4) {
            F2 n[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const F2 y = f2_mul(f2_add(f2(x[8 * w + t + 2 * i], x[8 * w + t + 2 * i + 1]), f2(-lf, -lf)), f2(inv, inv));
                n[i] = f2_add(f2_add(y, f2(WHOLE, WHOLE)), f2(-WHOLE, -WHOLE));
                const float2 d = f2_get(f2_fma(n[i], f2(-1.f, -1.f), y));
                off = max_nan(off, max_nan(fabsf(d.x), fabsf(d.y)));
            }
            const float2 a = f2_get(n[0]), b = f2_get(n[1]);
            const float four = fmaf(fmaf(b.y, 16.f, b.x), 256.f, fmaf(a.y, 16.f, a.x));
            bits |= (__float_as_uint(__fadd_rn(four, WHOLE)) & 0xffffu) << (4 * t);
        }
        if (__builtin_expect(wide || !(off < 0.49999f), 0)) {
            float y[8];
#pragma unroll
            for (int t = 0; t < 8; ++t) y[t] = x[8 * w + t];
            bits = kv4_numbers(y, lf, sf, inv);
        }
        words[w * GROUPS] = bits;
    }
    if (lane % PART == 0) static_cast<__half2 *>(is_k ? A.c.k_scale : A.c.v_scale)[at * GROUPS + group] = __halves2half2(sc, lo);
}

// Values at slots: thread = half a word (four values) of K and of V of READ4_ROWS rows, all loads out before the first is
// used; a warp's stores lie together. Grid (rows / READ4_ROWS, half words of a row / 256).
constexpr int READ4_ROWS = 4;
template <int HD>
__global__ void __launch_bounds__(KV4_THREADS) kv4_read_kernel(fyb_kv4_cache c, const int *slots, size_t rows, float *k, float *v,
    unsigned shift, unsigned *error)
{
    constexpr unsigned PER = HD / 4, GROUPS = HD / KV4_GROUP;
    const unsigned per_row = c.kv_heads * PER, j = blockIdx.y * KV4_THREADS + threadIdx.x;
    if (j >= per_row) return;
    const unsigned head = j / PER, e = j % PER * 4, group = e / KV4_GROUP, word = e % KV4_GROUP / 8 * GROUPS + group;
    const size_t r0 = (size_t)blockIdx.x * READ4_ROWS;
    int slot[READ4_ROWS];
    unsigned kw[READ4_ROWS], vw[READ4_ROWS];
    __half2 ks[READ4_ROWS], vs[READ4_ROWS];
#pragma unroll
    for (int u = 0; u < READ4_ROWS; ++u) slot[u] = r0 + u < rows ? slots[r0 + u] : -1;
#pragma unroll
    for (int u = 0; u < READ4_ROWS; ++u) {
        kw[u] = vw[u] = 0;
        ks[u] = vs[u] = __half2half2(__ushort_as_half(0));
        if (slot[u] < 0) continue;
        if (slot[u] >= (int)(c.blocks << shift)) { raise_error(error, ERR_BOUNDS); continue; }
        const size_t at = (((size_t)(slot[u] >> shift) * c.kv_heads + head) << shift) + ((unsigned)slot[u] & ((1u << shift) - 1));
        kw[u] = static_cast<const unsigned *>(c.k)[at * (HD / 8) + word];
        vw[u] = static_cast<const unsigned *>(c.v)[at * (HD / 8) + word];
        ks[u] = static_cast<const __half2 *>(c.k_scale)[at * GROUPS + group];
        vs[u] = static_cast<const __half2 *>(c.v_scale)[at * GROUPS + group];
    }
    auto four = [&](unsigned w, __half2 scale_low) {
        const float2 s = __half22float2(scale_low);
        w >>= e & 4 ? 16 : 0;
        return make_float4(kv4_value(w, 0, s), kv4_value(w, 1, s), kv4_value(w, 2, s), kv4_value(w, 3, s));
    };
#pragma unroll
    for (int u = 0; u < READ4_ROWS; ++u) {
        if (r0 + u >= rows) break;
        reinterpret_cast<float4 *>(k)[(r0 + u) * per_row + j] = four(kw[u], ks[u]);
        reinterpret_cast<float4 *>(v)[(r0 + u) * per_row + j] = four(vw[u], vs[u]);
    }
}

template <typename T> static void append_launch(const Kv4Append &A, unsigned grid, cudaStream_t s)
{
    const bool q = A.q_rows > 0;
    if (A.c.head_dim == 128) {
        if (q) kv4_append_kernel<T, 128, true><<<grid, KV4_THREADS, 0, s>>>(A);
        else kv4_append_kernel<T, 128, false><<<grid, KV4_THREADS, 0, s>>>(A);
    } else {
        if (q) kv4_append_kernel<T, 64, true><<<grid, KV4_THREADS, 0, s>>>(A);
        else kv4_append_kernel<T, 64, false><<<grid, KV4_THREADS, 0, s>>>(A);
    }
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
    if (!slots || (rope && !positions) || off_element(width, k, v) || (heads && off_element(width, q, q_out))) return -1;
    A.c = *cache;
    A.slots = slots; A.positions = positions;
    A.k = k; A.v = v; A.k_stride = k_stride; A.v_stride = v_stride; A.rows = rows;
    A.q = RopeRows{q, q_out, q_stride, q_out_stride, heads};
    A.shift = kv4_shift(cache);
    A.error = error;
    // 16-byte accesses to rows and tables: the values of a thread rotate alike, their tables' rows are aligned
    A.vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && k_stride % el == 0 && v_stride % el == 0;
    if (rope) A.vec = A.vec && rope_vectors(A.rope, hd, width, A.q) && A.rope.dims % (A.rope.layout == 0 ? KV4_EACH : 2 * KV4_EACH) == 0 &&
                    ((uintptr_t)A.rope.cos | (uintptr_t)A.rope.sin) % 16 == 0;
    cudaStream_t s = (cudaStream_t)stream;
    A.grid = kv4_grid(2 * kv * (hd / KV4_EACH));
    const size_t ctas = (rows + A.grid.rows - 1) / A.grid.rows * A.grid.parts;
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
    const dim3 grid((unsigned)((rows + READ4_ROWS - 1) / READ4_ROWS), (cache->kv_heads * (cache->head_dim / 4) + KV4_THREADS - 1) / KV4_THREADS);
    if (grid.y > 65535) return -1;
    cudaStream_t s = (cudaStream_t)stream;
    if (cache->head_dim == 128) kv4_read_kernel<128><<<grid, KV4_THREADS, 0, s>>>(*cache, slots, rows, k, v, kv4_shift(cache), error);
    else kv4_read_kernel<64><<<grid, KV4_THREADS, 0, s>>>(*cache, slots, rows, k, v, kv4_shift(cache), error);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
