// kv8.cu - rows into and out of the paged 8-bit KV cache.
//
// Append: a block's scale is s' = max(s, max|x| (1 / top)) over the values it
// was ever given (top 127 or 448, its reciprocal rounded to F32); a new value
// is stored as round(x / s'), and where s' > s the block's older tokens are
// stored anew as round(q (s / s')). Every product and quotient is the IEEE one
// in F32, so the stored bytes are defined to the bit. By its bytes (rows in, a
// byte a value out) bound by memory; what it takes for prompts is latency, a
// run's rows being looked at twice (4534 bf16 rows of 8 heads, K rotated: 26 us,
// 4.3 us of bytes; issue slots 0.40 used, 5.4 of 13 cycles an instruction spent on loads).
//
// The rows of one block are neighbours in the slot list, but for rows that are
// left out, so the first of them (the row whose predecessor lies in another
// block) speaks for the block: one CTA takes its whole run for one KV head of K
// or of V, and no two CTAs touch the same block of a head. A K row left out for
// its position still belongs to its block's run; a row without a slot belongs to
// none and ends none.
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
    RopeRows q;       // rotated in the same launch where rows are few (heads 0: none)
    RopeWork work;
    unsigned shift, window, parts, q_rows;  // parts: CTAs of a window; q_rows: CTAs of a row of q
    bool vec, many;
    unsigned *error;
};

// E consecutive values of one head's row as they lie there; and as they are stored, rotated when `turn` (half pairs
// fetch the other half, which the same CTA has in its cache).
template <typename T, int E> FYB_DEV RopePack<T, E> kv8_get(const Kv8Append &A, const T *p)
{
    return A.vec ? rope_get<T, E, true>(p) : rope_get<T, E, false>(p);
}
template <typename T, int E> FYB_DEV void kv8_values(const Kv8Append &A, const RopePack<T, E> &own, const T *row, unsigned e,
    bool turn, size_t tab, float (&x)[E])
{
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = row_value(own.t[i]);
    if (!turn || e >= A.rope.dims) return;
    const float *c = A.rope.cos + tab, *s = A.rope.sin + tab;
    if (A.rope.layout == 0) {
        if (E == 4 && A.vec && e + 4 <= A.rope.dims) {
            const float2 cv = *reinterpret_cast<const float2 *>(c + e / 2), sv = *reinterpret_cast<const float2 *>(s + e / 2);
            rope_turn(x[0], x[1], cv.x, sv.x);
            rope_turn(x[E - 2], x[E - 1], cv.y, sv.y);
            return;
        }
#pragma unroll
        for (int i = 0; i < E; i += 2)
            if (e + i < A.rope.dims) rope_turn(x[i], x[i + 1], c[(e + i) / 2], s[(e + i) / 2]);
    } else {
        const unsigned pairs = A.rope.dims / 2;
        const bool low = e < pairs;  // dims / 2 is a multiple of E: a run lies in one half
        const unsigned p = low ? e : e - pairs;
        const RopePack<T, E> y = kv8_get<T, E>(A, row + (low ? e + pairs : e - pairs));
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float o = row_value(y.t[i]);
            if (low) rope_turn(x[i], o, c[p + i], s[p + i]); else rope_turn(o, x[i], c[p + i], s[p + i]);
        }
    }
}

// q rows: CTA = 256 items of one row
template <typename T, int HD> FYB_DEV void kv8_turn_q(const Kv8Append &A, unsigned cta)
{
    const size_t r = cta / A.q_rows;
    const unsigned i = cta % A.q_rows * KV8_THREADS + threadIdx.x;
    const unsigned groups = A.many ? (A.q.heads + ROPE_HEADS - 1) / ROPE_HEADS : A.q.heads;
    unsigned head, item;  // heads head, head + groups, ...
    if (!rope_place(A.work, groups, i, head, item)) return;
    const int pos = A.positions[r];
    const T *in = static_cast<const T *>(A.q.in) + r * A.q.in_stride + (size_t)head * HD;
    T *out = static_cast<T *>(A.q.out) + r * A.q.out_stride + (size_t)head * HD;
    auto at = [&](const float *&c, const float *&s) {
        if (pos < 0 || (unsigned)pos >= A.rope.rows) {
            if (i == 0) raise_error(A.error, ERR_BOUNDS);
            return false;
        }
        const size_t t = (size_t)pos * (A.rope.dims / 2);
        c = A.rope.cos + t;
        s = A.rope.sin + t;
        return true;
    };
    constexpr int V = 16 / sizeof(T);
    if (A.many)
        rope_item<T, V, true, ROPE_HEADS>(in, out, (size_t)groups * HD, (A.q.heads - head + groups - 1) / groups,
                                          A.rope.dims, A.rope.layout, item, at);
    else if (A.vec) rope_item<T, V, true, 1>(in, out, HD, 1, A.rope.dims, A.rope.layout, item, at);
    else if (A.rope.layout == 0) rope_item<T, 2, false, 1>(in, out, HD, 1, A.rope.dims, 0, item, at);
    else rope_item<T, 1, false, 1>(in, out, HD, 1, A.rope.dims, 1, item, at);
}

// Four stored bytes of values already divided by the scale.
template <unsigned FMT> FYB_DEV unsigned kv8_store4(float a, float b, float c, float d)
{
    if constexpr (FMT == FYB_KV8_INT8) {
        return kv8_store<FMT>(a) | kv8_store<FMT>(b) << 8 | kv8_store<FMT>(c) << 16 | kv8_store<FMT>(d) << 24;
    } else {
        const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        return lo | (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
    }
}

// round(y / now) of four finite values, as the IEEE quotient rounds. The product with the reciprocal is within 2^-22 of
// the quotient, relatively: where rounding it leaves no doubt the quotient rounds alike, and the division, ten times the
// instructions, is left to the others (one value in some thousands).
template <unsigned FMT> FYB_DEV unsigned kv8_quotients(const float (&y)[4], float now, float inv)
{
    float r[4];
    bool sure = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = __fmul_rn(y[e], inv);
    if constexpr (FMT == FYB_KV8_INT8) {
        unsigned q[4];  // the whole number in the low bits of r + 1.5 x 2^23
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float sum = __fadd_rn(r[e], 12582912.f);
            sure = sure && fabsf(r[e] - __fsub_rn(sum, 12582912.f)) < 0.4999f;  // |r| <= 128: off by 4e-5 at the most; false for NaN
            q[e] = __float_as_uint(sum);
        }
        if (sure) {  // -127..127 by the choice of the scale, but for roundings that `sure` leaves out
            const unsigned lo = __byte_perm(q[0], q[1], 0x0040), hi = __byte_perm(q[2], q[3], 0x0040);
            return __byte_perm(lo, hi, 0x5410);
        }
    } else {
        const float up = 1.f + 0x1p-20f, down = 1.f - 0x1p-20f;
        const unsigned a = kv8_store4<FMT>(r[0] * up, r[1] * up, r[2] * up, r[3] * up);
        const unsigned b = kv8_store4<FMT>(r[0] * down, r[1] * down, r[2] * down, r[3] * down);
        sure = a == b && inv <= 3.4028235e38f;
        if (sure) return a;
    }
    return kv8_store4<FMT>(__fdiv_rn(y[0], now), __fdiv_rn(y[1], now), __fdiv_rn(y[2], now), __fdiv_rn(y[3], now));
}

// CTAs: (window of rows, part), part = one KV head of K or of V; then those of q.
template <typename T, int HD, unsigned FMT>
__global__ void __launch_bounds__(KV8_THREADS, 4) kv8_append_kernel(Kv8Append A)
{
    // A warp's rows of a run: the first HOLD stay in registers between the two passes, others are fetched again (from
    // L1 and L2). 4534 rows of 8 KV heads, not rotated: held 1, 2, 4, 8 took 25, 21, 23, 33 us (8 no longer fit the
    // registers). The loops fetch one row at a time: two or three, unrolled, took 24 and 25 us, out of the instruction
    // cache.
    constexpr unsigned THREADS = KV8_THREADS;
    constexpr int E = HD / 32, WARPS = THREADS / 32, HOLD = 2;
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kv = A.c.kv_heads;
    const unsigned windows = (unsigned)((A.rows + A.window - 1) / A.window);
    if (blockIdx.x >= windows * A.parts) {
        kv8_turn_q<T, HD>(A, blockIdx.x - windows * A.parts);
        return;
    }
    const unsigned part = blockIdx.x % A.parts;
    const size_t row0 = (size_t)(blockIdx.x / A.parts) * A.window;
    __shared__ unsigned run_s, last_s, first_s, peak_s, bad_s, leaders_s[THREADS / 32];
    // slots (-1: none) and positions (-1: not stored) of the window and of a block's rows before and after it
    __shared__ int slot_s[255 + 256 + 256], pos_s[255 + 256 + 256];
    const bool is_k = part < kv, turn = is_k && A.rope.cos;
    const unsigned head = is_k ? part : part - kv, size = 1u << A.shift, back = size - 1;
    const T *src = static_cast<const T *>(is_k ? A.k : A.v) + (size_t)head * HD;
    const size_t stride = is_k ? A.k_stride : A.v_stride;
    unsigned char *pool = static_cast<unsigned char *>(is_k ? A.c.k : A.c.v);
    float *scales = is_k ? A.c.k_scale : A.c.v_scale;
    const int limit = (int)(A.c.blocks << A.shift);
    for (unsigned j = tid; j < back + A.window + size; j += THREADS) {
        const size_t r = row0 + j - back;  // past the end where there is no row before
        int slot = -1, pos = -1;
        if (r < A.rows) {
            slot = A.slots[r];
            pos = turn ? A.positions[r] : 0;
            if (slot < 0) {
                slot = pos = -1;
            } else if (slot >= limit) {
                slot = pos = -1;
                raise_error(A.error, ERR_BOUNDS);
            } else if (turn && (unsigned)pos >= A.rope.rows) {
                pos = -1;
                raise_error(A.error, ERR_BOUNDS);
            }
        }
        slot_s[j] = slot;
        pos_s[j] = pos;
    }
    __syncthreads();
    // the block of the window's row i (negative: a row before it), or -1 for a row without a slot
    auto block_of = [&](int i) { return slot_s[(int)back + i] >> A.shift; };
    // ---- the rows of the window that begin a run
    {
        bool leads = tid < A.window && block_of((int)tid) >= 0;
        if (leads) {
            int i = (int)tid - 1;
            while (i > (int)tid - (int)back && block_of(i) < 0) --i;
            leads = block_of(i) != block_of((int)tid);
        }
        const unsigned mask = __ballot_sync(0xffffffffu, leads);
        if (lane == 0) leaders_s[warp] = mask;
        __syncthreads();
    }
    for (unsigned w = 0; w < (A.window + 31) / 32; ++w)
    for (unsigned left = leaders_s[w]; left; left &= left - 1) {
        const unsigned i0 = 32 * w + (unsigned)__ffs((int)left) - 1;
        const size_t r0 = row0 + i0;
        const int b = block_of((int)i0);
        auto stored = [&](unsigned i) { return pos_s[back + i0 + i] >= 0; };
        // ---- the run of rows in block b: up to another block's, and to the last that is stored; its lowest offset
        if (tid == 0) { run_s = size; last_s = 0u; first_s = size; peak_s = 0u; bad_s = 0u; }
        __syncthreads();
        const int own = tid < size ? block_of((int)(i0 + tid)) : -1;
        const unsigned others = __ballot_sync(0xffffffffu, own >= 0 && own != b);
        const unsigned kept = __ballot_sync(0xffffffffu, own == b && stored(tid));
        if (lane == 0) {
            if (others) atomicMin(&run_s, 32 * warp + (unsigned)__ffs((int)others) - 1);
            if (kept) atomicMax(&last_s, 32 * warp + 32 - (unsigned)__clz((int)kept));
        }
        __syncthreads();
        const unsigned run = min(run_s, last_s);
        // the rows of it that this warp takes, warp + WARPS h for every bit h
        static_assert(WARPS * 32 >= 256, "the longest run");
        const unsigned mine = __ballot_sync(0xffffffffu, warp + WARPS * lane < run && stored(warp + WARPS * lane));
        if (own == b && tid < run_s) atomicMin(&first_s, (unsigned)slot_s[back + i0 + tid] & (size - 1));
        if (!run) {  // none of them is stored: the block stays as it is
            __syncthreads();
            continue;
        }
        const size_t at = (size_t)b * kv + head;
        const float before = scales[at];  // asked for early; counts only if the block holds older tokens
        // ---- largest magnitude
        float held[HOLD][E];
        float peak = 0.f;
        bool bad = false;
        auto row_at = [&](unsigned i) { return src + (r0 + i) * stride; };
        auto value = [&](unsigned i, const RopePack<T, E> &own, float (&y)[E]) {
            const size_t tab = turn ? (size_t)pos_s[back + i0 + i] * (A.rope.dims / 2) : 0;
            kv8_values<T, E>(A, own, row_at(i), lane * E, turn, tab, y);
        };
        auto look = [&](const float (&y)[E]) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float m = fabsf(y[e]);
                if (m <= 3.4028235e38f) peak = fmaxf(peak, m); else bad = true;
            }
        };
        {
            RopePack<T, E> raw[HOLD];
#pragma unroll
            for (int h = 0; h < HOLD; ++h)
                if (mine >> h & 1) raw[h] = kv8_get<T, E>(A, row_at(warp + h * WARPS) + lane * E);
#pragma unroll
            for (int h = 0; h < HOLD; ++h)
                if (mine >> h & 1) {
                    value(warp + h * WARPS, raw[h], held[h]);
                    look(held[h]);
                }
        }
        for (unsigned i = warp + HOLD * WARPS, more = mine >> HOLD; more; i += WARPS, more >>= 1) {
            if (!(more & 1)) continue;
            float y[E];
            value(i, kv8_get<T, E>(A, row_at(i) + lane * E), y);
            look(y);
        }
        if (bad) {
            raise_error(A.error, ERR_NONFINITE);
            bad_s = 1;
        }
        peak = warp_max(peak);
        if (lane == 0) atomicMax(&peak_s, __float_as_uint(peak));  // non-negative: ordered as integers
        __syncthreads();
        const unsigned first = first_s;
        const float was = first ? before : 0.f;
        const float now = fmaxf(was, kv8_scale(FMT, __uint_as_float(peak_s)));
        unsigned char *blk = pool + at * size * HD;
        if (now > was && first) {
            const float keep = __fdiv_rn(was, now);
            unsigned *words = reinterpret_cast<unsigned *>(blk);
            for (unsigned i = tid; i < first * HD / 4; i += THREADS) {
                const unsigned old = words[i];
                words[i] = kv8_store4<FMT>(__fmul_rn(kv8_number<FMT>(old & 0xffu), keep), __fmul_rn(kv8_number<FMT>(old >> 8 & 0xffu), keep),
                                           __fmul_rn(kv8_number<FMT>(old >> 16 & 0xffu), keep), __fmul_rn(kv8_number<FMT>(old >> 24), keep));
            }
        }
        // ---- stored values
        const bool plain = now > 0.f && !bad_s;
        const float inv = __frcp_rn(now);
        auto store = [&](unsigned i, const float (&y)[E]) {
            float q[4] = {0.f, 0.f, 0.f, 0.f};
            unsigned bytes;
            if (plain) {
#pragma unroll
                for (int e = 0; e < E; ++e) q[e] = y[e];
                bytes = kv8_quotients<FMT>(q, now, inv);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    q[e] = now > 0.f ? __fdiv_rn(y[e], now) : 0.f;
                    if (!(fabsf(y[e]) <= 3.4028235e38f)) q[e] = isnan(y[e]) ? 0.f : copysignf(kv8_top(FMT), y[e]);
                }
                bytes = kv8_store4<FMT>(q[0], q[1], q[2], q[3]);
            }
            unsigned char *dst = blk + ((unsigned)slot_s[back + i0 + i] & (size - 1)) * HD + lane * E;
            if constexpr (E == 4) *reinterpret_cast<unsigned *>(dst) = bytes;
            else *reinterpret_cast<unsigned short *>(dst) = (unsigned short)bytes;
        };
#pragma unroll
        for (int h = 0; h < HOLD; ++h)
            if (mine >> h & 1) store(warp + h * WARPS, held[h]);
        for (unsigned i = warp + HOLD * WARPS, more = mine >> HOLD; more; i += WARPS, more >>= 1) {
            if (!(more & 1)) continue;
            float y[E];
            value(i, kv8_get<T, E>(A, row_at(i) + lane * E), y);
            store(i, y);
        }
        __syncthreads();
        if (tid == 0) scales[at] = now;
    }
}

// Values at slots: thread = word j (four values) of K and of V of READ_ROWS rows, all loads out before the first is
// used. Grid (rows / READ_ROWS, words of a row / 256).
constexpr int READ_ROWS = 4;
template <unsigned FMT>
__global__ void __launch_bounds__(256) kv8_read_kernel(fyb_kv8_cache c, const int *slots, size_t rows, float *k, float *v,
    unsigned shift, unsigned *error)
{
    const unsigned per_head = c.head_dim / 4, per_row = c.kv_heads * per_head;
    const unsigned j = blockIdx.y * 256 + threadIdx.x, head = j / per_head, e = j % per_head;
    if (j >= per_row) return;
    const size_t r0 = (size_t)blockIdx.x * READ_ROWS;
    int slot[READ_ROWS];
    unsigned kw[READ_ROWS], vw[READ_ROWS];
    float ks[READ_ROWS], vs[READ_ROWS];
#pragma unroll
    for (int u = 0; u < READ_ROWS; ++u) slot[u] = r0 + u < rows ? slots[r0 + u] : -1;
#pragma unroll
    for (int u = 0; u < READ_ROWS; ++u) {
        kw[u] = vw[u] = 0;
        ks[u] = vs[u] = 0.f;
        if (slot[u] < 0) continue;
        if (slot[u] >= (int)(c.blocks << shift)) { raise_error(error, ERR_BOUNDS); continue; }
        const size_t at = (size_t)(slot[u] >> shift) * c.kv_heads + head;
        const size_t off = ((at << shift) + ((unsigned)slot[u] & ((1u << shift) - 1))) * per_head + e;
        kw[u] = static_cast<const unsigned *>(c.k)[off];
        vw[u] = static_cast<const unsigned *>(c.v)[off];
        ks[u] = c.k_scale[at];
        vs[u] = c.v_scale[at];
    }
    auto four = [](unsigned w, float s) {
        return make_float4(kv8_number<FMT>(w & 0xffu) * s, kv8_number<FMT>((w >> 8) & 0xffu) * s,
                           kv8_number<FMT>((w >> 16) & 0xffu) * s, kv8_number<FMT>(w >> 24) * s);
    };
#pragma unroll
    for (int u = 0; u < READ_ROWS; ++u) {
        if (r0 + u >= rows) break;
        reinterpret_cast<float4 *>(k)[(r0 + u) * per_row + j] = four(kw[u], ks[u]);
        reinterpret_cast<float4 *>(v)[(r0 + u) * per_row + j] = four(vw[u], vs[u]);
    }
}

template <typename T> static void append_launch(const Kv8Append &A, unsigned grid, cudaStream_t s)
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
    if ((rows && (!k || !v)) || k_stride < (size_t)kv * hd || v_stride < (size_t)kv * hd || (heads && !rope) || heads > 65536)
        return -1;
    if (rope && (rope_table_of(rope, &A.rope) || A.rope.dims > hd || (A.rope.layout != 0 && A.rope.dims % 8)))
        return -1;
    if (heads && ((rows && (!q || !q_out)) || q_stride < (size_t)heads * hd || q_out_stride < (size_t)heads * hd ||
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
    // K's interleaved pairs take two cosines and two sines in an access, q or no q: even table rows, on 8 bytes
    if (rope && A.rope.layout == 0)
        A.vec = A.vec && A.rope.dims % 4 == 0 && ((uintptr_t)A.rope.cos | (uintptr_t)A.rope.sin) % 8 == 0;
    // a CTA looks at one row while that makes at most 16 CTAs per SM; beyond,
    // at the rows of up to a block (a prompt's mostly follow one another), 8
    // CTAs per SM: what a CTA does once is then spread over its rows (4534 rows
    // of 8 heads, not rotated: 16 take 26 us where 8 take 21)
    A.window = 1;
    A.parts = 2 * kv;
    while (A.window < cache->block_size && rows / A.window * A.parts > (A.window == 1 ? 16 : 8) * 148) A.window *= 2;
    cudaStream_t s = (cudaStream_t)stream;
    A.q_rows = 0;
    if (heads && A.window > 1) {  // a launch more is little beside a prompt
        const int r = rope_run(type, A.rope, positions, rows, hd, A.q, RopeRows{}, error, s);
        if (r) return r;
    } else if (heads) {
        A.work = rope_work(hd, A.rope.dims, A.rope.layout, A.vec ? (unsigned)el : A.rope.layout == 0 ? 2u : 1u, q == q_out);
        A.many = A.vec && rope_many(rows, heads, A.work);
        const unsigned groups = A.many ? (heads + ROPE_HEADS - 1) / ROPE_HEADS : heads;
        A.q_rows = (unsigned)(((size_t)groups * (A.work.turned + A.work.copied) + KV8_THREADS - 1) / KV8_THREADS);
    }
    const size_t ctas = (rows + A.window - 1) / A.window * A.parts + rows * A.q_rows;
    if (ctas > 0x7fffffffu) return -1;
    const unsigned grid = (unsigned)ctas;
    if (type == T_F32) append_launch<float>(A, grid, s);
    else if (type == T_F16) append_launch<__half>(A, grid, s);
    else append_launch<__nv_bfloat16>(A, grid, s);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int fyb_kv8_read(const fyb_kv8_cache *cache, const int32_t *slots, size_t rows, float *k, float *v,
    uint32_t *error, void *stream)
{
    if (kv8_check(cache) || (rows && (!k || !v)) || ((uintptr_t)k | (uintptr_t)v) % 16 || rows > 0x7fffffffu) return -1;
    if (!rows) return 0;
    if (!slots) return -1;
    const unsigned words = cache->kv_heads * (cache->head_dim / 4);
    const dim3 grid((unsigned)((rows + READ_ROWS - 1) / READ_ROWS), (words + 255) / 256);
    if (grid.y > 65535) return -1;
    if (cache->format == FYB_KV8_INT8)
        kv8_read_kernel<FYB_KV8_INT8><<<grid, 256, 0, (cudaStream_t)stream>>>(*cache, slots, rows, k, v, kv8_shift(cache), error);
    else
        kv8_read_kernel<FYB_KV8_E4M3><<<grid, 256, 0, (cudaStream_t)stream>>>(*cache, slots, rows, k, v, kv8_shift(cache), error);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
