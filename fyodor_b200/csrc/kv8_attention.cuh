// kv8_attention.cuh - how the attention over the paged 8-bit cache is split
// over the GPU, shared by its two kernels (kv8_decode.cu: few query rows
// per KV head, kv8_tiles.cuh: many).
//
// Work is a line of units. A segment is the cache that one row tile of one
// request attends in one KV head, a unit TILE positions of it. CTA c of C takes
// units [U c / C, U (c + 1) / C): every CTA streams the same number of tiles
// whatever the lengths, its loads running on from one segment to the next. A
// segment that crosses CTAs leaves one partial (maximum, sum, weighted values)
// per CTA; the last CTA to finish its part joins them in CTA order, so results
// do not depend on timing and no CTA waits for another.
#pragma once
#include "kv8.cuh"
#include <cuda.h>

namespace fyb {

struct Kv8Attention {
    fyb_kv8_cache c;
    const int *lengths, *row_start, *table;
    size_t table_stride, q_stride, out_stride;
    const void *q;
    void *out;
    unsigned rows, requests, max_rows, heads, group, shift, type;
    unsigned row_tile;    // query tokens of one row tile
    float scale;          // score factor x log2(e)
    unsigned *counters;   // [grid] arrivals at the segment that begins in CTA c and ends beyond it; zero between calls
    float2 *part_ml;      // [2 grid][rows of a tile] (maximum, sum)
    float *part_o;        // [2 grid][rows of a tile][head_dim]
    unsigned *error;
};

// Largest grid of either kernel, three CTAs per SM; the workspace is sized for it.
constexpr unsigned KA_GRID = 3 * 148;
constexpr size_t KA_COUNTER_BYTES = (KA_GRID * 4 + 255) / 256 * 256;

// ---- segments and units ------------------------------------------------------
struct Kv8Request {
    int len, n, first, rows;  // cached tokens, rows it brings, its first row, rows computed of them
};
FYB_DEV Kv8Request kv8_request(const Kv8Attention &A, unsigned r, bool complain)
{
    Kv8Request q;
    q.first = A.row_start ? max(0, min(A.row_start[r], (int)A.rows)) : (int)r;
    q.n = A.row_start ? max(0, min(A.row_start[r + 1], (int)A.rows) - q.first) : 1;
    q.rows = min(q.n, (int)A.max_rows);
    q.len = max(0, A.lengths[r]);
    bool bad = q.rows < q.n;
    if ((unsigned long long)q.len > (unsigned long long)A.table_stride << A.shift) { q.len = 0; bad = true; }
    if (bad && complain) raise_error(A.error, ERR_BOUNDS);
    return q;
}
// Positions attended by any row of row tile i, and its units per KV head
// (one at least: rows that attend nothing are written too).
FYB_DEV int kv8_attended(const Kv8Attention &A, const Kv8Request &q, int i)
{
    return max(0, q.len - q.n + min(q.rows, (i + 1) * (int)A.row_tile));
}
template <int TILE> FYB_DEV int kv8_tiles(const Kv8Attention &A, const Kv8Request &q, int i)
{
    return max(1, (kv8_attended(A, q, i) + TILE - 1) / TILE);
}
FYB_DEV int kv8_row_tiles(const Kv8Attention &A, const Kv8Request &q)
{
    return (q.rows + (int)A.row_tile - 1) / (int)A.row_tile;
}
template <int TILE> FYB_DEV unsigned kv8_units(const Kv8Attention &A, const Kv8Request &q)
{
    unsigned u = 0;
    for (int i = 0; i < kv8_row_tiles(A, q); ++i) u += (unsigned)kv8_tiles<TILE>(A, q, i);
    return u * A.c.kv_heads;
}
// CTAs that take part, and where their ranges begin. Few units go to fewer
// CTAs, LEAST each: a tile more takes a CTA 0.35 us, joining parts 3 us.
template <int LEAST> FYB_DEV unsigned kv8_ctas(unsigned U) { return min(gridDim.x, max(1u, U / LEAST)); }
FYB_DEV unsigned kv8_cta_begin(unsigned U, unsigned C, unsigned c)
{
    return c >= C ? U : (unsigned)((unsigned long long)U * c / C);
}
// The CTA whose range holds unit u.
FYB_DEV unsigned kv8_cta_of(unsigned U, unsigned C, unsigned u)
{
    return (unsigned)((((unsigned long long)u + 1) * C - 1) / U);
}

// Longest segment that goes whole to a CTA. Many rows: 4 requests of 500 to 800
// with eight rows of four heads take 31 us on the line's ranges and 21 so, one
// of 1000 with 100 rows 46 and 33; one of 1200 with eight rows, 21.6 and 24.3,
// is beyond it.
constexpr unsigned KA_WHOLE = 8;

// Where a CTA stands on the line of units.
struct Kv8Place {
    unsigned units, ctas, begin, end;  // all units and the CTAs that share them; this CTA's
    unsigned request, before;       // request of `begin`, units before it
};
// Every thread of the CTA (THREADS of them) calls this once. Where no segment is
// longer than KA_WHOLE units and every segment can have a CTA, each gets one: no
// parts to join, and a request's result does not depend on the others (16
// requests of 20 to 60 tokens: 17.6 us on the line's ranges, 6.2 so; one of 300
// with eight rows of four heads: 28.8 and 17.3).
template <int TILE, int THREADS, int LEAST> FYB_DEV Kv8Place kv8_place(const Kv8Attention &A)
{
    __shared__ uint2 warp_sum[THREADS / 32];
    __shared__ unsigned found[4], longest;
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kv = A.c.kv_heads;
    const unsigned per = (A.requests + THREADS - 1) / THREADS, r0 = min(tid * per, A.requests),
                   r1 = min(r0 + per, A.requests);
    unsigned units = 0, segments = 0, most = 0;
    for (unsigned r = r0; r < r1; ++r) {
        const Kv8Request q = kv8_request(A, r, blockIdx.x == 0);
        const int tiles = kv8_row_tiles(A, q);
        units += kv8_units<TILE>(A, q);
        segments += (unsigned)tiles * kv;
        if (tiles) most = max(most, (unsigned)kv8_tiles<TILE>(A, q, tiles - 1));  // the last row tile attends most
    }
    uint2 upto = make_uint2(units, segments);
#pragma unroll
    for (unsigned o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, upto.x, o), y = __shfl_up_sync(0xffffffffu, upto.y, o);
        if (lane >= o) { upto.x += x; upto.y += y; }
    }
    if (lane == 31) warp_sum[warp] = upto;
    if (tid < 4) found[tid] = 0;
    if (tid == 0) longest = 0;
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) atomicMax(&longest, most);
    unsigned before = upto.x - units, segments_before = upto.y - segments, total = 0, all = 0;
    for (unsigned w = 0; w < THREADS / 32; ++w) {
        if (w < warp) { before += warp_sum[w].x; segments_before += warp_sum[w].y; }
        total += warp_sum[w].x;
        all += warp_sum[w].y;
    }
    __syncthreads();
    Kv8Place p;
    p.units = total;
    const bool whole = longest <= KA_WHOLE && all <= gridDim.x;  // a segment for each CTA
    p.ctas = whole ? all : kv8_ctas<LEAST>(total);
    p.begin = kv8_cta_begin(total, p.ctas, blockIdx.x);
    p.end = kv8_cta_begin(total, p.ctas, blockIdx.x + 1);
    if (whole ? segments && segments_before <= blockIdx.x && blockIdx.x < segments_before + segments
              : units && before <= p.begin && p.begin < before + units) {
        unsigned r = r0, at = before, seg = segments_before;
        for (;; ++r) {
            const Kv8Request q = kv8_request(A, r, false);
            const unsigned u = kv8_units<TILE>(A, q), n = (unsigned)kv8_row_tiles(A, q) * kv;
            if (whole ? blockIdx.x < seg + n : p.begin < at + u) break;
            at += u;
            seg += n;
        }
        found[0] = r;
        found[1] = at;
        if (whole) {
            // segment blockIdx.x - seg of the request: its units
            const Kv8Request q = kv8_request(A, r, false);
            unsigned left = blockIdx.x - seg, u = at;
            int i = 0;
            for (; left >= kv; ++i, left -= kv) u += (unsigned)kv8_tiles<TILE>(A, q, i) * kv;
            const unsigned tiles = (unsigned)kv8_tiles<TILE>(A, q, i);
            found[2] = u + left * tiles;
            found[3] = u + (left + 1) * tiles;
        }
    }
    __syncthreads();
    p.request = found[0];
    p.before = found[1];
    if (whole) {
        p.begin = found[2];
        p.end = found[3];
    }
    return p;
}

// A CTA's part of a segment: units [t0, t1) of its `tiles`.
struct Kv8Segment {
    Kv8Request q;
    unsigned request, head;
    int row_tile, t0, t1, tiles;
    unsigned first_unit;   // line unit of tile 0
};
// Walks a CTA's segments in order.
template <int TILE> struct Kv8Walk {
    const Kv8Attention &A;
    unsigned at, end, r, before;
    int i, tiles_i;
    Kv8Request q;
    unsigned i_before;     // units of the request before row tile i
    FYB_DEV Kv8Walk(const Kv8Attention &a, const Kv8Place &p) : A(a), at(p.begin), end(p.end), r(p.request), before(p.before)
    {
        if (at < end) open();
    }
    FYB_DEV void open()
    {
        q = kv8_request(A, r, false);
        i = 0;
        i_before = 0;
        tiles_i = kv8_row_tiles(A, q) ? kv8_tiles<TILE>(A, q, 0) : 0;
    }
    FYB_DEV bool next(Kv8Segment &s)
    {
        if (at >= end) return false;
        for (;;) {
            const unsigned size = (unsigned)tiles_i * A.c.kv_heads;
            if (at < before + i_before + size) break;
            i_before += size;
            if (i + 1 < kv8_row_tiles(A, q)) {
                tiles_i = kv8_tiles<TILE>(A, q, ++i);
            } else {
                before += i_before;
                if (++r >= A.requests) { at = end; return false; }
                open();
            }
        }
        const unsigned x = at - before - i_before;
        s.q = q;
        s.request = r;
        s.row_tile = i;
        s.tiles = tiles_i;
        s.head = x / (unsigned)tiles_i;
        s.t0 = (int)(x % (unsigned)tiles_i);
        s.t1 = min(tiles_i, s.t0 + (int)(end - at));
        s.first_unit = at - (unsigned)s.t0;
        at += (unsigned)(s.t1 - s.t0);
        return true;
    }
};

// Maximum and sum over groups of G lanes; every lane of the warp takes part.
template <int G> FYB_DEV float group_max(float x)
{
#pragma unroll
    for (int o = G / 2; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
template <int G> FYB_DEV float group_sum(float x)
{
#pragma unroll
    for (int o = G / 2; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// ---- joining the parts of a segment -------------------------------------------
// `threads` threads hold the segment's part as ml[R] and o[R][HD] in shared
// memory; bar(): a barrier over them. Writes the rows out when the CTA has the
// whole segment; otherwise leaves a partial, and the last CTA to do so joins
// all parts. valid(row, &src): whether row is a query row, and which.
template <int R, int HD, int THREADS, typename Bar, typename Put>
FYB_DEV void kv8_finish(const Kv8Attention &A, const Kv8Segment &s, const Kv8Place &place, unsigned tid, const float2 *ml,
    const float *o, unsigned rows, float *weights, unsigned max_weights, unsigned *flag, Bar bar, Put put)
{
    if (s.t0 == 0 && s.t1 == s.tiles) {
        for (unsigned i = tid; i < rows * (HD / 4); i += THREADS) {
            const unsigned row = i / (HD / 4);
            float4 v = reinterpret_cast<const float4 *>(o)[i];
            const float l = ml[row].y, n = l > 0.f || isnan(l) ? 1.f / l : 0.f;
            v.x *= n; v.y *= n; v.z *= n; v.w *= n;
            put(row, i % (HD / 4), v);
        }
        return;
    }
    const unsigned c0 = kv8_cta_of(place.units, place.ctas, s.first_unit);
    const unsigned c1 = kv8_cta_of(place.units, place.ctas, s.first_unit + (unsigned)s.tiles - 1);
    // the segment that ends a CTA's range goes to its second slot, any other to its first
    const unsigned slot = 2 * blockIdx.x + (blockIdx.x == c0 ? 1 : 0);
    for (unsigned i = tid; i < rows * (HD / 4); i += THREADS)
        reinterpret_cast<float4 *>(A.part_o + (size_t)slot * R * HD)[i] = reinterpret_cast<const float4 *>(o)[i];
    for (unsigned i = tid; i < rows; i += THREADS) A.part_ml[(size_t)slot * R + i] = ml[i];
    __threadfence();
    bar();
    if (tid == 0) *flag = atomicAdd(&A.counters[c0], 1u) == c1 - c0;
    bar();
    if (!*flag) return;
    __threadfence();
    if (tid == 0) A.counters[c0] = 0;
    const unsigned parts = c1 - c0 + 1;
    auto slot_of = [&](unsigned p) { return (size_t)(2 * (c0 + p) + (p == 0 ? 1 : 0)); };
    // weights of the parts: 2^(m - max m) / sum, as many rows at a time as fit,
    // the threads shared out among the rows: it is L2's latency that takes time
    constexpr unsigned G = THREADS / R < 32 ? THREADS / R : 32;
    static_assert(G > 0 && (G & (G - 1)) == 0 && THREADS / G >= R, "");
    const unsigned batch = max(1u, min(rows, max_weights / parts));
    for (unsigned row0 = 0; row0 < rows; row0 += batch) {
        const unsigned some = min(batch, rows - row0);
        bar();
        const unsigned i = tid / G, lane = tid % G;
        float m = -INFINITY, l = 0.f;
        if (i < some)
            for (unsigned p = lane; p < parts; p += G) m = fmaxf(m, __ldcg(&A.part_ml[slot_of(p) * R + row0 + i].x));
        m = group_max<G>(m);
        if (i < some)
            for (unsigned p = lane; p < parts; p += G) {
                const float2 x = __ldcg(&A.part_ml[slot_of(p) * R + row0 + i]);
                const float w = exp2f(x.x - m);
                weights[p * some + i] = w;
                l += x.y * w;
            }
        l = group_sum<G>(l);
        const float n = l > 0.f || isnan(l) ? 1.f / l : 0.f;
        if (i < some)
            for (unsigned p = lane; p < parts; p += G) weights[p * some + i] *= n;
        bar();
        for (unsigned i = tid; i < some * (HD / 4); i += THREADS) {
            const unsigned row = i / (HD / 4);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (unsigned p = 0; p < parts; ++p) {
                const float4 x = __ldcg(reinterpret_cast<const float4 *>(A.part_o + slot_of(p) * R * HD) +
                                        (size_t)row0 * (HD / 4) + i);
                const float w = weights[p * some + row];
                v.x = fmaf(w, x.x, v.x); v.y = fmaf(w, x.y, v.y); v.z = fmaf(w, x.z, v.z); v.w = fmaf(w, x.w, v.w);
            }
            put(row0 + row, i % (HD / 4), v);
        }
    }
    bar();
}

// Four values of one query row in the rows' type.
FYB_DEV float4 kv8_load4(const void *p, unsigned type, size_t at)
{
    float x[4];
    if (type == T_F32) {
        const float *f = static_cast<const float *>(p) + at;
        if (((uintptr_t)f & 15) == 0) return *reinterpret_cast<const float4 *>(f);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = f[i];
    } else if (type == T_F16) {
        const __half *f = static_cast<const __half *>(p) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __half2float(f[i]);
    } else {
        const __nv_bfloat16 *f = static_cast<const __nv_bfloat16 *>(p) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __bfloat162float(f[i]);
    }
    return make_float4(x[0], x[1], x[2], x[3]);
}
FYB_DEV void kv8_store4(void *p, unsigned type, size_t at, float4 v)
{
    const float x[4] = {v.x, v.y, v.z, v.w};
    if (type == T_F32) {
        float *f = static_cast<float *>(p) + at;
        if (((uintptr_t)f & 15) == 0) { *reinterpret_cast<float4 *>(f) = v; return; }
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = x[i];
    } else if (type == T_F16) {
        __half *f = static_cast<__half *>(p) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __float2half_rn(x[i]);
    } else {
        __nv_bfloat16 *f = static_cast<__nv_bfloat16 *>(p) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __float2bfloat16_rn(x[i]);
    }
}

// ---- tiles of the cache by TMA -------------------------------------------------
// A tensor map over K or V as token rows of head_dim bytes, boxes of one block
// (64 rows at most) in the swizzle of head_dim bytes: 16-byte chunk c of token
// row t lies at chunk c ^ (t & 7) (128-byte rows) or c ^ (t >> 1 & 3) (64-byte
// rows), so eight token rows of one chunk are read without bank conflicts.
int kv8_tensor_map(CUtensorMap *map, const fyb_kv8_cache &c, const void *pool);
FYB_DEV void tma_load_rows(void *dst, const CUtensorMap *map, int row, uint64_t *bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        :: "r"(smem_u32(dst)), "l"(map), "r"(0), "r"(row), "r"(smem_u32(bar)) : "memory");
}
template <int HD> FYB_DEV unsigned kv8_swizzle(unsigned row) { return HD == 128 ? row & 7u : (row >> 1) & 3u; }

FYB_DEV void mbar_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(smem_u32(bar)) : "memory");
}
FYB_DEV float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four stored bytes as two fp16 pairs (bytes 0, 1 and 2, 3), exactly.
template <unsigned FMT> FYB_DEV void kv8_halves(unsigned x, unsigned &a, unsigned &b)
{
    if constexpr (FMT == FYB_KV8_INT8) {
        // byte + 128 under the high byte of 1024 is the half 1152 + value
        x ^= 0x80808080u;
        const __half2 bias = __float2half2_rn(1152.f);
        const unsigned lo = __byte_perm(x, 0x64646464u, 0x4140), hi = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 p = __hsub2(*reinterpret_cast<const __half2 *>(&lo), bias);
        const __half2 q = __hsub2(*reinterpret_cast<const __half2 *>(&hi), bias);
        a = *reinterpret_cast<const unsigned *>(&p);
        b = *reinterpret_cast<const unsigned *>(&q);
    } else {
        asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
            : "=r"(a), "=r"(b) : "r"(x));
    }
}

int launch_kv8_decode(const Kv8Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned grid, cudaStream_t s);
constexpr unsigned KV8_DECODE_ROWS = 8;  // most query rows per KV head of the decode kernel

}  // namespace fyb
