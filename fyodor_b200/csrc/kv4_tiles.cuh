// kv4_tiles.cuh - attention over the paged 4-bit cache for many query rows of 16
// bits per KV head (drafts, prompt chunks), on the 5th-generation tensor cores. One
// instantiation per head dimension and row tile (kv4_tiles_inst.cu).
//
// Per tile of 128 positions, with the query rows in the 128 lanes of tensor memory:
//
//   S[row][position] = Q K^T        tcgen05.mma kind::f16, M = 128, N = 128, K = head_dim
//   P = 2^(S factor - m)            one thread a row
//   O[row][hd] += P V               P from tensor memory, N = head_dim, K = 128 positions
//
// K and V come as 4-bit tiles by TMA; four warps each make fp16 rows low + scale n
// of them in shared memory, one rounding (2^-11 of the value, a step of the cache
// is a fifteenth of its group's range), in the order of a word's numbers: 0 4 1 5
// 2 6 3 7. q lies in the same order, the output is put back.
//
// Row tiles of 256 rows (prompt chunks) are two groups of 128 lanes, each with four
// softmax warps, S and O of its own, over the same K and V: a tile is converted once for
// both. A group makes and hands on the weights of half a tile at a time, P in the place
// of scores that have been read, and the groups are half a tile apart, so one group's
// products run while the other's weights are made. Row tiles of 64 or 32 rows (drafts):
// one group, whose lanes hold two or four copies of the rows; copy c takes the positions
// of its part of a tile, its P (in the upper half of S) being 0 elsewhere: every thread
// has positions to do, and what the copies hold is joined like any parts. One O leaves
// room for S of two tiles and for q in tensor memory, which saves its reads and its
// place in shared memory.
//
// Bound, at 256 rows, by the chain of a half tile's products and weights: a tile of 128
// positions takes 4200 cycles, of which its products alone would take 2050 and its
// exponentials 2050; a chunk of 500 rows of four heads at 16000 161 us (800 TFLOP/s,
// 0.49 of the measured rate; weights of a whole tile at a time 205, products of 64 columns for
// the half tiles 259, since q is then read twice as often). At 32 rows by the products of
// full 128-lane tiles, 1250 of a tile's 1820 cycles, and the MMA warp's waits: 32 ragged
// drafts of eight rows of four heads 249 us, 0.38 of the measured copy. What runs once a
// segment costs as much as 8 tiles (6 of 256 rows), and its instructions more than its
// data.
//
// The maximum m of a row moves only when a weight is above 2^8 (with 2^4 a chunk of 500
// at 16000 took 170 us, with 2^8 160).
//
// K, V and the weights are rounded to fp16 once each (the sum of the weights is not):
// fp16 rows are 3.0e-4 to 4.1e-4 of the norm off at 20 to 9000 tokens (5.0e-4 where K
// has strong channels), their rounded output alone 2.1e-4; bf16 rows are at their
// output's rounding.
#pragma once
#include "kv4_attention.cuh"
#include "kt_mma.cuh"

namespace fyb {

constexpr int K4T_CONV = 4, K4T_META = 8;
FYB_HOST_DEV constexpr unsigned k4t_segs(int NR) { return NR == 256 ? 2 : 4; }   // segments handed on at a time (room for no more)
FYB_HOST_DEV constexpr int k4t_groups(int NR) { return NR == 256 ? 2 : 1; }      // groups of four softmax warps
FYB_HOST_DEV constexpr int k4t_threads(int NR) { return 32 * (4 * k4t_groups(NR) + 2 * K4T_CONV + 3); }

// A segment's beginning and end, in tiles (drafts as above: with 4 tiles 266 us, 6 259, 8 242, 10 243; the chunk with 9 181, 6 174, 3 176)
FYB_HOST_DEV constexpr int k4t_cost(int NR) { return NR == 256 ? 6 : 8; }

template <int HD, int NR> struct K4tShape {
    static constexpr int ROW = HD / 2, SCALES = HD / 64 * 4;                 // bytes of a token's row, of its scales
    static constexpr int RAW_S = K4_TILE * ROW, RAW = RAW_S + 1024;           // a tile of K or V as it lies in the cache, and its scales
    static constexpr bool Q_TM = NR < 256;                                   // q in tensor memory
    // raw tiles on their way: as many as there is room for
    static constexpr int KS = HD == 64 || Q_TM ? 4 : 2, VS = HD == 64 || Q_TM ? 4 : 1;
    static constexpr int HALF = 128 * 128, TILE = HD / 64 * HALF;            // fp16 rows of 64 values in 128 bytes
    static constexpr int O_COLS = 32, O_STRIDE = O_COLS + 4;                  // columns of O of copies at a time, floats between lanes of them
    static constexpr int OFF_K = 0, OFF_V = 2 * TILE, OFF_Q = 4 * TILE, OFF_RK = OFF_Q + (Q_TM ? 0 : 2 * TILE), OFF_RV = OFF_RK + KS * RAW,
                         OFF_O = OFF_RV + VS * RAW, STAGED = Q_TM ? 128 * O_STRIDE : 0, OFF_END = OFF_O + STAGED * 4;
    // tensor memory columns: two S with P in the upper half, O of each group, q
    static constexpr int P = 64, O = 256, Q = 256 + HD;
};
template <int NR> struct K4tShared {
    static constexpr unsigned SEGS = k4t_segs(NR);
    Kv8Segment seg[SEGS], walked[k4t_threads(NR) / 32];
    Kv8Place place;
    uint64_t seg_full[SEGS], seg_empty[SEGS], rk_full[4], rk_empty[4], rv_full[4], rv_empty[4], k_full[2], k_empty[2],
        v_full[2], v_empty[2], s_full[2], p_full[4], o_done[4], o_free[2], q_full[SEGS], q_empty, meta_full[K4T_META], drained;
    float factor[SEGS][k4t_groups(NR) * 128];  // score factor of each lane's row
    float2 ml[NR < 256 ? 128 : 1];
    unsigned here[K4T_META];                       // which groups of 16 positions of a tile are loaded
    uint32_t tmem;
    unsigned flag, dead;
};

template <int COST> static __device__ __noinline__ void k4t_segment(const Kv4Attention &A, const Kv8Place &place, unsigned k, Kv8Segment *s)
{
    Kv8Walk<K4_TILE, COST> walk(A, place);
    for (unsigned i = 0; i <= k; ++i)
        if (!walk.next(*s)) { s->t1 = 0; break; }
}

// Eight numbers of a word as fp16 values low + scale n, in the order 0 4 1 5 2 6 3 7. A number under the bits of 1024
// (or, four bits higher, of 64) is that much more, taken off exactly; then one fused multiply-add.
FYB_DEV uint4 k4t_values(unsigned x, __half2 scale, __half2 low)
{
    unsigned out[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned y = x >> (8 * i);
        const unsigned a = (y & 0x000f000fu) | 0x64006400u, b = (y & 0x00f000f0u) | 0x54005400u;
        const __half2 u = __hfma2(__hsub2(*reinterpret_cast<const __half2 *>(&a), __float2half2_rn(1024.f)), scale, low);
        const __half2 v = __hfma2(__hsub2(*reinterpret_cast<const __half2 *>(&b), __float2half2_rn(64.f)), scale, low);
        out[2 * i] = *reinterpret_cast<const unsigned *>(&u);
        out[2 * i + 1] = *reinterpret_cast<const unsigned *>(&v);
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// Eight values of a query row of 16 bits as they lie; vec: in one access. (What runs once a segment is kept small: its
// instructions come from L2, 128 bytes in some 600 cycles.)
static __device__ __noinline__ uint4 k4t_gather8(const unsigned short *q)
{
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __ldg(q + 2 * i) | (unsigned)__ldg(q + 2 * i + 1) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}
FYB_DEV uint4 k4t_load8(const Kv4Attention &A, size_t at)
{
    const unsigned short *q = static_cast<const unsigned short *>(A.q) + at;
    return A.vec ? __ldg(reinterpret_cast<const uint4 *>(q)) : k4t_gather8(q);
}
// 16 bytes global -> shared by this thread, and until all that it asked for have come.
FYB_DEV void k4t_async16(void *dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(smem_u32(dst)), "l"(src) : "memory");
}
FYB_DEV void k4t_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Sizes of the two values of a word, the larger of each of two words: bits without a sign are in order, NaN last.
FYB_DEV unsigned k4t_larger(unsigned x, unsigned y) { return __vmaxu2(x & 0x7fff7fffu, y & 0x7fff7fffu); }
FYB_DEV float2 k4t_two(bool f16, unsigned w) { return f16 ? kt_unpack(w) : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
// Power of two that a row with this largest size is multiplied by, to lie below 2^13.
FYB_DEV int k4t_up(bool f16, unsigned sizes)
{
    const float2 y = k4t_two(f16, sizes);
    return 12 - kt_exponent(fmaxf(y.x, y.y));
}
// Eight values times 2^e (and the sign of scale) as fp16, in the order of a word's numbers.
FYB_DEV uint4 k4t_halves(bool f16, uint4 q, int e, float scale)
{
    const float up = copysignf(kt_power(min(e, 127)), scale), up2 = kt_power(e - min(e, 127));
    const float2 a = k4t_two(f16, q.x), b = k4t_two(f16, q.y), c = k4t_two(f16, q.z), d = k4t_two(f16, q.w);
    auto pair = [&](float y, float z) { return kt_pack(y * up * up2, z * up * up2); };
    return make_uint4(pair(a.x, c.x), pair(a.y, c.y), pair(b.x, d.x), pair(b.y, d.y));
}

// Partials lie as [4 columns][row]: a warp's rows, a lane each, are written and read side by side (as rows of head_dim
// values each 16 bytes were a sector of their own: a prompt's partial took 12000 to 20000 cycles to be seen).
template <int NR, int HD> FYB_DEV size_t k4t_part(unsigned slot, unsigned piece, unsigned row)
{
    return ((size_t)slot * (HD / 4) + piece) * NR + row;
}
// Where row `row` of a segment lies in the output, and eight of its values.
FYB_DEV size_t k4t_out(const Kv4Attention &A, unsigned first_row, unsigned head, unsigned row, unsigned hd)
{
    return (size_t)(first_row + row / A.group) * A.out_stride + (size_t)(head * A.group + row % A.group) * hd;
}
FYB_DEV void k4t_write(const Kv4Attention &A, size_t out, float4 lo, float4 hi)
{
    if (A.vec_out) {
        auto two = [&](float x, float y) {
            if (A.type == T_F16) return kt_pack(x, y);
            const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
            return *reinterpret_cast<const unsigned *>(&h);
        };
        *reinterpret_cast<uint4 *>(static_cast<unsigned short *>(A.out) + out) =
            make_uint4(two(lo.x, lo.y), two(lo.z, lo.w), two(hi.x, hi.y), two(hi.z, hi.w));
    } else {
        kv8_store4(A.out, A.type, out, lo);
        kv8_store4(A.out, A.type, out + 4, hi);
    }
}

// Row tiles of 256: the parts of the segment that begins in each CTA of the tiles kernel and goes on in others, joined in
// order, 32 rows a CTA, a lane each, and the warps share the columns. L2's latency is what takes time: four parts of PIECES
// pieces are on their way at once. A launch of its own, so that all SMs join: by the segment's last CTA, as below, a prompt
// of 64 rows of four heads at 16000 took 86 us instead of 59, one of 500 rows 174 instead of 167.
constexpr int K4T_JOIN = 256;
template <int HD, int NR> __global__ void __launch_bounds__(K4T_JOIN) kv4_join_kernel(const __grid_constant__ Kv4Attention A)
{
    constexpr unsigned PIECES = HD / 4 / (K4T_JOIN / 32), PARTS = 4;
    const K4tJoin j = A.join[blockIdx.x];
    const unsigned row = blockIdx.y * 32 + (threadIdx.x & 31), c = threadIdx.x / 32 * PIECES, parts = j.last - blockIdx.x + 1;
    if (row >= j.rows) return;
    auto slot_of = [&](unsigned p) { return 2 * (blockIdx.x + p) + (p == 0 ? 1 : 0); };
    float m = -3.4e38f, l = 0.f;
    float4 v[PIECES];
#pragma unroll
    for (unsigned u = 0; u < PIECES; ++u) v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (unsigned p = 0; p < parts; p += PARTS) {
        float4 x[PARTS][PIECES];
        float2 ml[PARTS];
#pragma unroll
        for (unsigned i = 0; i < PARTS; ++i) {
            ml[i] = make_float2(-3.4e38f, 0.f);
            if (p + i < parts) ml[i] = __ldcg(&A.part_ml[(size_t)slot_of(p + i) * NR + row]);
#pragma unroll
            for (unsigned u = 0; u < PIECES; ++u) {
                x[i][u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (p + i < parts) x[i][u] = __ldcg(reinterpret_cast<const float4 *>(A.part_o) + k4t_part<NR, HD>(slot_of(p + i), c + u, row));
            }
        }
        float top = m;
#pragma unroll
        for (unsigned i = 0; i < PARTS; ++i) top = fmaxf(top, ml[i].x);
        const float old = ex2(m - top);
        m = top;
        l *= old;
#pragma unroll
        for (unsigned u = 0; u < PIECES; ++u) { v[u].x *= old; v[u].y *= old; v[u].z *= old; v[u].w *= old; }
#pragma unroll
        for (unsigned i = 0; i < PARTS; ++i) {
            const float w = ex2(ml[i].x - m);
            l = fmaf(w, ml[i].y, l);
#pragma unroll
            for (unsigned u = 0; u < PIECES; ++u) {
                v[u].x = fmaf(w, x[i][u].x, v[u].x); v[u].y = fmaf(w, x[i][u].y, v[u].y);
                v[u].z = fmaf(w, x[i][u].z, v[u].z); v[u].w = fmaf(w, x[i][u].w, v[u].w);
            }
        }
    }
    const float n = l > 0.f || isnan(l) ? 1.f / l : 0.f;
    const size_t out = k4t_out(A, j.first_row, j.head, row, HD);
#pragma unroll
    for (unsigned u = 0; u < PIECES; u += 2) {
        auto times = [&](float4 y) { return make_float4(y.x * n, y.y * n, y.z * n, y.w * n); };
        k4t_write(A, out + 4 * (c + u), times(v[u]), times(v[u + 1]));
    }
}

// Row tiles of 64 or 32: the CTA's partial is written, and the last CTA of the segment joins them all (a launch more took
// 32 ragged drafts of 32 rows from 242 to 250 us, 16 requests of 32 rows at 8100 from 77 to 81).
template <int NR, int HD, int THREADS, typename Bar, typename Put>
FYB_DEV void k4t_join(const Kv4Attention &A, const Kv8Parts &of, unsigned tid, unsigned rows, unsigned *flag, Bar bar, Put put)
{
    constexpr unsigned LANES = THREADS / NR, PIECES = 4, PARTS = 4;
    __threadfence();
    bar();
    if (tid == 0) *flag = atomicAdd(&A.counters[of.first], 1u) == of.last - of.first;
    bar();
    if (!*flag) return;
    __threadfence();
    if (tid == 0) A.counters[of.first] = 0;
    const unsigned parts = of.last - of.first + 1, row = tid % NR;
    if (row >= rows) return;
    auto slot_of = [&](unsigned p) { return 2 * (of.first + p) + (p == 0 ? 1 : 0); };
    float m = -3.4e38f, l = 0.f;
#pragma unroll 4
    for (unsigned p = 0; p < parts; ++p) m = fmaxf(m, __ldcg(&A.part_ml[(size_t)slot_of(p) * NR + row].x));
#pragma unroll 4
    for (unsigned p = 0; p < parts; ++p) {
        const float2 y = __ldcg(&A.part_ml[(size_t)slot_of(p) * NR + row]);
        l = fmaf(ex2(y.x - m), y.y, l);
    }
    const float n = l > 0.f || isnan(l) ? 1.f / l : 0.f;
#pragma unroll 1
    for (unsigned c = tid / NR * PIECES; c < HD / 4; c += LANES * PIECES) {
        float4 v[PIECES];
#pragma unroll
        for (unsigned u = 0; u < PIECES; ++u) v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (unsigned p = 0; p < parts; p += PARTS) {
            float4 x[PARTS][PIECES];
            float w[PARTS];
#pragma unroll
            for (unsigned i = 0; i < PARTS; ++i) {
                w[i] = -INFINITY;
                if (p + i < parts) w[i] = __ldcg(&A.part_ml[(size_t)slot_of(p + i) * NR + row].x);
#pragma unroll
                for (unsigned u = 0; u < PIECES; ++u) {
                    x[i][u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (p + i < parts) x[i][u] = __ldcg(reinterpret_cast<const float4 *>(A.part_o) + k4t_part<NR, HD>(slot_of(p + i), c + u, row));
                }
            }
#pragma unroll
            for (unsigned i = 0; i < PARTS; ++i) {
                const float f = ex2(w[i] - m) * n;
#pragma unroll
                for (unsigned u = 0; u < PIECES; ++u) {
                    v[u].x = fmaf(f, x[i][u].x, v[u].x); v[u].y = fmaf(f, x[i][u].y, v[u].y);
                    v[u].z = fmaf(f, x[i][u].z, v[u].z); v[u].w = fmaf(f, x[i][u].w, v[u].w);
                }
            }
        }
#pragma unroll
        for (unsigned u = 0; u < PIECES; u += 2) put(row, c + u, v[u], v[u + 1]);
    }
}

template <int HD, int NR>
__global__ void __launch_bounds__(k4t_threads(NR), 1) kv4_tiles_kernel(const __grid_constant__ Kv4Attention A, const __grid_constant__ CUtensorMap kmap,
    const __grid_constant__ CUtensorMap vmap)
{
    using S = K4tShape<HD, NR>;
    constexpr unsigned CONV = K4T_CONV, GROUPS = k4t_groups(NR), SOFT = 4 * GROUPS, W_CONV = SOFT, W_TMA = SOFT + 2 * CONV, W_MMA = W_TMA + 2;
    constexpr unsigned CP = GROUPS == 2 ? 1 : 128 / NR, HALVES = GROUPS, CW = 128 / CP / HALVES, CHUNKS = CW / 32;   // copies, and the positions and blocks of 32 taken at a time
    constexpr unsigned SEGS = k4t_segs(NR);
    constexpr int G64 = HD / 64;
    extern __shared__ unsigned char k4t_smem[];
    unsigned char *ring = k4t_smem + ((1024u - (smem_u32(k4t_smem) & 1023u)) & 1023u);
    K4tShared<NR> &sh = *reinterpret_cast<K4tShared<NR> *>(ring + S::OFF_END);
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), kv = A.c.kv_heads, GR = A.group;
    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(sh.rk_full + i, 1); mbar_init(sh.rk_empty + i, CONV);
            mbar_init(sh.rv_full + i, 1); mbar_init(sh.rv_empty + i, CONV);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(sh.k_full + i, CONV); mbar_init(sh.k_empty + i, 1);
            mbar_init(sh.v_full + i, CONV); mbar_init(sh.v_empty + i, 1);
            mbar_init(sh.s_full + i, 1); mbar_init(sh.o_free + i, 4);
        }
        for (int i = 0; i < 4; ++i) { mbar_init(sh.p_full + i, 4); mbar_init(sh.o_done + i, 1); }
        mbar_init(&sh.q_empty, 1); mbar_init(&sh.drained, 1);
        for (int i = 0; i < K4T_META; ++i) mbar_init(sh.meta_full + i, 1);
        for (unsigned i = 0; i < SEGS; ++i) {
            mbar_init(sh.q_full + i, S::Q_TM ? 4 : 2 * CONV);
            mbar_init(sh.seg_full + i, 1);
            mbar_init(sh.seg_empty + i, SOFT + 2 * CONV + 2);
        }
        sh.dead = 0;
        fence_barrier_init();
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    kt_fence_before();
    {
        const Kv8Place place = kv8_place<K4_TILE, k4t_threads(NR), 2, k4t_cost(NR)>(A);  // CTA barriers inside
        if (tid == 0) sh.place = place;
    }
    __syncthreads();
    kt_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    unsigned n = 0, seg = 0;  // tiles and segments of this CTA so far
    volatile unsigned *dead = &sh.dead;  // a wait ran out: nobody waits any more, the error word is set
    auto wait = [&](uint64_t *bar, unsigned parity) { kt_wait(bar, parity, dead); };
    auto arrive = [&](uint64_t *bar) { __syncwarp(); if (lane == 0) mbar_arrive(bar); };
    // The segment that comes next; done() with it before the next is asked for. Once a wait has run out every warp
    // walks by itself: all of them still take the same steps, so none is left at a barrier.
    auto next = [&]() -> const Kv8Segment * {
        wait(sh.seg_full + seg % SEGS, seg / SEGS);
        const Kv8Segment *s = sh.seg + seg % SEGS;
        if (__builtin_expect(*dead, 0)) {
            s = sh.walked + warp;
            if (lane == 0) k4t_segment<k4t_cost(NR)>(A, sh.place, seg, sh.walked + warp);
            __syncwarp();
        }
        return s->t1 ? s : nullptr;
    };
    auto done = [&] { arrive(sh.seg_empty + seg % SEGS); ++seg; };

    if (warp < SOFT) {
        // ================================================== softmax
        // this thread's lane of tensor memory, its row, and its first position of a tile
        const unsigned wg = warp >> 2, at = tid & 127, rho = GROUPS == 2 ? tid : at % NR, first = CP > 1 ? at / NR * CW : 0;
        const uint32_t lanes = (warp & 3) << 21;
        const uint32_t o_at = tmem + lanes + S::O + wg * HD;
        float *stage = reinterpret_cast<float *>(ring + S::OFF_O);
        unsigned k = 0;  // tiles of this group so far
        bool goes_on = false;  // the last segment, in the next CTA
        auto bar = [] { asm volatile("bar.sync 1, %0;" :: "n"(32 * SOFT) : "memory"); };
        constexpr float LAG = 8.f, P_UP = 6.f;  // weights are 2^P_UP times themselves, clear of fp16's smallest numbers, and up to 2^14
        constexpr unsigned FAR = 0x4b800000u;  // bits of 2^24
        while (const Kv8Segment *sp = next()) {
            const Kv8Segment &s = *sp;
            const int t0 = s.t0, t1 = s.t1, j0 = s.row_tile * (int)A.row_tile;
            const int nrows = min((int)A.row_tile, s.q.rows - j0) * (int)GR;
            const int limit = (int)rho < nrows ? s.q.len - s.q.n + j0 + (int)(rho / GR) + 1 : 0;  // positions the row attends
            const int all = max(0, s.q.len - s.q.n + j0 + 1);                                      // positions every row attends
            wait(sh.q_full + seg % SEGS, seg / SEGS);
            const float f = sh.factor[seg % SEGS][GROUPS == 2 ? tid : at];
            float m = -3.4e38f, l = 0.f;   // m: the maximum less P_UP
            const bool mine = GROUPS == 1 || wg == 0 || nrows > 128;  // whether the group has rows
            const unsigned tiles = (unsigned)(t1 - t0);
            if (!mine) n += tiles;
            for (int t = t0; mine && t < t1; ++t, ++n, ++k) {
                wait(sh.meta_full + n % K4T_META, n / K4T_META);
                const unsigned here = sh.here[n % K4T_META];
#pragma unroll 1
                for (unsigned h = 0; h < HALVES; ++h) {
                    // S: the group's, or the tile's of two, its weights (P); what it waits for has come k, or k / 2, times before
                    const unsigned b = GROUPS == 2 ? 2 * wg + h : k & 1, turn = GROUPS == 2 ? k : k >> 1;
                    const unsigned from = GROUPS == 2 ? 64 * h : first;  // first position in the tile
                    const unsigned of = GROUPS == 2 ? wg : b;
                    if (h == 0) {
                        wait(sh.s_full + of, turn);
                        kt_fence_after();
                    }
                    const uint32_t s_of = tmem + lanes + of * 128, s_at = s_of + from, p_at = s_of + (GROUPS == 2 ? from + 32 : S::P);
                    if (__builtin_expect(here != 0xffu || (t + 1) * K4_TILE > all, 0)) {
                        // what the row does not attend becomes -inf where it lies: the rest has one form, and fits the
                        // instruction cache with the other roles
#pragma unroll 1
                        for (unsigned c = 0; c < CW; c += 16) {
                            float y[16];
                            kt_ld16(s_at + c, y);
                            kt_wait_ld();
                            const int left = here >> ((from + c) / 16) & 1 ? limit - (t * K4_TILE + (int)(from + c)) : 0;
#pragma unroll
                            for (int i = 0; i < 16; ++i) y[i] = i < left ? y[i] : -INFINITY;
                            kt_st16(s_at + c, y);
                        }
                        kt_wait_st();
                    }
                    float x[CHUNKS][32], tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (unsigned c = 0; c < CHUNKS; ++c) kt_ld32(s_at + 32 * c, x[c]);
                    kt_wait_ld();
#pragma unroll
                    for (unsigned c = 0; c < CHUNKS; ++c)
#pragma unroll
                        for (int i = 0; i < 32; i += 2) tops[i / 2 % 4] = fmaxf(tops[i / 2 % 4], fmaxf(x[c][i], x[c][i + 1]));
                    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * f;
                    float fx = f;
                    const bool up = top - m > LAG + P_UP, far = (__float_as_uint(top) & 0x7fffffffu) - FAR < 0x7f800000u - FAR;
                    if (__any_sync(0xffffffffu, up || far)) {
                        if (__any_sync(0xffffffffu, far)) {
                            // rows of scores so large that m is off by a half and more of a unit: their products are rounded as
                            // m is, or a weight's exponent could be beyond fp16's (at 2^28 by half of 32). Asked with `up`, in
                            // one vote: ragged drafts 246 us without it, 249 so, 251 in a vote of its own
                            const float times = far ? f : 1.f;
#pragma unroll 1
                            for (unsigned c = 0; c < CW; c += 16) {
                                float y[16];
                                kt_ld16(s_at + c, y);
                                kt_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; ++i) y[i] *= times;
                                kt_st16(s_at + c, y);
                            }
                            kt_wait_st();
#pragma unroll
                            for (unsigned c = 0; c < CHUNKS; ++c) kt_ld32(s_at + 32 * c, x[c]);
                            kt_wait_ld();
                            if (far) fx = 1.f;
                        }
                        // ---- new maxima, and the sums so far in their units
                        const float now = up ? top - P_UP : m, alpha = up ? ex2(m - now) : 1.f;
                        m = now;
                        l *= alpha;
                        if (t > t0 || h) {
                            if (GROUPS == 2) wait(sh.o_done + (b ^ 1), h ? k : k - 1); else wait(sh.o_done + (b ^ 1), (k - 1) >> 1);
                            kt_fence_after();
#pragma unroll 1
                            for (int c = 0; c < HD; c += 16) {
                                float y[16];
                                kt_ld16(o_at + c, y);
                                kt_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; ++i) y[i] *= alpha;
                                kt_st16(o_at + c, y);
                            }
                            kt_wait_st();
                        }
                    }
                    // ---- weights: P takes the place of scores that have been read
                    const F2 f2x = f2(fx, fx), mx = f2(-m, -m);
                    F2 sums[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
                    if constexpr (CP > 1) {  // 0 for the positions of the other copies
                        float z[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) z[i] = 0.f;
#pragma unroll
                        for (unsigned c = 0; c < 64; c += 16)
                            if (c < first / 2 || c >= (first + CW) / 2) kt_st16(p_at + c, z);
                    }
#pragma unroll
                    for (unsigned c = 0; c < CHUNKS; ++c) {
                        unsigned w[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 e = f2_get(f2_fma(f2(x[c][i], x[c][i + 1]), f2x, mx));
                            const float p0 = ex2(e.x), p1 = ex2(e.y);
                            sums[i / 2 % 2] = f2_add(sums[i / 2 % 2], f2(p0, p1));
                            w[i / 2] = kt_pack(p0, p1);
                        }
                        kt_st16(p_at + first / 2 + 16 * c, reinterpret_cast<const float *>(w));
                    }
                    const float2 l2 = f2_get(f2_add(sums[0], sums[1]));
                    l += l2.x + l2.y;
                    kt_wait_st();
                    kt_fence_before();
                    arrive(sh.p_full + b);
                }
            }
            // ---- the segment's part
            const bool whole = s.t0 == 0 && s.t1 == s.tiles;
            const Kv8Parts of = kv8_parts(s, sh.place);
            auto place_of = [&](unsigned row) { return k4t_out(A, (unsigned)(s.q.first + j0), s.head, row, HD); };
            // columns 8 chunk.. of a row, in the order of a word's numbers
            auto leave = [&](unsigned row, size_t out, unsigned chunk, const float *z) {
                const float4 lo = make_float4(z[0], z[2], z[4], z[6]), hi = make_float4(z[1], z[3], z[5], z[7]);
                if (!whole) {
                    float4 *o = reinterpret_cast<float4 *>(A.part_o) + k4t_part<NR, HD>(of.slot, 2 * chunk, row);
                    o[0] = lo;
                    o[NR] = hi;
                } else {
                    k4t_write(A, out + 8 * chunk, lo, hi);
                }
            };
            if constexpr (GROUPS == 2) {
                if (mine) {
                    wait(sh.o_done + 2 * wg + 1, k - 1);
                    kt_fence_after();
                    const float own = !whole ? 1.f : l > 0.f || isnan(l) ? 1.f / l : 0.f;
                    const bool real = (int)rho < nrows;
                    const size_t out = real ? place_of(rho) : 0;
#pragma unroll 1
                    for (unsigned c = 0; c < HD; c += 16) {
                        float y[16];
                        kt_ld16(o_at + c, y);
                        kt_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[i] *= own;
                        if (real) {
                            leave(rho, out, c / 8, y);
                            leave(rho, out, c / 8 + 1, y + 8);
                        }
                    }
                    kt_fence_before();
                    arrive(sh.o_free + wg);
                    if (!whole && real) A.part_ml[(size_t)of.slot * NR + rho] = make_float2(m, l);
                }
            } else {
                // what the copies hold of a row, joined
                wait(sh.o_done + ((k - 1) & 1), (k - 1) >> 1);
                kt_fence_after();
                sh.ml[tid] = make_float2(m, l);
                bar();
                float own;
                {
                    float top = -INFINITY, sum = 0.f;
#pragma unroll
                    for (unsigned p = 0; p < CP; ++p) top = fmaxf(top, sh.ml[p * NR + rho].x);
#pragma unroll
                    for (unsigned p = 0; p < CP; ++p) {
                        const float2 y = sh.ml[p * NR + rho];
                        sum = fmaf(y.y, ex2(y.x - top), sum);
                    }
                    own = ex2(m - top);
                    if (whole) own *= sum > 0.f || isnan(sum) ? 1.f / sum : 0.f;
                    if (!whole && (int)tid < nrows) A.part_ml[(size_t)of.slot * NR + tid] = make_float2(top, sum);
                }
#pragma unroll 1
                for (unsigned c = 0; c < HD; c += S::O_COLS) {
                    float y[S::O_COLS];
                    kt_ld32(o_at + c, y);
                    kt_wait_ld();
#pragma unroll
                    for (int i = 0; i < S::O_COLS; i += 4)
                        *reinterpret_cast<float4 *>(stage + tid * S::O_STRIDE + i) = make_float4(y[i] * own, y[i + 1] * own, y[i + 2] * own, y[i + 3] * own);
                    bar();
#pragma unroll 1
                    for (unsigned i = tid; i < (unsigned)nrows * (S::O_COLS / 8); i += 32 * SOFT) {
                        const unsigned row = i / (S::O_COLS / 8), part = i % (S::O_COLS / 8);
                        float z[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) z[j] = 0.f;
#pragma unroll
                        for (unsigned p = 0; p < CP; ++p)
#pragma unroll
                            for (int j = 0; j < 8; j += 4) {
                                const float4 u = *reinterpret_cast<const float4 *>(stage + (p * NR + row) * S::O_STRIDE + 8 * part + j);
                                z[j] += u.x; z[j + 1] += u.y; z[j + 2] += u.z; z[j + 3] += u.w;
                            }
                        leave(row, place_of(row), c / 8 + part, z);
                    }
                    bar();
                }
                kt_fence_before();
                arrive(sh.o_free);
            }
            if constexpr (GROUPS == 1) {
                if (!whole) {
                    k4t_join<NR, HD, 32 * SOFT>(A, of, tid, (unsigned)nrows, &sh.flag, bar, [&](unsigned row, unsigned piece, float4 lo, float4 hi) {
                        k4t_write(A, place_of(row) + 4 * piece, lo, hi);
                    });
                    bar();
                }
            } else if (!whole && t0 == 0) {  // goes on in other CTAs
                if (tid == 0) A.join[blockIdx.x] = K4tJoin{of.last, (unsigned)nrows, (unsigned)(s.q.first + j0), s.head};
                goes_on = true;
            }
            done();
        }
        if (GROUPS == 2 && !goes_on && tid == 0) A.join[blockIdx.x].rows = 0;
    } else if (warp < W_TMA) {
        // ================================================== K or V, 4 bits to fp16 rows; q
        const bool f16 = A.type == T_F16, is_v = warp >= W_CONV + CONV;
        const unsigned by_group = 65536 / GR + 1;  // rho times it: off by less than rho / 65536, so by less than 1 / GR
        const unsigned cw = (warp - W_CONV) % CONV, ct = cw * 32 + lane;
        constexpr unsigned TOKENS = K4_TILE / CONV;  // of a warp, eight lanes a token
        const unsigned j = lane & 7, tok0 = cw * TOKENS + (lane >> 3);
        while (const Kv8Segment *sp = next()) {
            const Kv8Segment &s = *sp;
            const int any = kv8_attended(A, s.q, s.row_tile), t0 = s.t0, t1 = s.t1;
            if (GROUPS == 2 || (!is_v && cw < 4)) {
                // ---- q rows by a power of two each. The score factor's sign goes with q: a row's largest product is its
                // largest score
                const int j0 = s.row_tile * (int)A.row_tile, nrows = min((int)A.row_tile, s.q.rows - j0) * (int)GR;
                const size_t q0 = (size_t)(s.q.first + j0) * A.q_stride + (size_t)s.head * GR * HD;
                auto at_of = [&](unsigned rho) {
                    const unsigned j = rho * by_group >> 16;  // rho / GR
                    return q0 + j * A.q_stride + (rho - j * GR) * HD;
                };
                // at least the smallest normal number: -inf times it stays -inf; NaN stays
                auto factor_of = [&](int e) {
                    const float y = fabsf(A.scale) * kt_power(-e);
                    return y < 1.17549435e-38f ? 1.17549435e-38f : y;
                };
                if constexpr (S::Q_TM) {
                    // to tensor memory, a thread a lane's row
                    const unsigned rho = ct % NR;
                    const bool real = (int)rho < nrows;
                    const size_t at = at_of(real ? rho : 0);
                    unsigned top = 0;
#pragma unroll 1
                    for (int i = 0; real && i < HD; i += 64) {
                        uint4 x[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u) x[u] = k4t_load8(A, at + i + 8 * u);
#pragma unroll
                        for (int u = 0; u < 8; ++u) top = k4t_larger(top, k4t_larger(k4t_larger(x[u].x, x[u].y), k4t_larger(x[u].z, x[u].w)));
                    }
                    const int e = k4t_up(f16, top);
                    if (seg) wait(&sh.q_empty, seg - 1);  // the last segment's products have read their q
                    kt_fence_after();
#pragma unroll 1
                    for (int i = 0; i < HD; i += 32) {
                        uint4 h[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) h[u] = real ? k4t_halves(f16, k4t_load8(A, at + i + 8 * u), e, A.scale) : make_uint4(0, 0, 0, 0);
                        kt_st16(tmem + (cw << 21) + S::Q + i / 2, reinterpret_cast<const float *>(h));
                    }
                    kt_wait_st();
                    sh.factor[seg % SEGS][ct] = factor_of(e);
                    kt_fence_before();
                } else {
                    // to shared memory, eight values a lane: all rows as they lie first, and then each in its place
                    constexpr unsigned LANES = HD / 8, STEP = 32 / LANES, STEPS = NR / (2 * CONV) / STEP;  // lanes of a row, rows of a load
                    const unsigned piece = lane % LANES, row0 = (warp - W_CONV) * STEPS * STEP + lane / LANES;
                    auto place = [&](unsigned rho) {
                        return ring + S::OFF_Q + rho / 128 * S::TILE + piece / 8 * S::HALF + rho % 128 * 128 + ((piece % 8 ^ (rho & 7u)) << 4);
                    };
                    if (seg) wait(&sh.q_empty, seg - 1);  // the last segment's products have read their q
#pragma unroll 4
                    for (unsigned i = 0; i < STEPS; ++i) {
                        const unsigned rho = row0 + i * STEP;
                        uint4 *to = reinterpret_cast<uint4 *>(place(rho));
                        if ((int)rho >= nrows) *to = make_uint4(0, 0, 0, 0);
                        else if (A.vec) k4t_async16(to, static_cast<const unsigned short *>(A.q) + at_of(rho) + 8 * piece);
                        else *to = k4t_load8(A, at_of(rho) + 8 * piece);
                    }
                    k4t_async_wait();
#pragma unroll 2
                    for (unsigned i = 0; i < STEPS; ++i) {
                        const unsigned rho = row0 + i * STEP;
                        uint4 *at = reinterpret_cast<uint4 *>(place(rho));
                        const uint4 x = *at;
                        const unsigned top = k4t_larger(k4t_larger(x.x, x.y), k4t_larger(x.z, x.w));
                        const int e = k4t_up(f16, __reduce_max_sync(((1u << LANES) - 1) << (lane / LANES * LANES), max(top >> 16, top & 0xffffu)));
                        *at = k4t_halves(f16, x, e, A.scale);
                        if (piece == 0) sh.factor[seg % SEGS][rho] = factor_of(e);
                    }
                }
                fence_proxy_async();
                arrive(sh.q_full + seg % SEGS);
            }
            for (int t = t0; t < t1; ++t, ++n) {
                const unsigned b = n & 1, stages = is_v ? S::VS : S::KS, st = n % stages;
                wait((is_v ? sh.rv_full : sh.rk_full) + st, n / stages);
                if (n >= 2) wait((is_v ? sh.v_empty : sh.k_empty) + b, (n >> 1) - 1);
                const unsigned char *raw = ring + (is_v ? S::OFF_RV : S::OFF_RK) + st * S::RAW, *scales = raw + S::RAW_S;
                unsigned char *dst = ring + (is_v ? S::OFF_V : S::OFF_K) + b * S::TILE;
                // V of positions that no row attends, or never loaded, is 0 and not what lies there (a NaN stays one times 0)
                wait(sh.meta_full + n % K4T_META, n / K4T_META);
                const unsigned here = sh.here[n % K4T_META];
                const bool patchy = is_v && (here != 0xffu || any < (t + 1) * K4_TILE);
                // four tokens' words and scales at a time, before the first of their stores (which they might overlap, as
                // far as the compiler can tell: a token after the other took 1500 cycles a tile)
#pragma unroll
                for (unsigned i0 = 0; i0 < TOKENS / 4; i0 += 4) {
                    unsigned w[4][G64], sc[4][G64];
#pragma unroll
                    for (unsigned i = 0; i < 4; ++i) {
                        const unsigned tok = tok0 + 4 * (i0 + i);
                        if constexpr (G64 == 2) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(raw + kv4_at<HD>(tok, 8 * j));
                            const uint2 y = *reinterpret_cast<const uint2 *>(scales + tok * 8);
                            w[i][0] = x.x; w[i][1] = x.y;
                            sc[i][0] = y.x; sc[i][1] = y.y;
                        } else {
                            w[i][0] = *reinterpret_cast<const unsigned *>(raw + kv4_at<HD>(tok, 4 * j));
                            sc[i][0] = *reinterpret_cast<const unsigned *>(scales + tok * 4);
                        }
                    }
                    if (__builtin_expect(patchy, 0)) {
#pragma unroll
                        for (unsigned i = 0; i < 4; ++i) {
                            const unsigned tok = tok0 + 4 * (i0 + i);
                            const bool is = t * K4_TILE + (int)tok < any && (here >> (tok / 16) & 1);
#pragma unroll
                            for (int h = 0; h < G64; ++h) sc[i][h] = is ? sc[i][h] : 0;
                        }
                    }
#pragma unroll
                    for (unsigned i = 0; i < 4; ++i) {
                        const unsigned tok = tok0 + 4 * (i0 + i), sw = ((j ^ (tok & 7u)) << 4) + tok * 128;
#pragma unroll
                        for (int h = 0; h < G64; ++h) {
                            const __half2 sl = *reinterpret_cast<const __half2 *>(&sc[i][h]);
                            *reinterpret_cast<uint4 *>(dst + h * S::HALF + sw) = k4t_values(w[i][h], __low2half2(sl), __high2half2(sl));
                        }
                    }
                }
                arrive((is_v ? sh.rv_empty : sh.rk_empty) + st);
                fence_proxy_async();
                arrive((is_v ? sh.v_full : sh.k_full) + b);
            }
            done();
        }
    } else if (warp < W_MMA) {
        // ================================================== TMA: a warp for K, which walks the line, and one for V (one for
        // both took 1850 cycles a tile, as long as the tile)
        const bool is_v = warp > W_TMA;
        const unsigned size = 1u << A.shift, box = min(size, (unsigned)K4_TILE), per = K4_TILE / box, stages = is_v ? S::VS : S::KS;
        const CUtensorMap *map = is_v ? &vmap : &kmap;
        const __half2 *scale = is_v ? A.vs : A.ks;
        uint64_t *full = is_v ? sh.rv_full : sh.rk_full, *empty = is_v ? sh.rv_empty : sh.rk_empty;
        const unsigned raw = smem_u32(ring + (is_v ? S::OFF_RV : S::OFF_RK)), lane_at = lane % per * box;
        __syncwarp();
        Kv8Walk<K4_TILE, k4t_cost(NR)> walk(A, sh.place);
        Kv8Segment own;
        for (;;) {
            const Kv8Segment *s = &own;
            if (is_v) {
                s = next();
                if (!s) break;
            } else {
                const bool more = walk.next(own);
                if (seg >= SEGS) wait(sh.seg_empty + seg % SEGS, seg / SEGS - 1);
                if (lane == 0 && !*dead) {
                    if (more) sh.seg[seg % SEGS] = own; else sh.seg[seg % SEGS].t1 = 0;
                    mbar_arrive(sh.seg_full + seg % SEGS);
                }
                __syncwarp();
                if (!more) break;
            }
            const int blocks = (kv8_attended(A, s->q, s->row_tile) + (int)size - 1) >> A.shift, t1 = s->t1;
            const int *ids = A.table + (size_t)s->request * A.table_stride;
            const unsigned head = s->head;
            int have = -1, id = 0;  // lane holds block 32 * have + lane
            for (int t = s->t0; t < t1; ++t, ++n) {
                const int b0 = t * K4_TILE >> A.shift;
                if (b0 / 32 != have) {
                    have = b0 / 32;
                    const int b = have * 32 + (int)lane;
                    id = b < blocks ? ids[b] : -1;
                    if (b < blocks && (unsigned)id >= A.c.blocks) {  // negative ones too
                        raise_error(A.error, ERR_BOUNDS);
                        id = -1;
                    }
                }
                const unsigned st = n % stages;
                const int block = __shfl_sync(0xffffffffu, id, (b0 & 31) + (int)(lane % per));
                const bool load = lane < per && block >= 0;
                const unsigned boxes = __ballot_sync(0xffffffffu, load);
                if (n >= stages) wait(empty + st, n / stages - 1);
                if (!is_v) {  // groups of 16 positions whose block is among the loaded ones
                    const unsigned groups = __ballot_sync(0xffffffffu, lane < K4_TILE / 16 && (boxes >> (lane * 16 / box) & 1));
                    if (lane == 0) {
                        sh.here[n % K4T_META] = groups;
                        mbar_arrive(sh.meta_full + n % K4T_META);
                    }
                }
                if (lane == 0) {
                    if (boxes) mbar_expect_tx(full + st, __popc(boxes) * box * (S::ROW + S::SCALES)); else mbar_arrive(full + st);
                }
                __syncwarp();
                if (load && !*dead) {
                    const unsigned row = (((unsigned)block * kv + head) << A.shift) + ((unsigned)(t * K4_TILE) & (size - 1));
                    const unsigned dst = raw + st * S::RAW, bar = smem_u32(full + st);
                    k4_load_rows(dst + lane_at * S::ROW, map, (int)(row / (128 / S::ROW)), bar);
                    k4_copy(dst + S::RAW_S + lane_at * S::SCALES, scale + (size_t)row * G64, box * S::SCALES, bar);
                }
                __syncwarp();
            }
            if (is_v) done(); else ++seg;
        }
        if (*dead) {  // copies in flight land before the CTA leaves its shared memory
            for (unsigned i = 0; i < min(n, stages); ++i) {
                const unsigned k = n - 1 - i;
                mbar_wait_bounded(full + k % stages, k / stages & 1);
            }
        }
    } else {
        // ================================================== MMA
        // The warp runs as one and an elected lane issues: operands then sit in uniform registers.
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t qs = kt_desc(smem_u32(ring + S::OFF_Q), 16), ks = kt_desc(smem_u32(ring + S::OFF_K), 16),
                       vs = kt_desc(smem_u32(ring + S::OFF_V), S::HALF);
        // what has been asked for so far: scores and values of each group (tiles), segments of a group
        unsigned scored[2] = {0, 0}, valued[2] = {0, 0}, segs[2] = {0, 0};
        // scores of tile t of the segment
        auto ask = [&](unsigned g, int t, bool last_group, bool last) {
            const unsigned tile = n + (unsigned)t, b = GROUPS == 2 ? g : tile & 1, turn = GROUPS == 2 ? scored[g] : tile >> 1;
            if (g == 0) wait(sh.k_full + (tile & 1), tile >> 1);
            if (turn) wait(sh.o_done + (GROUPS == 2 ? 2 * g + 1 : b), turn - 1);  // P in this S has been read
            kt_fence_after();
            __syncwarp();
            if (kt_elect()) {
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const uint64_t step = (uint64_t)((k / 4 * S::HALF + k % 4 * 32) >> 4), kt = ks + ((tile & 1) * S::TILE >> 4) + step;
                    if constexpr (S::Q_TM) kt_mma(tm + b * 128, tm + S::Q + 8 * k, kt, kt_idesc(128, false), k > 0);
                    else kt_mma_ss(tm + b * 128, qs + (g * S::TILE >> 4) + step, kt, kt_idesc(128, false), k > 0);
                }
                if (last_group) kt_commit(sh.k_empty + (tile & 1));
                kt_commit(sh.s_full + b);
                if (last_group && last) kt_commit(&sh.q_empty);
            }
            __syncwarp();
            ++scored[g];
        };
        // values of it, or of its half h for one of two groups
        auto give = [&](unsigned g, unsigned h, int t, bool last_group) {
            const unsigned tile = n + (unsigned)t, b = GROUPS == 2 ? 2 * g + h : tile & 1, turn = GROUPS == 2 ? valued[g] : tile >> 1;
            const bool first = t == 0 && h == 0;
            if (g == 0 && h == 0) wait(sh.v_full + (tile & 1), tile >> 1);
            wait(sh.p_full + b, turn);
            if (first && segs[g]) wait(sh.o_free + g, segs[g] - 1);
            kt_fence_after();
            __syncwarp();
            if (kt_elect()) {
                const uint32_t from = tm + (GROUPS == 2 ? g * 128 + h * 64 + 32 : b * 128 + S::P);
#pragma unroll
                for (int k = 0; k < K4_TILE / 16 / (int)HALVES; ++k)
                    kt_mma(tm + S::O + g * HD, from + 8 * k, vs + (((tile & 1) * S::TILE + h * 8192 + k * 2048) >> 4), kt_idesc(HD, true), !first || k);
                if (last_group && h + 1 == HALVES) kt_commit(sh.v_empty + (tile & 1));
                kt_commit(sh.o_done + b);
            }
            __syncwarp();
            if (h + 1 == HALVES) ++valued[g];
            if (first) ++segs[g];
        };
        while (const Kv8Segment *s = next()) {
            wait(sh.q_full + seg % SEGS, seg / SEGS);
            const int tiles = s->t1 - s->t0;
            const int nrows = min((int)A.row_tile, s->q.rows - s->row_tile * (int)A.row_tile) * (int)GR;
            const bool two = GROUPS == 2 && nrows > 128;
            if constexpr (GROUPS == 1) {
                // scores a tile ahead of values
                ask(0, 0, true, tiles == 1);
#pragma unroll 1
                for (int t = 0; t < tiles; ++t) {
                    if (t + 1 < tiles) ask(0, t + 1, true, t + 2 == tiles);
                    give(0, 0, t, true);
                }
            } else {
                // P takes the place of scores, so a group's next scores come after all its values; the other group is half a
                // tile behind, so one's products run while the other's weights are made
                ask(0, 0, !two, tiles == 1);
                if (two) ask(1, 0, true, tiles == 1);
#pragma unroll 1
                for (int t = 0; t < tiles; ++t) {
                    give(0, 0, t, !two);
                    if (two && t) {
                        give(1, 1, t - 1, true);
                        ask(1, t, true, t + 1 == tiles);
                    }
                    give(0, 1, t, !two);
                    if (t + 1 < tiles) ask(0, t + 1, !two, t + 2 == tiles);
                    if (two) give(1, 0, t, true);
                }
                if (two) give(1, 1, tiles - 1, true);
            }
            n += (unsigned)tiles;
            done();
        }
        if (kt_elect()) {
            kt_commit(&sh.drained);
            mbar_wait_bounded(&sh.drained, 0);
        }
        __syncwarp();
    }
    kt_fence_before();
    __syncthreads();
    if (tid == 0 && *dead) raise_error(A.error, ERR_TIMEOUT);
    if (warp == W_MMA) {
        kt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
    }
}

template <int HD, int NR>
int kv4_tiles_go(const Kv4Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned grid, cudaStream_t s)
{
    constexpr size_t smem = 1024 + K4tShape<HD, NR>::OFF_END + sizeof(K4tShared<NR>);
    static_assert(smem <= 227 * 1024, "shared memory of one CTA");
    static std::atomic<unsigned> allowed{0};
    if (allow_shared((const void *)kv4_tiles_kernel<HD, NR>, smem, allowed)) return -2;
    kv4_tiles_kernel<HD, NR><<<grid, k4t_threads(NR), smem, s>>>(A, k, v);
    if constexpr (NR == 256) kv4_join_kernel<HD, NR><<<dim3(grid, NR / 32), K4T_JOIN, 0, s>>>(A);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace fyb
