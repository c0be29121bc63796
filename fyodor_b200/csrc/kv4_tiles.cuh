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
// P lies in the upper half of its S. Row tiles of 128 rows (prompt chunks): two
// groups of softmax warps take tiles in turn, each with maxima, sums and O of its own.
// Row tiles of 64 or 32 rows (drafts): the lanes hold two or four copies of the rows,
// and copy c takes the positions of its part of a tile, its P being 0 elsewhere: every
// thread has positions to do, and what the copies hold is joined like any parts. One
// group and one O leave room for q in tensor memory, which saves its reads and its
// place in shared memory.
//
// The maximum m of a row moves only when a score is more than 2^8 above it.
#pragma once
#include "kv4_attention.cuh"
#include "kt_mma.cuh"

namespace fyb {

constexpr int K4T_CONV = 4, K4T_META = 8, K4T_SEGS = 4;
FYB_HOST_DEV constexpr int k4t_groups(int NR) { return NR == 128 ? 2 : 1; }      // groups of four softmax warps
FYB_HOST_DEV constexpr int k4t_threads(int NR) { return 32 * (4 * k4t_groups(NR) + 2 * K4T_CONV + 2); }

template <int HD, int NR> struct K4tShape {
    static constexpr int ROW = HD / 2, SCALES = HD / 64 * 4;                 // bytes of a token's row, of its scales
    static constexpr int RAW_V = K4_TILE * ROW, RAW_KS = 2 * RAW_V, RAW_VS = RAW_KS + K4_TILE * SCALES,
                         RAW = RAW_VS + K4_TILE * SCALES, STAGES = HD == 64 || NR < 128 ? 4 : 2;
    static constexpr int HALF = 128 * 128, TILE = HD / 64 * HALF;             // fp16 rows of 64 values in 128 bytes
    static constexpr int O_STRIDE = 20;                                       // floats between lanes of 16 columns of O on their way out
    static constexpr bool Q_TM = NR < 128;                                    // q in tensor memory
    static constexpr int OFF_K = 0, OFF_V = 2 * TILE, OFF_Q = 4 * TILE, OFF_RAW = (Q_TM ? 4 : 5) * TILE, OFF_O = OFF_RAW + STAGES * RAW,
                         OFF_END = OFF_O + k4t_groups(NR) * 128 * O_STRIDE * 4;
    // tensor memory columns: S of two tiles with P in the upper half, O of each group, q
    static constexpr int P = 64, O = 256, Q = 256 + HD;
};
template <int NR> struct K4tShared {
    Kv8Segment seg[K4T_SEGS], walked[k4t_threads(NR) / 32];
    Kv8Place place;
    uint64_t seg_full[K4T_SEGS], seg_empty[K4T_SEGS], raw_full[4], raw_empty[4], k_full[2], k_empty[2], v_full[2], v_empty[2],
        s_full[2], p_full[2], o_done[2], o_free[2], q_full[K4T_SEGS], q_empty, meta_full[K4T_META], drained;
    float factor[K4T_SEGS][128];                 // score factor of each lane's row
    float2 ml[k4t_groups(NR) * 128], joined[NR];
    unsigned here[K4T_META], raw_here[4];        // which groups of 16 positions are loaded, by tile and by stage
    uint32_t tmem;
    unsigned flag, dead;
};

static __device__ __noinline__ void k4t_segment(const Kv4Attention &A, const Kv8Place &place, unsigned k, Kv8Segment *s)
{
    Kv8Walk<K4_TILE> walk(A, place);
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

// Eight values of a query row of 16 bits; vec: in one access.
FYB_DEV void k4t_load8(const Kv4Attention &A, size_t at, float4 &a, float4 &b)
{
    if (A.vec) {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(static_cast<const unsigned short *>(A.q) + at));
        auto two = [&](unsigned w) {
            return A.type == T_F16 ? kt_unpack(w) : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        };
        const float2 p = two(u.x), q = two(u.y), r = two(u.z), s = two(u.w);
        a = make_float4(p.x, p.y, q.x, q.y);
        b = make_float4(r.x, r.y, s.x, s.y);
    } else {
        a = kv8_load4(A.q, A.type, at);
        b = kv8_load4(A.q, A.type, at + 4);
    }
}

template <int HD, int NR>
__global__ void __launch_bounds__(k4t_threads(NR), 1) kv4_tiles_kernel(const __grid_constant__ Kv4Attention A, const __grid_constant__ CUtensorMap kmap,
    const __grid_constant__ CUtensorMap vmap)
{
    using S = K4tShape<HD, NR>;
    constexpr unsigned GROUPS = k4t_groups(NR), SOFT = 4 * GROUPS, W_CONV = SOFT, W_TMA = SOFT + 2 * K4T_CONV, W_MMA = W_TMA + 1;
    constexpr unsigned CP = 128 / NR, CW = 128 / CP, CHUNKS = CW / 32;   // copies, and the positions and blocks of 32 of a copy
    constexpr int G64 = HD / 64;
    extern __shared__ unsigned char k4t_smem[];
    unsigned char *ring = k4t_smem + ((1024u - (smem_u32(k4t_smem) & 1023u)) & 1023u);
    K4tShared<NR> &sh = *reinterpret_cast<K4tShared<NR> *>(ring + S::OFF_END);
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), kv = A.c.kv_heads, GR = A.group;
    if (tid == 0) {
        for (int i = 0; i < S::STAGES; ++i) { mbar_init(sh.raw_full + i, 1); mbar_init(sh.raw_empty + i, 2 * K4T_CONV); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(sh.k_full + i, K4T_CONV); mbar_init(sh.k_empty + i, 1);
            mbar_init(sh.v_full + i, K4T_CONV); mbar_init(sh.v_empty + i, 1);
            mbar_init(sh.s_full + i, 1); mbar_init(sh.p_full + i, 4);
            mbar_init(sh.o_done + i, 1); mbar_init(sh.o_free + i, 4);
        }
        mbar_init(&sh.q_empty, 1); mbar_init(&sh.drained, 1);
        for (int i = 0; i < K4T_META; ++i) mbar_init(sh.meta_full + i, 1);
        for (int i = 0; i < K4T_SEGS; ++i) { mbar_init(sh.q_full + i, K4T_CONV); mbar_init(sh.seg_full + i, 1); mbar_init(sh.seg_empty + i, SOFT + 2 * K4T_CONV + 1); }
        sh.dead = 0;
        fence_barrier_init();
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    kt_fence_before();
    {
        const Kv8Place place = kv8_place<K4_TILE, k4t_threads(NR), 2>(A);  // CTA barriers inside
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
        wait(sh.seg_full + seg % K4T_SEGS, seg / K4T_SEGS);
        const Kv8Segment *s = sh.seg + seg % K4T_SEGS;
        if (__builtin_expect(*dead, 0)) {
            s = sh.walked + warp;
            if (lane == 0) k4t_segment(A, sh.place, seg, sh.walked + warp);
            __syncwarp();
        }
        return s->t1 ? s : nullptr;
    };
    auto done = [&] { arrive(sh.seg_empty + seg % K4T_SEGS); ++seg; };

    if (warp < SOFT) {
        // ================================================== softmax
        const unsigned wg = warp >> 2, at = tid & 127, rho = at % NR, first = at / NR * CW;  // lane of tensor memory; its row and first position of a tile
        const uint32_t lanes = (warp & 3) << 21;
        const uint32_t o_at = tmem + lanes + S::O + wg * HD;
        float *stage = reinterpret_cast<float *>(ring + S::OFF_O);
        auto bar = [] { asm volatile("bar.sync 1, %0;" :: "n"(32 * SOFT) : "memory"); };
        constexpr float P_UP = 6.f;  // weights are 2^6 times themselves, clear of fp16's smallest numbers; the largest is 2^14
        while (const Kv8Segment *sp = next()) {
            const Kv8Segment &s = *sp;
            const int t0 = s.t0, t1 = s.t1, j0 = s.row_tile * (int)A.row_tile;
            const int nrows = min((int)A.row_tile, s.q.rows - j0) * (int)GR;
            const int limit = (int)rho < nrows ? s.q.len - s.q.n + j0 + (int)(rho / GR) + 1 : 0;  // positions the row attends
            const int all = max(0, s.q.len - s.q.n + j0 + 1);                                      // positions every row attends
            wait(sh.q_full + seg % K4T_SEGS, seg / K4T_SEGS);
            const float f = sh.factor[seg % K4T_SEGS][at];
            float m = -3.4e38f, l = 0.f;   // m: the maximum less P_UP
            unsigned mine = 0;             // tiles of this group so far
            for (int t = t0; t < t1; ++t, ++n) {
                const unsigned b = n & 1;
                if (GROUPS == 2 && b != wg) continue;
                wait(sh.meta_full + n % K4T_META, n / K4T_META);
                const unsigned here = sh.here[n % K4T_META];
                wait(sh.s_full + b, n >> 1);
                kt_fence_after();
                const uint32_t s_at = tmem + lanes + b * 128 + first, p_at = tmem + lanes + b * 128 + S::P;
                if (__builtin_expect(here != 0xffu || (t + 1) * K4_TILE > all, 0)) {
                    // what the row does not attend becomes -inf where it lies: the rest has one form, and fits the
                    // instruction cache with the other roles
#pragma unroll 1
                    for (unsigned c = 0; c < CW; c += 16) {
                        float y[16];
                        kt_ld16(s_at + c, y);
                        kt_wait_ld();
                        const int left = here >> ((first + c) / 16) & 1 ? limit - (t * K4_TILE + (int)(first + c)) : 0;
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[i] = i < left ? y[i] : -INFINITY;
                        kt_st16(s_at + c, y);
                    }
                    kt_wait_st();
                }
                constexpr unsigned KEEP = CHUNKS < 2 ? CHUNKS : 2;  // blocks that stay in registers between the two looks at them
                float x[KEEP][32], tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (unsigned c = 0; c < CHUNKS; c += KEEP) {
#pragma unroll
                    for (unsigned k = 0; k < KEEP; ++k) kt_ld32(s_at + 32 * (c + k), x[k]);
                    kt_wait_ld();
#pragma unroll
                    for (unsigned k = 0; k < KEEP; ++k)
#pragma unroll
                        for (int i = 0; i < 32; i += 2) tops[i / 2 % 4] = fmaxf(tops[i / 2 % 4], fmaxf(x[k][i], x[k][i + 1]));
                }
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * f;
                const bool up = top - m > 8.f + P_UP;
                if (__any_sync(0xffffffffu, up)) {
                    // ---- new maxima, and the sums so far in their units
                    const float now = up ? top - P_UP : m, alpha = up ? ex2(m - now) : 1.f;
                    m = now;
                    l *= alpha;
                    if (mine) {
                        if (GROUPS == 2) wait(sh.o_done + b, (n >> 1) - 1); else wait(sh.o_done + (b ^ 1), (n - 1) >> 1);
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
                // ---- weights, blocks from the last to the first: P takes the place of scores that have been read
                const F2 f2x = f2(f, f), mx = f2(-m, -m);
                F2 sums[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
                auto weights = [&](float (&y)[32], unsigned c) {
                    unsigned w[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 e = f2_get(f2_fma(f2(y[i], y[i + 1]), f2x, mx));
                        const float p0 = ex2(e.x), p1 = ex2(e.y);
                        sums[i / 2 % 2] = f2_add(sums[i / 2 % 2], f2(p0, p1));
                        w[i / 2] = kt_pack(p0, p1);
                    }
                    kt_st16(p_at + first / 2 + 16 * c, reinterpret_cast<const float *>(w));
                };
                if constexpr (CP > 1) {  // 0 for the positions of the other copies
                    float z[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[i] = 0.f;
#pragma unroll
                    for (unsigned c = 0; c < 64; c += 16)
                        if (c < first / 2 || c >= (first + CW) / 2) kt_st16(p_at + c, z);
                }
#pragma unroll
                for (unsigned c = CHUNKS; c; c -= KEEP) {
                    if (c != CHUNKS) {
#pragma unroll
                        for (unsigned k = 0; k < KEEP; ++k) kt_ld32(s_at + 32 * (c - KEEP + k), x[k]);
                        kt_wait_ld();
                    }
#pragma unroll
                    for (unsigned k = KEEP; k; --k) weights(x[k - 1], c - KEEP + k - 1);
                }
                const float2 l2 = f2_get(f2_add(sums[0], sums[1]));
                l += l2.x + l2.y;
                kt_wait_st();
                kt_fence_before();
                arrive(sh.p_full + b);
                ++mine;
            }
            // ---- the segment's part: what copies and groups hold of a row, joined
            if (mine) {
                const unsigned last = n - 1 - (GROUPS == 2 && ((n - 1) & 1) != wg ? 1 : 0);
                wait(sh.o_done + (last & 1), last >> 1);
            }
            kt_fence_after();
            sh.ml[tid] = make_float2(m, l);
            bar();
            const bool whole = s.t0 == 0 && s.t1 == s.tiles;
            constexpr unsigned PARTS = GROUPS * CP;
            float own;
            {
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (unsigned p = 0; p < PARTS; ++p) top = fmaxf(top, sh.ml[p * NR + rho].x);
#pragma unroll
                for (unsigned p = 0; p < PARTS; ++p) {
                    const float2 y = sh.ml[p * NR + rho];
                    sum = fmaf(y.y, ex2(y.x - top), sum);
                }
                own = ex2(m - top);
                if (whole) own *= sum > 0.f || isnan(sum) ? 1.f / sum : 0.f;
                if (tid < NR) sh.joined[rho] = make_float2(top, sum);
            }
            const Kv8Parts of = kv8_parts(s, sh.place);
            auto put = [&](unsigned row, unsigned chunk, float4 v) {
                const size_t r = (size_t)(s.q.first + j0 + (int)(row / GR));
                kv8_store4(A.out, A.type, r * A.out_stride + (size_t)(s.head * GR + row % GR) * HD + 4 * chunk, v);
            };
#pragma unroll 1
            for (unsigned c = 0; c < HD; c += 16) {
                float y[16];
                if (mine) {
                    kt_ld16(o_at + c, y);
                    kt_wait_ld();
                }
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4 *>(stage + tid * S::O_STRIDE + i) = mine ? make_float4(y[i] * own, y[i + 1] * own, y[i + 2] * own, y[i + 3] * own)
                                                                                      : make_float4(0.f, 0.f, 0.f, 0.f);
                bar();
                for (unsigned i = tid; i < (unsigned)nrows * 2; i += 32 * SOFT) {
                    const unsigned row = i >> 1, half = i & 1;
                    float z[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[j] = 0.f;
#pragma unroll
                    for (unsigned p = 0; p < PARTS; ++p)
#pragma unroll
                        for (int j = 0; j < 8; j += 4) {
                            const float4 u = *reinterpret_cast<const float4 *>(stage + (p * NR + row) * S::O_STRIDE + 8 * half + j);
                            z[j] += u.x; z[j + 1] += u.y; z[j + 2] += u.z; z[j + 3] += u.w;
                        }
                    const float4 lo = make_float4(z[0], z[2], z[4], z[6]), hi = make_float4(z[1], z[3], z[5], z[7]);
                    const unsigned chunk = (c + 8 * half) / 4;
                    if (whole) {
                        put(row, chunk, lo);
                        put(row, chunk + 1, hi);
                    } else {
                        float4 *o = reinterpret_cast<float4 *>(A.part_o + ((size_t)of.slot * NR + row) * HD);
                        o[chunk] = lo;
                        o[chunk + 1] = hi;
                    }
                }
                bar();
            }
            kt_fence_before();
            arrive(sh.o_free + wg);
            if (!whole) {
                if ((int)tid < nrows) A.part_ml[(size_t)of.slot * NR + tid] = sh.joined[tid];
                kv8_arrive<NR, HD, 32 * SOFT>(A, of, tid, (unsigned)nrows, stage, GROUPS * 128 * S::O_STRIDE, &sh.flag, bar, put);
                bar();
            }
            done();
        }
    } else if (warp < W_TMA) {
        // ================================================== K or V, 4 bits to fp16 rows; q
        const bool is_v = warp >= W_CONV + K4T_CONV;
        const unsigned cw = (warp - W_CONV) % K4T_CONV, ct = cw * 32 + lane;
        const unsigned j = lane & 7, tok0 = cw * 32 + (lane >> 3);  // eight lanes a token, a warp 32 tokens
        while (const Kv8Segment *sp = next()) {
            const Kv8Segment &s = *sp;
            const int any = kv8_attended(A, s.q, s.row_tile), t0 = s.t0, t1 = s.t1;
            if (!is_v) {
                // ---- q rows by a power of two each. The score factor's sign goes with q: a row's largest product is its
                // largest score
                const int j0 = s.row_tile * (int)A.row_tile, nrows = min((int)A.row_tile, s.q.rows - j0) * (int)GR;
                auto at_of = [&](unsigned rho) {
                    return (size_t)(s.q.first + j0 + (int)(rho / GR)) * A.q_stride + (size_t)(s.head * GR + rho % GR) * HD;
                };
                auto size_of = [](float4 a) { return fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))); };
                auto halves = [&](float4 a, float4 b, int e) {
                    const float up = copysignf(kt_power(min(e, 127)), A.scale), up2 = kt_power(e - min(e, 127));
                    auto pair = [&](float y, float z) { return kt_pack(y * up * up2, z * up * up2); };
                    return make_uint4(pair(a.x, b.x), pair(a.y, b.y), pair(a.z, b.z), pair(a.w, b.w));
                };
                // at least the smallest normal number: -inf times it stays -inf
                auto factor_of = [&](int e) { return fmaxf(ldexpf(fabsf(A.scale), -e), 1.17549435e-38f); };
                if constexpr (S::Q_TM) {
                    // to tensor memory, a thread a lane's row
                    const unsigned rho = ct % NR;
                    const bool real = (int)rho < nrows;
                    const size_t at = at_of(real ? rho : 0);
                    float top = 0.f;
                    if (real) {
#pragma unroll 8
                        for (int i = 0; i < HD; i += 8) {
                            float4 a, b;
                            k4t_load8(A, at + i, a, b);
                            top = fmaxf(top, fmaxf(size_of(a), size_of(b)));
                        }
                    }
                    const int e = 12 - kt_exponent(top);
                    if (seg) wait(&sh.q_empty, seg - 1);  // the last segment's products have read their q
                    kt_fence_after();
#pragma unroll 2
                    for (int i = 0; i < HD; i += 32) {
                        uint4 h[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
                            if (real) k4t_load8(A, at + i + 8 * u, a, b);
                            h[u] = halves(a, b, e);
                        }
                        kt_st16(tmem + (cw << 21) + S::Q + i / 2, reinterpret_cast<const float *>(h));
                    }
                    kt_wait_st();
                    sh.factor[seg % K4T_SEGS][ct] = factor_of(e);
                    kt_fence_before();
                } else {
                    // to shared memory, eight values a lane
                    constexpr unsigned LANES = HD / 8, STEP = 32 / LANES, STEPS = NR / K4T_CONV / STEP, AHEAD = 4;  // lanes of a row, rows of a load
                    const unsigned piece = lane % LANES;
#pragma unroll 1
                    for (unsigned i = 0; i < STEPS; i += AHEAD) {
                        float4 x[AHEAD][2];
#pragma unroll
                        for (unsigned u = 0; u < AHEAD; ++u) {
                            const unsigned rho = (cw * STEPS + i + u) * STEP + lane / LANES;
                            x[u][0] = x[u][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if ((int)rho < nrows) k4t_load8(A, at_of(rho) + 8 * piece, x[u][0], x[u][1]);
                        }
                        if (seg && i == 0) wait(&sh.q_empty, seg - 1);  // the last segment's products have read their q
#pragma unroll
                        for (unsigned u = 0; u < AHEAD; ++u) {
                            const unsigned rho = (cw * STEPS + i + u) * STEP + lane / LANES;
                            const int e = 12 - kt_exponent(group_max<LANES>(fmaxf(size_of(x[u][0]), size_of(x[u][1]))));
                            *reinterpret_cast<uint4 *>(ring + S::OFF_Q + piece / 8 * S::HALF + rho * 128 + ((piece % 8 ^ (rho & 7u)) << 4)) =
                                halves(x[u][0], x[u][1], e);
                            if (piece == 0) sh.factor[seg % K4T_SEGS][rho] = factor_of(e);
                        }
                    }
                }
                fence_proxy_async();
                arrive(sh.q_full + seg % K4T_SEGS);
            }
            for (int t = t0; t < t1; ++t, ++n) {
                const unsigned b = n & 1, st = n % S::STAGES;
                wait(sh.raw_full + st, n / S::STAGES);
                if (n >= 2) wait((is_v ? sh.v_empty : sh.k_empty) + b, (n >> 1) - 1);
                const unsigned char *raw = ring + S::OFF_RAW + st * S::RAW + (is_v ? S::RAW_V : 0);
                const unsigned char *scales = ring + S::OFF_RAW + st * S::RAW + (is_v ? S::RAW_VS : S::RAW_KS);
                unsigned char *dst = ring + (is_v ? S::OFF_V : S::OFF_K) + b * S::TILE;
                // V of positions that no row attends, or never loaded, is 0 and not what lies there (a NaN stays one times 0)
                const unsigned here = sh.raw_here[st];
                const bool patchy = is_v && (here != 0xffu || any < (t + 1) * K4_TILE);
                // four tokens' words and scales at a time, before the first of their stores (which they might overlap, as
                // far as the compiler can tell: a token after the other took 1500 cycles a tile)
#pragma unroll
                for (unsigned i0 = 0; i0 < 8; i0 += 4) {
                    unsigned w[4][G64], sc[4][G64];
#pragma unroll
                    for (unsigned i = 0; i < 4; ++i) {
                        const unsigned tok = tok0 + 4 * (i0 + i);
                        if constexpr (G64 == 2) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(raw + tok * 64 + ((8 * j) ^ ((tok >> 1 & 3) << 4)));
                            const uint2 y = *reinterpret_cast<const uint2 *>(scales + tok * 8);
                            w[i][0] = x.x; w[i][1] = x.y;
                            sc[i][0] = y.x; sc[i][1] = y.y;
                        } else {
                            w[i][0] = *reinterpret_cast<const unsigned *>(raw + tok * 32 + 4 * j);
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
                arrive(sh.raw_empty + st);
                fence_proxy_async();
                arrive((is_v ? sh.v_full : sh.k_full) + b);
            }
            done();
        }
    } else if (warp == W_TMA) {
        // ================================================== TMA
        const unsigned size = 1u << A.shift, box = min(size, (unsigned)K4_TILE), per = K4_TILE / box;
        __syncwarp();
        Kv8Walk<K4_TILE> walk(A, sh.place);
        Kv8Segment s;
        for (;; ++seg) {
            const bool more = walk.next(s);
            if (seg >= K4T_SEGS) wait(sh.seg_empty + seg % K4T_SEGS, seg / K4T_SEGS - 1);
            if (lane == 0 && !*dead) {
                if (more) sh.seg[seg % K4T_SEGS] = s; else sh.seg[seg % K4T_SEGS].t1 = 0;
                mbar_arrive(sh.seg_full + seg % K4T_SEGS);
            }
            __syncwarp();
            if (!more) break;
            const int blocks = (kv8_attended(A, s.q, s.row_tile) + (int)size - 1) >> A.shift;
            const int *ids = A.table + (size_t)s.request * A.table_stride;
            int have = -1, id = 0;  // lane holds block 32 * have + lane
            for (int t = s.t0; t < s.t1; ++t, ++n) {
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
                const unsigned st = n % S::STAGES;
                if (n >= S::STAGES) wait(sh.raw_empty + st, n / S::STAGES - 1);
                const int own = __shfl_sync(0xffffffffu, id, (b0 & 31) + (int)(lane % per));
                const bool load = lane < per && own >= 0;
                const unsigned boxes = __ballot_sync(0xffffffffu, load);
                // groups of 16 positions whose block is among the loaded ones
                const unsigned groups = __ballot_sync(0xffffffffu, lane < K4_TILE / 16 && (boxes >> (lane * 16 / box) & 1));
                if (lane == 0) {
                    sh.here[n % K4T_META] = groups;
                    sh.raw_here[st] = groups;
                    mbar_arrive(sh.meta_full + n % K4T_META);
                    if (boxes) mbar_expect_tx(sh.raw_full + st, __popc(boxes) * 2 * box * (S::ROW + S::SCALES)); else mbar_arrive(sh.raw_full + st);
                }
                __syncwarp();
                if (load && !*dead) {
                    const unsigned row = (((unsigned)own * kv + s.head) << A.shift) + ((unsigned)(t * K4_TILE) & (size - 1));
                    unsigned char *dst = ring + S::OFF_RAW + st * S::RAW;
                    tma_load_rows(dst + lane * box * S::ROW, &kmap, (int)row, sh.raw_full + st);
                    tma_load_rows(dst + S::RAW_V + lane * box * S::ROW, &vmap, (int)row, sh.raw_full + st);
                    bulk_copy_g2s(dst + S::RAW_KS + lane * box * S::SCALES, A.ks + (size_t)row * G64, box * S::SCALES, sh.raw_full + st);
                    bulk_copy_g2s(dst + S::RAW_VS + lane * box * S::SCALES, A.vs + (size_t)row * G64, box * S::SCALES, sh.raw_full + st);
                }
                __syncwarp();
            }
        }
        if (*dead) {  // copies in flight land before the CTA leaves its shared memory
            for (unsigned i = 0; i < min(n, (unsigned)S::STAGES); ++i) {
                const unsigned k = n - 1 - i;
                mbar_wait_bounded(sh.raw_full + k % S::STAGES, k / S::STAGES & 1);
            }
        }
    } else {
        // ================================================== MMA
        // The warp runs as one and an elected lane issues: operands then sit in uniform registers.
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t qs = kt_desc(smem_u32(ring + S::OFF_Q), 16), ks = kt_desc(smem_u32(ring + S::OFF_K), 16),
                       vs = kt_desc(smem_u32(ring + S::OFF_V), S::HALF);
        unsigned at = 0;  // tiles whose scores have been asked for
        auto scores = [&](bool last) {
            const unsigned b = at & 1;
            wait(sh.k_full + b, at >> 1);
            if (at >= 2) wait(sh.o_done + b, (at >> 1) - 1);  // P of the tile before the last, in this S, has been read
            kt_fence_after();
            __syncwarp();
            if (kt_elect()) {
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const uint64_t step = (uint64_t)((k / 4 * S::HALF + k % 4 * 32) >> 4);
                    if constexpr (S::Q_TM) kt_mma(tm + b * 128, tm + S::Q + 8 * k, ks + (b * S::TILE >> 4) + step, kt_idesc(128, false), k > 0);
                    else kt_mma_ss(tm + b * 128, qs + step, ks + (b * S::TILE >> 4) + step, kt_idesc(128, false), k > 0);
                }
                kt_commit(sh.k_empty + b);
                kt_commit(sh.s_full + b);
                if (last) kt_commit(&sh.q_empty);
            }
            __syncwarp();
            ++at;
        };
        while (const Kv8Segment *s = next()) {
            wait(sh.q_full + seg % K4T_SEGS, seg / K4T_SEGS);
            const int tiles = s->t1 - s->t0;
            unsigned begun = 0;  // groups whose O of this segment holds something
#pragma unroll 1
            for (int t = -1; t < tiles; ++t) {  // scores one tile ahead of values
                if (t + 1 < tiles) scores(t + 2 == tiles);
                if (t < 0) continue;
                const unsigned b = n & 1, g = GROUPS == 2 ? b : 0;
                wait(sh.v_full + b, n >> 1);
                wait(sh.p_full + b, n >> 1);
                if (!(begun >> g & 1) && seg) wait(sh.o_free + g, seg - 1);
                kt_fence_after();
                __syncwarp();
                if (kt_elect()) {
#pragma unroll
                    for (int k = 0; k < K4_TILE / 16; ++k)
                        kt_mma(tm + S::O + g * HD, tm + b * 128 + S::P + 8 * k, vs + ((b * S::TILE + k * 2048) >> 4),
                               kt_idesc(HD, true), (begun >> g & 1) || k);
                    kt_commit(sh.v_empty + b);
                    kt_commit(sh.o_done + b);
                }
                __syncwarp();
                begun |= 1u << g;
                ++n;
            }
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
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace fyb
