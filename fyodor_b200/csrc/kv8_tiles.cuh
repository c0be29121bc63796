// kv8_tiles.cuh - attention over the paged 8-bit cache for many query rows per
// KV head (drafts, prompt chunks), on the 5th-generation tensor cores. One
// instantiation per head dimension and format (kv8_tiles_inst.cu).
//
// Per tile of 128 positions, N = 32 or 64 query rows of one KV head:
//
//   D1[position][row] = K Q^T       tcgen05.mma kind::f16, M = 128, K = head_dim
//   P = 2^(D1 scale - m) v_scale    one thread per position and half the rows
//   D2[hd][row] += V^T P^T          M = 128, K = 128 positions
//
// K and V come as 8-bit tiles by TMA and are converted to fp16 in shared memory
// (exact); both products read the converted tile as it lies, [position][hd] in
// 128-byte swizzled rows: K as a K-major, V as an M-major operand. The weights,
// and q of F32 rows, are two fp16 halves hi + lo (22 bits, an MMA each); q of
// 16-bit rows is one half, which holds it (a bf16 value 2^24 below its tile's
// largest loses bits that no score shows). Row sums, maxima and accumulators
// are F32.
//
// The maximum m of a row moves only when a score is more than 2^8 above it, so
// D2 stays in tensor memory across tiles and is rescaled a few times a segment.
//
// Roles: warps 0-7 softmax (two groups of four, a group takes half the rows),
// 8-11 conversion and q, 12 TMA, 13 MMA. Per tile at N = 64 the softmax issues
// about 9 instructions a score, 580 cycles; the conversions 380; the MMAs of F32
// rows 1024, of 16-bit rows 768; the tile's bytes pass an SM in 1480 cycles.
#pragma once
#include "kv8_attention.cuh"

namespace fyb {

constexpr int KT_TILE = 128, KT_SOFT = 8, KT_CONV = 4, KT_THREADS = 32 * (KT_SOFT + KT_CONV + 2), KT_META = 8;

// ---- tcgen05 -------------------------------------------------------------------
// Operand in 128-byte swizzled rows, eight-row groups 1024 bytes apart. K-major:
// a row is 64 K values of one M/N index. M/N-major: a row is 64 M/N values of one
// K index, `lead` bytes to the next 64.
FYB_DEV uint64_t kt_desc(unsigned addr, unsigned lead)
{
    return (uint64_t)(addr >> 4 & 0x3FFFu) | (uint64_t)(lead >> 4) << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61;
}
// F32 accumulator, fp16 operands, M = 128; mn: both operands M/N-major
FYB_HOST_DEV constexpr uint32_t kt_idesc(unsigned N, bool mn)
{
    return 1u << 4 | (mn ? 3u << 15 : 0u) | N >> 3 << 17 | 128u >> 4 << 24;
}
FYB_DEV void kt_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
FYB_DEV void kt_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 :: "r"(smem_u32(bar)) : "memory");
}
FYB_DEV void kt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
FYB_DEV void kt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 16 consecutive columns of this thread's TMEM lane
FYB_DEV void kt_ld16(uint32_t addr, float *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
                   "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
                 : "r"(addr) : "memory");
}
FYB_DEV void kt_st16(uint32_t addr, const float *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 :: "r"(addr), "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]),
                    "f"(r[8]), "f"(r[9]), "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15])
                 : "memory");
}
FYB_DEV void kt_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
FYB_DEV void kt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

FYB_DEV unsigned kt_pack(float lo, float hi)  // fp16 pair
{
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned *>(&p);
}
FYB_DEV float2 kt_unpack(unsigned p) { return __half22float2(*reinterpret_cast<const __half2 *>(&p)); }
FYB_DEV int kt_exponent(float x) { return x > 0.f ? max(-126, (int)(__float_as_uint(x) >> 23) - 127) : 0; }
FYB_DEV float kt_power(int e) { return e < -126 ? __uint_as_float(1u << max(0, e + 149)) : __uint_as_float((unsigned)(min(e, 127) + 127) << 23); }

template <int HD, int N, int QP> struct KtShape {
    static constexpr int STAGE = KT_TILE * HD, F16 = KT_TILE * 256;  // an 8-bit tile; a converted one (128 values a row)
    static constexpr int QB = N * HD * 2, PB = KT_TILE * 128;        // one half of q; one half of P
    static constexpr int P_STAGES = QP * N * HD < 16384 ? 2 : 1;  // what fits
    static constexpr int OFF_K8 = 0, OFF_V8 = OFF_K8 + 2 * STAGE, OFF_KF = OFF_V8 + 2 * STAGE, OFF_VF = OFF_KF + F16,
                         OFF_Q = OFF_VF + F16, OFF_P = OFF_Q + QP * QB, OFF_END = OFF_P + P_STAGES * 2 * PB;
};
template <int N> struct KtShared {
    float ks[KT_META][KT_TILE / 16], vs[KT_META][KT_TILE / 16];  // scales by 16 positions; ks NaN: not loaded
    float m[N], own[N], top[4][N], sum[4][N];
    int limit[N];                                                 // positions a row attends
    float2 ml[N];
    float factor[2], row_factor[2][N], q_top[KT_CONV];            // score factors: of the tile's q, and beside it of a row
    int uneven[2];                                                // whether some row has a factor of its own
    uint64_t k8_full[2], k8_empty[2], v8_full[2], v8_empty[2], kf_full, kf_empty, vf_full, d1_full[2], d1_empty[2],
        p_full[2], o_done[2], q_full[2], q_empty[2], meta_full[KT_META], drained;
    uint32_t tmem;
    unsigned flag, dead;
};

template <int HD, unsigned FMT, int N, int QP>
__global__ void __launch_bounds__(KT_THREADS, 1) kv8_tiles_kernel(Kv8Attention A, const __grid_constant__ CUtensorMap kmap,
    const __grid_constant__ CUtensorMap vmap)
{
    using S = KtShape<HD, N, QP>;
    constexpr int C = N / 2, TM = N == 64 ? 256 : 128;  // columns of a softmax thread; TMEM columns
    constexpr int KH = HD / 64;
    extern __shared__ unsigned char kt_smem[];
    unsigned char *ring = kt_smem + ((1024u - (smem_u32(kt_smem) & 1023u)) & 1023u);
    KtShared<N> &sh = *reinterpret_cast<KtShared<N> *>(ring + S::OFF_END);
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kv = A.c.kv_heads, G = A.group;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(sh.k8_full + i, 1); mbar_init(sh.k8_empty + i, KT_CONV);
            mbar_init(sh.v8_full + i, 1); mbar_init(sh.v8_empty + i, KT_CONV);
            mbar_init(sh.d1_full + i, 1); mbar_init(sh.d1_empty + i, KT_SOFT);
            mbar_init(sh.p_full + i, KT_SOFT); mbar_init(sh.o_done + i, 1);
            mbar_init(sh.q_full + i, KT_CONV); mbar_init(sh.q_empty + i, KT_SOFT);
        }
        mbar_init(&sh.kf_full, KT_CONV); mbar_init(&sh.kf_empty, 1); mbar_init(&sh.vf_full, KT_CONV);
        for (int i = 0; i < KT_META; ++i) mbar_init(sh.meta_full + i, 1);
        mbar_init(&sh.drained, 1);
        sh.dead = 0;
        fence_barrier_init();
    }
    if (warp == KT_SOFT + KT_CONV + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&sh.tmem)), "r"(TM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (KH == 1)  // head_dim 64: the upper 64 rows of D2 come from zeros
        for (unsigned i = tid; i < S::F16 / 2 / 16; i += KT_THREADS)
            reinterpret_cast<uint4 *>(ring + S::OFF_VF + S::F16 / 2)[i] = make_uint4(0, 0, 0, 0);
    kt_fence_before();
    const Kv8Place place = kv8_place<KT_TILE, KT_THREADS>(A);  // CTA barriers inside
    kt_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem, d2 = tmem + 2 * N;
    Kv8Walk<KT_TILE> walk(A, place);
    Kv8Segment s;
    unsigned n = 0;  // tiles of this CTA so far
    volatile unsigned *dead = &sh.dead;  // a wait ran out: nobody waits any more, the error word is set
    auto wait = [&](uint64_t *bar, unsigned parity) {
        if (*dead || mbar_wait_bounded(bar, parity & 1)) return;
        *dead = 1;
        raise_error(A.error, ERR_TIMEOUT);
    };
    auto arrive = [&](uint64_t *bar) { __syncwarp(); if (lane == 0) mbar_arrive(bar); };

    if (warp < KT_SOFT) {
        // ================================================== softmax
        const unsigned group = warp >> 2, pos = (warp & 3) * 32 + lane, col = group * C;
        const uint32_t lanes = ((warp & 3) * 32u) << 16;
        auto group_bar = [&] { asm volatile("bar.sync %0, 128;" :: "r"(3 + group) : "memory"); };
        auto group_or = [&](bool x) {
            unsigned r;
            asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.or.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
                         : "=r"(r) : "r"((unsigned)x), "r"(3 + group) : "memory");
            return r != 0;
        };
        auto bar = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        constexpr float P_SCALE = 32.f;
        unsigned seg = 0;
        while (walk.next(s)) {
            const int j0 = s.row_tile * (int)A.row_tile, nrows = min((int)A.row_tile, s.q.rows - j0) * (int)G;
            const int all = max(0, s.q.len - s.q.n + j0 + 1);  // positions every row attends
            if (pos < C) {
                const int row = (int)(col + pos);
                sh.limit[row] = row < nrows ? s.q.len - s.q.n + j0 + row / (int)G + 1 : 0;
                sh.m[row] = -3.4e38f;
            }
            wait(sh.q_full + (seg & 1), seg >> 1);
            const float factor = sh.factor[seg & 1];
            const bool uneven = sh.uneven[seg & 1];
            if (pos < C) sh.own[col + pos] = sh.row_factor[seg & 1][col + pos];
            arrive(sh.q_empty + (seg & 1));
            ++seg;
            group_bar();
            float l[C], vref = 0.f;
            int vexp = -200;
#pragma unroll
            for (int i = 0; i < C; ++i) l[i] = 0.f;
            for (int t = s.t0; t < s.t1; ++t, ++n) {
                const unsigned b = n & 1, slot = n % KT_META;
                wait(sh.meta_full + slot, n / KT_META);
                const float ks = sh.ks[slot][pos >> 4], vs = sh.vs[slot][pos >> 4];
                // largest value scale of the tile
                int e = -200;
#pragma unroll
                for (int i = 0; i < KT_TILE / 16; ++i) {
                    const float v = sh.vs[slot][i];
                    if (v > 0.f) e = max(e, max(kt_exponent(v) + 1, -100));
                }
                wait(sh.d1_full + b, n >> 1);
                kt_fence_after();
                float x[C];
#pragma unroll
                for (int i = 0; i < C; i += 16) kt_ld16(tmem + lanes + b * N + col + i, x + i);
                kt_wait_ld();
                kt_fence_before();
                arrive(sh.d1_empty + b);
                const float f = factor * ks;
                if (uneven) {
#pragma unroll
                    for (int i = 0; i < C; ++i) x[i] *= sh.own[col + i];
                }
                const int at = t * KT_TILE + (int)pos;
                float over = -INFINITY;
                if (t * KT_TILE + KT_TILE <= all && !__any_sync(0xffffffffu, isnan(ks))) {
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        x[i] *= f;
                        over = fmaxf(over, x[i] - sh.m[col + i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        x[i] = at < sh.limit[col + i] && !isnan(ks) ? x[i] * f : -INFINITY;
                        over = fmaxf(over, x[i] - sh.m[col + i]);
                    }
                }
                if (group_or(over > 8.f || e > vexp)) {
                    // ---- new maxima, and D2 and l in their units
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        const float top = warp_max(x[i]);
                        if (lane == 0) sh.top[warp & 3][col + i] = top;
                    }
                    group_bar();
                    float down = 1.f;
                    if (e > vexp) {
                        down = vexp < -126 ? 0.f : kt_power(vexp - e);
                        vexp = e;
                        vref = kt_power(-e) * P_SCALE;
                    }
                    const bool has = t > s.t0;
                    if (has) {
                        wait(sh.o_done + (b ^ 1), (n - 1) >> 1);
                        kt_fence_after();
                    }
#pragma unroll
                    for (int i0 = 0; i0 < C; i0 += 16) {
                        float y[16];
                        if (has) { kt_ld16(d2 + lanes + col + i0, y); kt_wait_ld(); }
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const unsigned c = col + i0 + i;
                            const float old = sh.m[c];
                            const float top = fmaxf(fmaxf(sh.top[0][c], sh.top[1][c]), fmaxf(sh.top[2][c], sh.top[3][c]));
                            const float alpha = top > old + 8.f ? ex2(old - top) : 1.f;  // each row by its own scores
                            l[i0 + i] *= alpha;
                            y[i] *= alpha * down;
                        }
                        if (has) { kt_st16(d2 + lanes + col + i0, y); kt_wait_st(); }
                    }
                    group_bar();
                    if (pos < C) {
                        const unsigned c = col + pos;
                        const float top = fmaxf(fmaxf(sh.top[0][c], sh.top[1][c]), fmaxf(sh.top[2][c], sh.top[3][c]));
                        if (top > sh.m[c] + 8.f) sh.m[c] = top;
                    }
                    group_bar();
                }
                // ---- weights, in halves, to shared memory
                const float wv = vs * vref;
                if (n >= S::P_STAGES) {
                    const unsigned k = n - S::P_STAGES;
                    wait(sh.o_done + (k & 1), k >> 1);
                }
                unsigned char *row = ring + S::OFF_P + n % S::P_STAGES * 2 * S::PB + pos * 128;
#pragma unroll
                for (int i = 0; i < C; i += 8) {
                    unsigned h[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float p0 = ex2(x[i + j] - sh.m[col + i + j]), p1 = ex2(x[i + j + 1] - sh.m[col + i + j + 1]);
                        l[i + j] += p0;
                        l[i + j + 1] += p1;
                        const float w0 = p0 * wv, w1 = p1 * wv;
                        h[j / 2] = kt_pack(w0, w1);
                        const float2 u = kt_unpack(h[j / 2]);
                        lo[j / 2] = kt_pack(w0 - u.x, w1 - u.y);
                    }
                    const unsigned chunk = (((col + i) >> 3) ^ (pos & 7u)) << 4;
                    *reinterpret_cast<uint4 *>(row + chunk) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(row + S::PB + chunk) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                fence_proxy_async();
                kt_fence_before();
                arrive(sh.p_full + n % S::P_STAGES);
            }
            // ---- the segment's part: sums over positions, D2 in F32
            wait(sh.o_done + ((n - 1) & 1), (n - 1) >> 1);
            kt_fence_after();
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const float v = warp_sum(l[i]);
                if (lane == 0) sh.sum[warp & 3][col + i] = v;
            }
            const float back = vexp < -126 ? 0.f : kt_power(vexp) / P_SCALE;
            float *o = reinterpret_cast<float *>(ring + S::OFF_P);  // P has been read
            bar();
#pragma unroll
            for (int i0 = 0; i0 < C; i0 += 16) {
                float y[16];
                kt_ld16(d2 + lanes + col + i0, y);
                kt_wait_ld();
                if (HD == 128 || pos < HD) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[(col + i0 + i) * HD + pos] = y[i] * back;
                }
            }
            kt_fence_before();
            if (pos < C) {
                const unsigned c = col + pos;
                sh.ml[c] = make_float2(sh.m[c], sh.sum[0][c] + sh.sum[1][c] + sh.sum[2][c] + sh.sum[3][c]);
            }
            bar();
            kv8_finish<N, HD, 32 * KT_SOFT>(A, s, place.units, tid, sh.ml, o, (unsigned)nrows, o, N * HD, &sh.flag, bar,
                [&](unsigned rho, unsigned chunk, float4 v) {
                    const size_t r = (size_t)(s.q.first + j0 + (int)(rho / G));
                    kv8_store4(A.out, A.type, r * A.out_stride + (size_t)(s.head * G + rho % G) * HD + 4 * chunk, v);
                });
            bar();
        }
    } else if (warp < KT_SOFT + KT_CONV) {
        // ================================================== q, and 8 bits to fp16
        const unsigned ct = tid - 32 * KT_SOFT;
        constexpr int PER = 128 / N, QV = HD / PER;  // threads of a q row, values of a thread
        constexpr unsigned RC = HD / 16, STEP = 128 / RC;  // chunks of an 8-bit row; rows that the threads take at once
        auto conv_bar = [] { asm volatile("bar.sync 2, 128;" ::: "memory"); };
        auto convert = [&](unsigned src, unsigned dst, int rows, unsigned slot) {
            const unsigned c = ct % RC, r0 = ct / RC;
#pragma unroll
            for (unsigned i = 0; i < KT_TILE / STEP; ++i) {
                const unsigned r = r0 + i * STEP;
                uint4 v = *reinterpret_cast<const uint4 *>(ring + src + r * HD + ((c ^ kv8_swizzle<HD>(r)) << 4));
                // rows past the last position or never loaded: 0, not what lies there (a NaN stays one times 0)
                if (rows >= 0 && ((int)r >= rows || isnan(sh.ks[slot][r >> 4]))) v = make_uint4(0, 0, 0, 0);
                unsigned h[8];
                kv8_halves<FMT>(v.x, h[0], h[1]);
                kv8_halves<FMT>(v.y, h[2], h[3]);
                kv8_halves<FMT>(v.z, h[4], h[5]);
                kv8_halves<FMT>(v.w, h[6], h[7]);
                const unsigned half = c / 4, k = 2 * (c % 4), z = r & 7u;
                unsigned char *row = ring + dst + half * (S::F16 / 2) + r * 128;
                // the two halves' lanes start on different banks
                const uint4 a = make_uint4(h[0], h[1], h[2], h[3]), b = make_uint4(h[4], h[5], h[6], h[7]);
                *reinterpret_cast<uint4 *>(row + (((k + half) ^ z) << 4)) = half ? b : a;
                *reinterpret_cast<uint4 *>(row + (((k + 1 - half) ^ z) << 4)) = half ? a : b;
            }
            fence_proxy_async();
        };
        auto keys = [&](unsigned i) {  // K of tile i
            wait(sh.k8_full + (i & 1), i >> 1);
            if (i) wait(&sh.kf_empty, i - 1);
            convert(S::OFF_K8 + (i & 1) * S::STAGE, S::OFF_KF, -1, 0);
            arrive(sh.k8_empty + (i & 1));
            arrive(&sh.kf_full);
        };
        unsigned seg = 0, k_at = 0;  // K tiles converted
        while (walk.next(s)) {
            const int j0 = s.row_tile * (int)A.row_tile, nrows = min((int)A.row_tile, s.q.rows - j0) * (int)G;
            const int any = kv8_attended(A, s.q, s.row_tile);
            // ---- q rows, by a power of two that all rows of the tile share; a row whose values are 2^12 below the
            // tile's largest gets its own, so that no row's low half runs into fp16's smallest numbers
            {
                const unsigned row = ct / PER, d0 = ct % PER * QV;
                float x[QV];
                float own = 0.f;
                auto size_of = [](float v) { v = fabsf(v); return v <= 3.4028235e38f ? v : 0.f; };  // 0 for inf and NaN
                if ((int)row < nrows) {
                    const size_t r = (size_t)(s.q.first + j0 + (int)(row / G));
                    const size_t base = r * A.q_stride + (size_t)(s.head * G + row % G) * HD + d0;
#pragma unroll
                    for (int i = 0; i < QV; i += 4) {
                        const float4 v = kv8_load4(A.q, A.type, base + i);
                        x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
                        own = fmaxf(own, fmaxf(fmaxf(size_of(v.x), size_of(v.y)), fmaxf(size_of(v.z), size_of(v.w))));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < QV; ++i) x[i] = 0.f;
                }
#pragma unroll
                for (int o = 1; o < PER; o <<= 1) own = fmaxf(own, __shfl_xor_sync(0xffffffffu, own, o));
                float top = warp_max(own);
                if (lane == 0) sh.q_top[warp - KT_SOFT] = top;
                conv_bar();
                top = fmaxf(fmaxf(sh.q_top[0], sh.q_top[1]), fmaxf(sh.q_top[2], sh.q_top[3]));
                const int below = own > 0.f ? kt_exponent(top) - kt_exponent(own) : 0, extra = below > 12 ? below : 0;
                const int common = 14 - kt_exponent(top), e = common + extra;
                const float up = kt_power(min(e, 127)), up2 = kt_power(e - min(e, 127));
                if (k_at) wait(&sh.kf_empty, k_at - 1);  // the last segment's products have read their q
                if (seg >= 2) wait(sh.q_empty + (seg & 1), (seg >> 1) - 1);
#pragma unroll
                for (int i = 0; i < QV; i += 8) {
                    unsigned h[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float a = x[i + j] * up * up2, b = x[i + j + 1] * up * up2;
                        h[j / 2] = kt_pack(a, b);
                        const float2 u = kt_unpack(h[j / 2]);
                        lo[j / 2] = kt_pack(a - u.x, b - u.y);
                    }
                    const unsigned d = d0 + i, chunk = d % 64 / 8;
                    unsigned char *q = ring + S::OFF_Q + d / 64 * (N * 128) + row * 128 + ((chunk ^ (row & 7u)) << 4);
                    *reinterpret_cast<uint4 *>(q) = make_uint4(h[0], h[1], h[2], h[3]);
                    if (QP == 2) *reinterpret_cast<uint4 *>(q + S::QB) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                if (ct == 0) sh.factor[seg & 1] = ldexpf(A.scale, -common);
                if (ct % PER == 0) sh.row_factor[seg & 1][row] = kt_power(-extra);
                fence_proxy_async();
                // and q_top can be written again
                unsigned some;
                asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.or.pred q, 2, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
                             : "=r"(some) : "r"((unsigned)extra) : "memory");
                if (ct == 0) sh.uneven[seg & 1] = (int)some;
                arrive(sh.q_full + (seg & 1));
                ++seg;
            }
            // K one tile ahead of V: V's buffer is free only when the tile before has been weighted
            keys(k_at++);
            for (int t = s.t0; t < s.t1; ++t, ++n) {
                if (t + 1 < s.t1) keys(k_at++);
                wait(sh.v8_full + (n & 1), n >> 1);
                if (n) wait(sh.o_done + ((n - 1) & 1), (n - 1) >> 1);
                convert(S::OFF_V8 + (n & 1) * S::STAGE, S::OFF_VF, any - t * KT_TILE < 0 ? 0 : any - t * KT_TILE, n % KT_META);
                arrive(sh.v8_empty + (n & 1));
                arrive(&sh.vf_full);
            }
        }
    } else if (warp == KT_SOFT + KT_CONV) {
        // ================================================== TMA
        const unsigned size = 1u << A.shift, box = min(size, 64u), per = KT_TILE / box;
        while (walk.next(s)) {
            const int blocks = (kv8_attended(A, s.q, s.row_tile) + (int)size - 1) >> A.shift;
            const int *ids = A.table + (size_t)s.request * A.table_stride;
            int have = -1, id = 0;  // lane holds block 32 * have + lane
            float ks = 0.f, vs = 0.f;
            for (int t = s.t0; t < s.t1; ++t, ++n) {
                const int b0 = t * KT_TILE >> A.shift;
                if (b0 / 32 != have) {
                    have = b0 / 32;
                    const int b = have * 32 + (int)lane;
                    id = b < blocks ? ids[b] : -1;
                    const bool ok = id >= 0 && (unsigned)id < A.c.blocks;
                    if (b < blocks && !ok) raise_error(A.error, ERR_BOUNDS);
                    ks = ok ? A.c.k_scale[(size_t)id * kv + s.head] : NAN;
                    vs = ok ? A.c.v_scale[(size_t)id * kv + s.head] : 0.f;
                    if (!ok) id = -1;
                }
                const unsigned b = n & 1, slot = n % KT_META;
                const unsigned group_block = (unsigned)(b0 & 31) + (lane % (KT_TILE / 16) * 16 >> min(A.shift, 7u));
                const float gk = __shfl_sync(0xffffffffu, ks, group_block & 31u), gv = __shfl_sync(0xffffffffu, vs, group_block & 31u);
                const unsigned box_block = (unsigned)(b0 & 31) + (lane % per * box >> A.shift);
                const int mine = __shfl_sync(0xffffffffu, id, box_block & 31u);
                const bool load = lane < per && mine >= 0;
                const unsigned boxes = __popc(__ballot_sync(0xffffffffu, load));
                const int row = (int)((((unsigned)mine * kv + s.head) << A.shift) + ((unsigned)(t * KT_TILE + (int)(lane % per * box)) & (size - 1)));
                if (n >= 2) wait(sh.k8_empty + b, (n >> 1) - 1);
                if (lane < KT_TILE / 16) { sh.ks[slot][lane] = gk; sh.vs[slot][lane] = gv; }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(sh.meta_full + slot);
                    if (boxes) mbar_expect_tx(sh.k8_full + b, boxes * box * HD); else mbar_arrive(sh.k8_full + b);
                }
                __syncwarp();
                if (load && !*dead) tma_load_rows(ring + S::OFF_K8 + b * S::STAGE + lane * box * HD, &kmap, row, sh.k8_full + b);
                if (n >= 2) wait(sh.v8_empty + b, (n >> 1) - 1);
                __syncwarp();
                if (lane == 0) {
                    if (boxes) mbar_expect_tx(sh.v8_full + b, boxes * box * HD); else mbar_arrive(sh.v8_full + b);
                }
                __syncwarp();
                if (load && !*dead) tma_load_rows(ring + S::OFF_V8 + b * S::STAGE + lane * box * HD, &vmap, row, sh.v8_full + b);
            }
        }
        if (*dead) {  // copies in flight land before the CTA leaves its shared memory
            for (unsigned i = 0; i < min(n, 2u); ++i) {
                mbar_wait_bounded(sh.k8_full + ((n - 1 - i) & 1), (n - 1 - i) >> 1 & 1);
                mbar_wait_bounded(sh.v8_full + ((n - 1 - i) & 1), (n - 1 - i) >> 1 & 1);
            }
        }
    } else if (lane == 0) {
        // ================================================== MMA
        const unsigned kf = smem_u32(ring + S::OFF_KF), vf = smem_u32(ring + S::OFF_VF), qs = smem_u32(ring + S::OFF_Q),
                       ps = smem_u32(ring + S::OFF_P);
        unsigned k_at = 0;
        auto scores = [&] {
            const unsigned b = k_at & 1;
            wait(&sh.kf_full, k_at);
            if (k_at >= 2) wait(sh.d1_empty + b, (k_at >> 1) - 1);
            kt_fence_after();
#pragma unroll
            for (int part = 0; part < QP; ++part)
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)
                    kt_mma(tmem + b * N, kt_desc(kf + k / 4 * (S::F16 / 2) + k % 4 * 32, 16),
                           kt_desc(qs + part * S::QB + k / 4 * (N * 128) + k % 4 * 32, 16), kt_idesc(N, false), part || k);
            kt_commit(&sh.kf_empty);
            kt_commit(sh.d1_full + b);
            ++k_at;
        };
        while (walk.next(s)) {
            scores();
            for (int t = s.t0; t < s.t1; ++t, ++n) {
                if (t + 1 < s.t1) scores();
                const unsigned b = n % S::P_STAGES;
                wait(&sh.vf_full, n);
                wait(sh.p_full + b, n / S::P_STAGES);
                kt_fence_after();
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int k = 0; k < KT_TILE / 16; ++k)
                        kt_mma(d2, kt_desc(vf + k * 2048, S::F16 / 2),
                               kt_desc(ps + (2 * b + (unsigned)part) * S::PB + k * 2048, S::PB), kt_idesc(N, true),
                               t > s.t0 || part || k);
                kt_commit(sh.o_done + (n & 1));
            }
        }
        kt_commit(&sh.drained);
        mbar_wait_bounded(&sh.drained, 0);
    }
    kt_fence_before();
    __syncthreads();
    if (warp == KT_SOFT + KT_CONV + 1) {
        kt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(TM) : "memory");
    }
}

template <int HD, unsigned FMT, int N, int QP>
int kv8_tiles_go(const Kv8Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned grid, cudaStream_t s)
{
    constexpr size_t smem = 1024 + KtShape<HD, N, QP>::OFF_END + sizeof(KtShared<N>);
    static_assert(smem <= 227 * 1024, "shared memory of one CTA");
    if (cudaFuncSetAttribute(kv8_tiles_kernel<HD, FMT, N, QP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
        cudaGetLastError();
        return -2;
    }
    kv8_tiles_kernel<HD, FMT, N, QP><<<grid, KT_THREADS, smem, s>>>(A, k, v);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace fyb
