// kv8_tiles.cuh - attention over the paged 8-bit cache for many query rows per
// KV head (drafts, prompt chunks), on the 5th-generation tensor cores. One
// instantiation per head dimension and format (kv8_tiles_inst.cu).
//
// Per tile of 128 positions, N = 32 or 64 query rows of one KV head:
//
//   D1[position][row] = K Q^T       tcgen05.mma kind::f16, M = 128, K = head_dim
//   P = 2^(D1 scale - m) v_scale    one thread per position and 16 rows
//   D2[hd][row] += V^T P^T          M = 128, K = 128 positions
//
// K and V come as 8-bit tiles by TMA; four warps convert them to fp16 (exact) on
// their way from shared to tensor memory, V transposed, where both products
// read them as operand A: a tile's fp16 form never loads shared memory, whose
// bandwidth bounds this kernel otherwise (operands staged there instead: 5800
// cycles a tile at N = 64). The weights, and q of F32 rows, are two fp16 halves
// hi + lo (22 bits, an MMA each); q of 16-bit rows is one half, which holds it
// (a bf16 value 2^24 below its tile's largest loses bits that no score shows).
//
// The maximum m of a row moves only when a score is more than 2^8 above it. The
// tensor core rounds its running sums towards zero, about 2^-26 a step, so D2
// gathers KT_FLUSH tiles and is then added to sums in shared memory, rounded to
// nearest (2000 steps in D2 alone: 3e-5 off), and a product's low halves go
// first, while the sum is small. Row sums and maxima are F32.
//
// Bound by the softmax warps' latency on one tile: taking out exponentials, low
// halves, flushes, conversions or MMAs one at a time changes less than 5 %. At
// N = 64 the row tiles of a long chunk also read K and V from L2 once each.
// Ragged drafts of 8 (32 requests of 128 to 32768, 32/8 heads, 0.97 GB): 280 us,
// 0.54 of a measured copy; a chunk of 500 rows at 16001: 354 us.
//
// Roles: N / 4 warps softmax (groups of four, 16 rows each; a thread has a
// position and its group's rows), four K, four V and q, one TMA, one MMA.
#pragma once
#include "kv8_attention.cuh"
#include "kt_mma.cuh"

namespace fyb {

constexpr int KT_TILE = 128, KT_CONV = 4, KT_META = 8;
// Warps: four softmax for every 16 rows; four that convert K and four that convert V, at 32 rows the same four (14
// warps: a thread has 128 registers; with 18 it has 96, 309 against 274 us for the ragged drafts of 8). At 64 rows 26
// warps have 72 each.
FYB_HOST_DEV constexpr int kt_soft(int N) { return N / 4; }
FYB_HOST_DEV constexpr bool kt_split(int N) { return N > 32; }
FYB_HOST_DEV constexpr int kt_conv(int N) { return kt_split(N) ? 2 * KT_CONV : KT_CONV; }
FYB_HOST_DEV constexpr int kt_threads(int N) { return 32 * (kt_soft(N) + kt_conv(N) + 2); }

constexpr int KT_FLUSH = 2;  // tiles D2 gathers before it is added to the sums

// The CTA's k-th segment, walked from the start; t1 = 0 past the last.
static __device__ __noinline__ void kt_segment(const Kv8Attention &A, const Kv8Place &place, unsigned k, Kv8Segment *s)
{
    Kv8Walk<KT_TILE> walk(A, place);
    for (unsigned i = 0; i <= k; ++i)
        if (!walk.next(*s)) { s->t1 = 0; break; }
}
// Sums of v[0..16) over the 32 lanes: lane i % 16 returns element i.
FYB_DEV float kt_sum16(float (&v)[16], unsigned lane)
{
#pragma unroll
    for (int half = 8; half; half /= 2) {
        const bool up = lane & (unsigned)half;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float give = up ? v[i] : v[i + half], keep = up ? v[i + half] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, half);
        }
    }
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
}
template <int HD, int N, int QP> struct KtShape {
    static constexpr int STAGE = KT_TILE * HD, STAGES = QP * N * HD > 8192 ? 2 : 3;  // an 8-bit tile; as many as fit
    static constexpr int QB = N * HD * 2, PB = KT_TILE * 128;                        // one half of q; one half of P
    static constexpr int OFF_K8 = 0, OFF_V8 = OFF_K8 + STAGES * STAGE, OFF_Q = OFF_V8 + STAGES * STAGE,
                         OFF_P = OFF_Q + QP * QB, OFF_O = OFF_P + 4 * PB, OFF_END = OFF_O + N * HD * 4;
    // tensor memory: D1 of two tiles, D2 of two flush periods, K and V of two tiles
    static constexpr int D1 = 0, D2 = 2 * N, K = 4 * N, V = K + HD, COLS = V + KT_TILE <= 256 ? 256 : 512;
};
// The CTA's parts of segments, walked by the TMA warp alone and handed to the others here: KT_SEGS of them at a
// time; t1 = 0 ends the line.
constexpr int KT_SEGS = 4;
template <int N> struct KtShared {
    Kv8Segment seg[KT_SEGS], walked[kt_threads(N) / 32];
    Kv8Place place;
    uint64_t seg_full[KT_SEGS], seg_empty[KT_SEGS];
    float ks[KT_META][KT_TILE / 16], vs[KT_META][KT_TILE / 16];  // scales by 16 positions; ks NaN: not loaded
    int exponent[KT_META], hole[KT_META];                         // 2^exponent is above every value scale of the tile; whether some were not loaded
    unsigned char lower[KT_META][N];                              // what a tile lowers its rows' maxima by
    alignas(16) float m[N];
    float own[N], alpha[N], top[4][N], sum[4][N];
    int limit[N];                                                 // positions a row attends
    float2 ml[N];
    float factor[2], row_factor[2][N], q_top[KT_CONV];            // score factors: of the tile's q, and beside it of a row
    int uneven[2];                                                // whether some row has a factor of its own
    uint64_t k8_full[3], k8_empty[3], v8_full[3], v8_empty[3], kf_full[2], kf_empty[2], vf_full[2], d1_full[2],
        d1_empty[2], p_full[2], o_done[2], q_full[2], q_empty[2], meta_full[KT_META], drained;
    uint32_t tmem;
    unsigned flag, dead;
};

template <int HD, unsigned FMT, int N, int QP>
__global__ void __launch_bounds__(kt_threads(N), 1) kv8_tiles_kernel(const __grid_constant__ Kv8Attention A, const __grid_constant__ CUtensorMap kmap,
    const __grid_constant__ CUtensorMap vmap)
{
    using S = KtShape<HD, N, QP>;
    constexpr int KT_SOFT = kt_soft(N), C = 16;  // softmax warps; columns of a softmax thread
    constexpr bool SPLIT = kt_split(N);
    constexpr unsigned W_TMA = KT_SOFT + kt_conv(N), W_MMA = W_TMA + 1;
    extern __shared__ unsigned char kt_smem[];
    unsigned char *ring = kt_smem + ((1024u - (smem_u32(kt_smem) & 1023u)) & 1023u);
    KtShared<N> &sh = *reinterpret_cast<KtShared<N> *>(ring + S::OFF_END);
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), kv = A.c.kv_heads, G = A.group;
    if (tid == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            mbar_init(sh.k8_full + i, 1); mbar_init(sh.k8_empty + i, KT_CONV);
            mbar_init(sh.v8_full + i, 1); mbar_init(sh.v8_empty + i, KT_CONV);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(sh.kf_full + i, KT_CONV); mbar_init(sh.kf_empty + i, 1); mbar_init(sh.vf_full + i, KT_CONV);
            mbar_init(sh.d1_full + i, 1); mbar_init(sh.d1_empty + i, KT_SOFT);
            mbar_init(sh.p_full + i, KT_SOFT); mbar_init(sh.o_done + i, 1);
            mbar_init(sh.q_full + i, KT_CONV); mbar_init(sh.q_empty + i, KT_SOFT);
        }
        for (int i = 0; i < KT_META; ++i) mbar_init(sh.meta_full + i, 1);
        for (int i = 0; i < KT_SEGS; ++i) { mbar_init(sh.seg_full + i, 1); mbar_init(sh.seg_empty + i, KT_SOFT + kt_conv(N) + 1); }
        mbar_init(&sh.drained, 1);
        sh.dead = 0;
        fence_barrier_init();
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&sh.tmem)), "r"(S::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    kt_fence_before();
    {
        const Kv8Place place = kv8_place<KT_TILE, kt_threads(N), 2>(A);  // CTA barriers inside
        if (tid == 0) sh.place = place;
    }
    __syncthreads();
    kt_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&sh.tmem;
    unsigned n = 0, seg = 0;  // tiles and segments of this CTA so far
    volatile unsigned *dead = &sh.dead;  // a wait ran out: nobody waits any more, the error word is set
    auto wait = [&](uint64_t *bar, unsigned parity) {
        kt_wait(bar, parity, dead);
    };
    auto arrive = [&](uint64_t *bar) { __syncwarp(); if (lane == 0) mbar_arrive(bar); };
    // The segment that comes next; done() with it before the next is asked for. Once a wait has run out every warp
    // walks by itself: all of them still take the same steps, so none is left at a barrier.
    auto next = [&]() -> const Kv8Segment * {
        wait(sh.seg_full + seg % KT_SEGS, seg / KT_SEGS);
        const Kv8Segment *s = sh.seg + seg % KT_SEGS;
        if (__builtin_expect(*dead, 0)) {
            s = sh.walked + warp;
            if (lane == 0) kt_segment(A, sh.place, seg, sh.walked + warp);
            __syncwarp();
        }
        return s->t1 ? s : nullptr;
    };
    auto done = [&] { arrive(sh.seg_empty + seg % KT_SEGS); ++seg; };

    // K of tile i: a thread converts its position's row, column c of its lane gets values 2c and 2c + 1
    auto keys = [&](unsigned i) {
        const unsigned ct = tid & 127;
        const uint32_t lanes = (ct & 96u) << 16;
        const unsigned st = i % S::STAGES, pos = ct;
        wait(sh.k8_full + st, i / S::STAGES);
        if (i >= 2) wait(sh.kf_empty + (i & 1), (i >> 1) - 1);
        kt_fence_after();
        const unsigned char *src = ring + S::OFF_K8 + st * S::STAGE + pos * HD;
        const unsigned z = kv8_swizzle<HD>(pos);
#pragma unroll 2
        for (unsigned c = 0; c < HD / 16; c += 2) {
            unsigned h[16];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint4 v = *reinterpret_cast<const uint4 *>(src + (((c + k) ^ z) << 4));
                kv8_halves<FMT>(v.x, h[8 * k], h[8 * k + 1]);
                kv8_halves<FMT>(v.y, h[8 * k + 2], h[8 * k + 3]);
                kv8_halves<FMT>(v.z, h[8 * k + 4], h[8 * k + 5]);
                kv8_halves<FMT>(v.w, h[8 * k + 6], h[8 * k + 7]);
            }
            kt_st16(tmem + S::K + (i & 1) * (HD / 2) + lanes + c * 8, reinterpret_cast<float *>(h));
        }
        arrive(sh.k8_empty + st);
        kt_wait_st();
        kt_fence_before();
        arrive(sh.kf_full + (i & 1));
    };

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
        auto bar = [] { asm volatile("bar.sync 1, %0;" :: "n"(32 * KT_SOFT) : "memory"); };
        constexpr float P_SCALE = 32.f;
        unsigned period = 0;
        while (const Kv8Segment *sp = next()) {
            const Kv8Segment &s = *sp;
            const int t0 = s.t0, t1 = s.t1;
            const int all = max(0, s.q.len - s.q.n + s.row_tile * (int)A.row_tile + 1);  // positions every row attends
            if (pos < C) {
                const int row = (int)(col + pos), j0 = s.row_tile * (int)A.row_tile;
                const int nrows = min((int)A.row_tile, s.q.rows - j0) * (int)G;
                sh.limit[row] = row < nrows ? s.q.len - s.q.n + j0 + row / (int)G + 1 : 0;
                sh.m[row] = -3.4e38f;
            }
            wait(sh.q_full + (seg & 1), seg >> 1);
            const float factor = sh.factor[seg & 1];
            const bool uneven = sh.uneven[seg & 1];
            if (pos < C) sh.own[col + pos] = sh.row_factor[seg & 1][col + pos];
            arrive(sh.q_empty + (seg & 1));
            group_bar();
            float l[C], vref = 0.f;  // l: sums of p
            int vexp = -200;
            float *o = reinterpret_cast<float *>(ring + S::OFF_O) + col * HD + pos;  // this thread's sums, HD apart
            const bool mine = HD == 128 || pos < HD;
#pragma unroll
            for (int i = 0; i < C; ++i) l[i] = 0.f;
            if (mine) {
#pragma unroll 8
                for (int i = 0; i < C; ++i) o[i * HD] = 0.f;
            }
            // adds the D2 of a finished period to o
            auto flush = [&](unsigned which) {
                kt_fence_after();
                float y[16];
                kt_ld16(tmem + S::D2 + (which & 1) * N + lanes + col, y);
                kt_wait_ld();
                if (mine) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i * HD] += y[i];
                }
                kt_fence_before();
            };
            bool pending = false;  // the period before has ended and is not in o yet
            bool fresh = true;     // some row may not have a maximum yet
            for (int t = t0; t < t1; ++t, ++n) {
                const unsigned b = n & 1, slot = n % KT_META;
                const int step = (t - t0) % KT_FLUSH;
                if (step == 0 && t > t0) { pending = true; ++period; }
                wait(sh.meta_full + slot, n / KT_META);
                const float ks = sh.ks[slot][pos >> 4], vs = sh.vs[slot][pos >> 4], f = factor * ks;
                const int e = sh.exponent[slot];
                const bool hole = sh.hole[slot], raw = fresh || hole || t * KT_TILE + KT_TILE > all, grow = e > vexp;
                float down = 1.f;
                if (__builtin_expect(grow, 0)) {
                    down = vexp < -126 ? 0.f : kt_power(vexp - e);
                    vexp = e;
                    vref = kt_power(-e) * P_SCALE;
                }
                fresh = fresh && hole;
                const float wv = vs * vref;
                if (n >= 2) wait(sh.o_done + b, (n >> 1) - 1);
                if (pending && step == 1) {  // its last tile is two back
                    flush(period - 1);
                    pending = false;
                }
                wait(sh.d1_full + b, n >> 1);
                kt_fence_after();
                const float4 *m4 = reinterpret_cast<const float4 *>(sh.m + col);
                float x[16];
                kt_ld16(tmem + S::D1 + lanes + b * N + col, x);
                kt_wait_ld();
                if (__builtin_expect(uneven, 0)) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] *= sh.own[col + i];
                }
                // x: the scores less m, or (raw) the scores themselves
                float over = -INFINITY;
                if (__builtin_expect(raw, 0)) {
                    const int at = isnan(ks) ? 0x7fffffff : t * KT_TILE + (int)pos;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        x[i] = at < sh.limit[col + i] ? x[i] * f : -INFINITY;
                        over = fmaxf(over, x[i] - sh.m[col + i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float4 m = m4[i / 4];
                        x[i] = fmaf(x[i], f, -m.x); x[i + 1] = fmaf(x[i + 1], f, -m.y);
                        x[i + 2] = fmaf(x[i + 2], f, -m.z); x[i + 3] = fmaf(x[i + 3], f, -m.w);
                        over = fmaxf(fmaxf(over, fmaxf(x[i], x[i + 1])), fmaxf(x[i + 2], x[i + 3]));
                    }
                }
                if (__builtin_expect(group_or(over > 8.f || grow), 0)) {
                    // ---- new maxima, and the sums so far in their units
                    if (!raw) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] += sh.m[col + i];
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const unsigned top = __reduce_max_sync(0xffffffffu, isnan(x[i]) ? 0u : float_order_key(x[i]));
                        if (lane == 0) sh.top[warp & 3][col + i] = top ? float_from_order_key(top) : -INFINITY;
                    }
                    group_bar();
                    if (pos < 16) {
                        const unsigned c = col + pos;
                        const float old = sh.m[c], top = fmaxf(fmaxf(sh.top[0][c], sh.top[1][c]), fmaxf(sh.top[2][c], sh.top[3][c]));
                        const bool up = top - old > 8.f;  // each row by its own scores; old + 8 could round up
                        // volatile: its address, formed ahead, is a register too many in the loop (48 bytes spilled,
                        // chunk 370 to 391 us)
                        const float now = (up ? top : old) - (float)*((volatile unsigned char *)&sh.lower[0][0] + (n % KT_META) * N + c);
                        sh.alpha[c] = now != old ? ex2(old - now) : 1.f;
                        sh.m[c] = now;
                    }
                    if (t > t0) wait(sh.o_done + (b ^ 1), (n - 1) >> 1);
                    if (pending) {
                        flush(period - 1);
                        pending = false;
                    }
                    kt_fence_after();
                    group_bar();
                    // four columns at a time: few registers where there are none to spare
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const uint32_t d2 = tmem + S::D2 + (period & 1) * N + lanes + col + i;
                        float y[4];
                        if (step) { kt_ld4(d2, y); kt_wait_ld(); }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float alpha = sh.alpha[col + i + j], both = alpha * down;
                            l[i + j] *= alpha;
                            if (mine) o[(i + j) * HD] *= both;
                            y[j] *= both;
                            x[i + j] -= sh.m[col + i + j];
                        }
                        if (step) { kt_st4(d2, y); kt_wait_st(); }
                    }
                    kt_fence_before();
                } else if (__builtin_expect(raw, 0)) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] -= sh.m[col + i];
                }
                // ---- weights, in halves, to shared memory
                unsigned char *row = ring + S::OFF_P + b * 2 * S::PB + pos * 128;
#pragma unroll
                for (int i = 0; i < 16; i += 8) {
                    unsigned h[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float p0 = ex2(x[i + j]), p1 = ex2(x[i + j + 1]);
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
                kt_fence_before();
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) { mbar_arrive(sh.d1_empty + b); mbar_arrive(sh.p_full + b); }
            }
            // ---- the segment's part: sums over positions, D2 in F32
            wait(sh.o_done + ((n - 1) & 1), (n - 1) >> 1);
#pragma unroll 1
            for (int back = pending ? 1 : 0; back >= 0; --back) flush(period - (unsigned)back);
            ++period;
            const float back = vexp < -126 ? 0.f : kt_power(vexp) / P_SCALE;
            if (mine) {
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i * HD] *= back;
            }
            float y[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = l[i];
            const float sum = kt_sum16(y, lane);
            if (lane < 16) sh.sum[warp & 3][col + lane] = sum;
            group_bar();
            if (pos < C) {
                const unsigned c = col + pos;
                sh.ml[c] = make_float2(sh.m[c], sh.sum[0][c] + sh.sum[1][c] + sh.sum[2][c] + sh.sum[3][c]);
            }
            bar();
            float *all_o = reinterpret_cast<float *>(ring + S::OFF_O);
            const int j0 = s.row_tile * (int)A.row_tile, nrows = min((int)A.row_tile, s.q.rows - j0) * (int)G;
            kv8_finish<N, HD, 32 * KT_SOFT>(A, s, sh.place, tid, sh.ml, all_o, (unsigned)nrows, all_o, N * HD, &sh.flag, bar,
                [&](unsigned rho, unsigned chunk, float4 v) {
                    const size_t r = (size_t)(s.q.first + j0 + (int)(rho / G));
                    kv8_store4(A.out, A.type, r * A.out_stride + (size_t)(s.head * G + rho % G) * HD + 4 * chunk, v);
                });
            bar();
            done();
        }
    } else if (SPLIT && warp < KT_SOFT + KT_CONV) {
        // ================================================== K, 8 bits to fp16
        unsigned k_at = 0;
        while (const Kv8Segment *s = next()) {
#pragma unroll 1
            for (int left = s->t1 - s->t0; left; --left) keys(k_at++);
            done();
        }
    } else if (warp < W_TMA) {
        // ================================================== q; V (and K), 8 bits to fp16
        const unsigned ct = tid & 127, cw = ct >> 5;
        unsigned k_at = 0;
        const uint32_t lanes = (cw * 32u) << 16;
        constexpr int PER = 128 / N, QV = HD / PER;  // threads of a q row, values of a thread
        auto conv_bar = [] { asm volatile("bar.sync 2, 128;" ::: "memory"); };
        // V of tile n, transposed: lane = head dimension, column c gets positions 2c and 2c + 1; positions from `rows`
        // on, or never loaded, are 0 and not what lies there (a NaN stays one times 0)
        auto values = [&](int rows) {
            const unsigned st = n % S::STAGES, slot = n % KT_META;
            wait(sh.v8_full + st, n / S::STAGES);
            if (n >= 2) wait(sh.o_done + (n & 1), (n >> 1) - 1);
            kt_fence_after();
            const bool patchy = sh.hole[slot] || rows < KT_TILE;
            if (cw < HD / 32) {
                const unsigned r = lane & 15, chunk = 2 * cw + (lane >> 4), t4 = lane & 3;
                const unsigned src = smem_u32(ring + S::OFF_V8 + st * S::STAGE) + r * HD + ((chunk ^ kv8_swizzle<HD>(r)) << 4);
#pragma unroll 1
                for (int j0 = 0; j0 < KT_TILE / 16; j0 += 4) {
                    unsigned lo[16], hi[16];  // dimensions 0..15 and 16..31 of the warp's, 64 positions
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        unsigned w[4];
                        asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(src + (j0 + j) * 16 * HD));
                        const int first = (j0 + j) * 16;
                        if (__builtin_expect(patchy, 0)) {
                            const int left = isnan(sh.ks[slot][j0 + j]) ? 0 : rows - first - 4 * (int)t4;
                            const unsigned keep = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << 8 * left) - 1;
                            w[0] &= keep; w[1] &= keep; w[2] &= keep; w[3] &= keep;
                        }
                        kv8_halves<FMT>(w[0], lo[4 * j], lo[4 * j + 1]);
                        kv8_halves<FMT>(w[1], lo[4 * j + 2], lo[4 * j + 3]);
                        kv8_halves<FMT>(w[2], hi[4 * j], hi[4 * j + 1]);
                        kv8_halves<FMT>(w[3], hi[4 * j + 2], hi[4 * j + 3]);
                    }
                    const uint32_t dst = tmem + S::V + (n & 1) * (KT_TILE / 2) + lanes + j0 * 8;
                    kt_st256(dst, lo);
                    kt_st256(dst + (16u << 16), hi);
                }
                kt_wait_st();
            }
            kt_fence_before();
            arrive(sh.v8_empty + st);
            arrive(sh.vf_full + (n & 1));
        };
        while (const Kv8Segment *sp = next()) {
            const Kv8Segment &s = *sp;
            const int j0 = s.row_tile * (int)A.row_tile, nrows = min((int)A.row_tile, s.q.rows - j0) * (int)G;
            const int any = kv8_attended(A, s.q, s.row_tile);
            // ---- q rows, by a power of two that all rows of the tile share; a row whose values are 2^12 below the
            // tile's largest gets its own, so that no row's low half runs into fp16's smallest numbers
            {
                const unsigned row = ct / PER, d0 = ct % PER * QV;
                const bool real = (int)row < nrows;
                const size_t r = (size_t)(s.q.first + j0 + (real ? (int)(row / G) : 0));
                const size_t base = r * A.q_stride + (size_t)(s.head * G + (real ? row % G : 0)) * HD + d0;
                float own = 0.f;
                auto size_of = [](float v) { v = fabsf(v); return v <= 3.4028235e38f ? v : 0.f; };  // 0 for inf and NaN
#pragma unroll 2
                for (int i = 0; i < QV; i += 4) {
                    const float4 v = kv8_load4(A.q, A.type, base + i);
                    own = fmaxf(own, fmaxf(fmaxf(size_of(v.x), size_of(v.y)), fmaxf(size_of(v.z), size_of(v.w))));
                }
                if (!real) own = 0.f;
#pragma unroll
                for (int o = 1; o < PER; o <<= 1) own = fmaxf(own, __shfl_xor_sync(0xffffffffu, own, o));
                float top = warp_max(own);
                if (lane == 0) sh.q_top[cw] = top;
                conv_bar();
                top = fmaxf(fmaxf(sh.q_top[0], sh.q_top[1]), fmaxf(sh.q_top[2], sh.q_top[3]));
                const int below = own > 0.f ? kt_exponent(top) - kt_exponent(own) : 0, extra = below > 12 ? below : 0;
                const int common = 14 - kt_exponent(top), e = common + extra;
                const float up = real ? kt_power(min(e, 127)) : 0.f, up2 = kt_power(e - min(e, 127));
                if (n) wait(sh.kf_empty + ((n - 1) & 1), (n - 1) >> 1);  // the last segment's products have read their q
                if (seg >= 2) wait(sh.q_empty + (seg & 1), (seg >> 1) - 1);
#pragma unroll 1
                for (int i = 0; i < QV; i += 8) {
                    unsigned h[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 8; j += 4) {
                        const float4 v = kv8_load4(A.q, A.type, base + i + j);
                        const float x0 = real ? v.x * up * up2 : 0.f, x1 = real ? v.y * up * up2 : 0.f,
                                    x2 = real ? v.z * up * up2 : 0.f, x3 = real ? v.w * up * up2 : 0.f;
                        h[j / 2] = kt_pack(x0, x1);
                        h[j / 2 + 1] = kt_pack(x2, x3);
                        const float2 a = kt_unpack(h[j / 2]), b = kt_unpack(h[j / 2 + 1]);
                        lo[j / 2] = kt_pack(x0 - a.x, x1 - a.y);
                        lo[j / 2 + 1] = kt_pack(x2 - b.x, x3 - b.y);
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
            }
            const int t1 = s.t1;
#pragma unroll 1
            for (int t = SPLIT ? s.t0 : s.t0 - 1; t < t1; ++t) {
                if (!SPLIT && t + 1 < t1) keys(k_at++);  // one tile ahead: V's buffer frees later
                if (!SPLIT && t < s.t0) continue;
                values(any - t * KT_TILE);
                ++n;
            }
            done();
        }
    } else if (warp == W_TMA) {
        // ================================================== TMA
        const unsigned size = 1u << A.shift, box = min(size, 64u), per = KT_TILE / box;
        __syncwarp();
        Kv8Walk<KT_TILE> walk(A, sh.place);
        Kv8Segment s;
        for (;; ++seg) {
            const bool more = walk.next(s);
            if (seg >= KT_SEGS) wait(sh.seg_empty + seg % KT_SEGS, seg / KT_SEGS - 1);
            if (lane == 0 && !*dead) {
                if (more) sh.seg[seg % KT_SEGS] = s; else sh.seg[seg % KT_SEGS].t1 = 0;
                mbar_arrive(sh.seg_full + seg % KT_SEGS);
            }
            __syncwarp();
            if (!more) break;
            const int blocks = (kv8_attended(A, s.q, s.row_tile) + (int)size - 1) >> A.shift;
            const int *ids = A.table + (size_t)s.request * A.table_stride;
            int have = -1, id = 0;  // lane holds block 32 * have + lane
            float ks = 0.f, vs = 0.f;
            int seen = -200;        // largest exponent so far
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
                const unsigned b = n % S::STAGES, slot = n % KT_META;
                const unsigned group_block = (unsigned)(b0 & 31) + (lane % (KT_TILE / 16) * 16 >> min(A.shift, 7u));
                const float gk = __shfl_sync(0xffffffffu, ks, group_block & 31u), gv = __shfl_sync(0xffffffffu, vs, group_block & 31u);
                const unsigned box_block = (unsigned)(b0 & 31) + (lane % per * box >> A.shift);
                const int mine = __shfl_sync(0xffffffffu, id, box_block & 31u);
                const bool load = lane < per && mine >= 0;
                const unsigned boxes = __popc(__ballot_sync(0xffffffffu, load));
                const int row = (int)((((unsigned)mine * kv + s.head) << A.shift) + ((unsigned)(t * KT_TILE + (int)(lane % per * box)) & (size - 1)));
                if (n >= S::STAGES) wait(sh.k8_empty + b, n / S::STAGES - 1);
                const bool hole = __any_sync(0xffffffffu, isnan(gk));
                const int ex = gv > 0.f ? max(kt_exponent(gv) + 1, -100) : -200, top = __reduce_max_sync(0xffffffffu, ex);
                // The tile's weights are relative to its largest value scale: a row that ends before the positions that
                // have it gets its maximum lowered by as much, or its weights would lose bits to tokens after it (scales
                // 2^15 apart, heads of one row each: 8e-5 of the row's largest value)
                int low[N / 32] = {};
                if (__builtin_expect(top > seen, 0)) {
#pragma unroll
                    for (int i = 0; i < N / 32; ++i) {
                        const int ends = s.q.len - s.q.n + s.row_tile * (int)A.row_tile + (int)((lane + 32 * i) / G) + 1 - t * KT_TILE;
                        int mine_ex = seen;
#pragma unroll 1
                        for (int g = 0; g < KT_TILE / 16; ++g) {
                            const int eg = __shfl_sync(0xffffffffu, ex, g);
                            if (16 * g < ends) mine_ex = max(mine_ex, eg);
                        }
                        low[i] = ends > 0 ? min(top - mine_ex, 64) : 0;
                    }
                    seen = top;
                }
#pragma unroll
                for (int i = 0; i < N / 32; ++i) sh.lower[slot][lane + 32 * i] = (unsigned char)low[i];
                if (lane < KT_TILE / 16) { sh.ks[slot][lane] = gk; sh.vs[slot][lane] = gv; sh.exponent[slot] = top; sh.hole[slot] = hole; }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(sh.meta_full + slot);
                    if (boxes) mbar_expect_tx(sh.k8_full + b, boxes * box * HD); else mbar_arrive(sh.k8_full + b);
                }
                __syncwarp();
                if (load && !*dead) tma_load_rows(ring + S::OFF_K8 + b * S::STAGE + lane * box * HD, &kmap, row, sh.k8_full + b);
                if (n >= S::STAGES) wait(sh.v8_empty + b, n / S::STAGES - 1);
                __syncwarp();
                if (lane == 0) {
                    if (boxes) mbar_expect_tx(sh.v8_full + b, boxes * box * HD); else mbar_arrive(sh.v8_full + b);
                }
                __syncwarp();
                if (load && !*dead) tma_load_rows(ring + S::OFF_V8 + b * S::STAGE + lane * box * HD, &vmap, row, sh.v8_full + b);
            }
        }
        if (*dead) {  // copies in flight land before the CTA leaves its shared memory
            for (unsigned i = 0; i < min(n, (unsigned)S::STAGES); ++i) {
                const unsigned k = n - 1 - i;
                mbar_wait_bounded(sh.k8_full + k % S::STAGES, k / S::STAGES & 1);
                mbar_wait_bounded(sh.v8_full + k % S::STAGES, k / S::STAGES & 1);
            }
        }
    } else {
        // ================================================== MMA
        // The warp runs as one and an elected lane issues: operands then sit in uniform registers. (With the role in
        // a branch of one lane an MMA took 135 cycles to issue, four times what it takes to run.)
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t qs = kt_desc(smem_u32(ring + S::OFF_Q), 16), ps = kt_desc(smem_u32(ring + S::OFF_P), S::PB);
        unsigned k_at = 0, period = 0;
        auto scores = [&] {
            const unsigned b = k_at & 1;
            wait(sh.kf_full + b, k_at >> 1);
            if (k_at >= 2) wait(sh.d1_empty + b, (k_at >> 1) - 1);
            kt_fence_after();
            __syncwarp();
            if (kt_elect()) {
                const uint32_t d = tm + S::D1 + b * N, a = tm + S::K + b * (HD / 2);
#pragma unroll
                for (int part = 0; part < QP; ++part)
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k)
                        kt_mma(d, a + 8 * k, qs + (((QP - 1 - part) * S::QB + k / 4 * (N * 128) + k % 4 * 32) >> 4),
                               kt_idesc(N, false), part || k);
                kt_commit(sh.kf_empty + b);
                kt_commit(sh.d1_full + b);
            }
            __syncwarp();
            ++k_at;
        };
        while (const Kv8Segment *s = next()) {
            wait(sh.q_full + (seg & 1), seg >> 1);
            const int tiles = s->t1 - s->t0;
#pragma unroll 1
            for (int t = -1; t < tiles; ++t) {  // scores one tile ahead of values
                if (t + 1 < tiles) scores();
                if (t < 0) continue;
                const unsigned b = n & 1;
                const int step = t % KT_FLUSH;
                if (step == 0 && t > 0) ++period;
                wait(sh.vf_full + b, n >> 1);
                wait(sh.p_full + b, n >> 1);
                kt_fence_after();
                __syncwarp();
                if (kt_elect()) {
                    const uint32_t d = tm + S::D2 + (period & 1) * N, a = tm + S::V + b * (KT_TILE / 2);
                    const uint64_t p = ps + (b * 2 * S::PB >> 4);
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int k = 0; k < KT_TILE / 16; ++k)
                            kt_mma(d, a + 8 * k, p + (((1 - part) * S::PB + k * 2048) >> 4), kt_idesc(N, true), step || part || k);
                    kt_commit(sh.o_done + b);
                }
                __syncwarp();
                ++n;
            }
            ++period;
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
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(S::COLS) : "memory");
    }
}

template <int HD, unsigned FMT, int N, int QP>
int kv8_tiles_go(const Kv8Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned grid, cudaStream_t s)
{
    constexpr size_t smem = 1024 + KtShape<HD, N, QP>::OFF_END + sizeof(KtShared<N>);
    static_assert(smem <= 227 * 1024, "shared memory of one CTA");
    static std::atomic<unsigned> allowed{0};
    if (allow_shared((const void *)kv8_tiles_kernel<HD, FMT, N, QP>, smem, allowed)) return -2;
    kv8_tiles_kernel<HD, FMT, N, QP><<<grid, kt_threads(N), smem, s>>>(A, k, v);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace fyb
