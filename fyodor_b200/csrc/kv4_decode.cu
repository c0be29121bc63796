// kv4_decode.cu - attention over the paged 4-bit cache for up to eight query
// rows per KV head: single tokens of grouped heads, short drafts.
//
// With k = low + scale n in groups of 64 dimensions, and q_g a group's part of q,
//
//   q . k = sum_g scale_g (q_g . n_g) + low_g sum(q_g)
//   o_g   = sum_t (p_t scale_tg) n_tg + sum_t p_t low_tg
//
// so the tensor cores multiply the whole numbers n themselves, S^T = N Q^T and
// O_g^T = N_g^T W_g^T with mma.sync m16n8k16: a masked word of the cache is
// already a pair of fp16 operands, the subnormal n 2^-22 (or 16 n 2^-22 for the upper
// number of a byte, which q and the output take back), with nothing to convert.
// Scales and lows meet the scores and the weights in F32.
//
// The tensor cores line products up by the operands' exponents, and a subnormal's
// is 2^-14 whatever its size: the higher a number's bits lie, the fewer are lost.
// Two bits further down (n 2^-24) a row of F32 of 257 tokens was 1.1e-5 off and not
// 1.6e-6, for 3 us of a ragged batch; numbers made normal, by an addition each, left
// 2.4e-7 and took 28. Sums of n are far larger than an output, and the accumulators round
// towards zero (a row of 30000 is 3.5e-4 off). So V's numbers count up from low in one
// group of 16 positions and down from the highest, with negative weights, in the next (the
// complement is part of the mask); -8 times the weights, by an MMA more each, took 15 us of
// a ragged batch. Five rows and more take that one nevertheless: their weights are
// rounded to one half, an error that goes with the numbers' size (fp16 rows at 8100:
// 2.8e-4 off and not 5.1e-4, for 4 us of 59). F32 rows of five and more, whose low halves
// share the accumulators of the high ones, have V's numbers made normal, less 8.
//
// q and the weights are two fp16 halves, hi + lo, 22 bits: with up to four rows
// the eight columns are the hi and lo halves of the rows, one MMA for both; with up
// to eight they are the rows, with low halves in an MMA of their own for F32 rows.
// Rows of 16 bits fit the high half, and at five rows and more their weights are
// rounded to it (2^-12 each at the most, of no common sign).
//
// Bound by the latency between dependent instructions of 12 consumer warps an SM: issue
// 0.57, the ALU pipe 54 %, no other pipe above that, fixed latencies the largest stall.
// 16 at 8100 with eight rows takes 59 us for 22 of bytes (0.38 of the measured copy), 32
// ragged requests of 128 to 32768 150 us for 99 (0.66). Three CTAs of four consumer warps
// and one for the copies fit an SM at 128 registers (when they took 147 us two CTAs of
// eight took 175, four of four, with fewer registers, 162).
#include "kv4_attention.cuh"

namespace fyb {

// SHARE: groups of 16 positions of a tile that a warp takes
constexpr int K4_COST = 3;  // a segment's beginning and end, in tiles (ragged 32 without them 147 us, with them 140, when it was measured)
constexpr int K4_WARPS = 4, K4_SHARE = K4_TILE / 16 / K4_WARPS, K4_THREADS = 32 * (K4_WARPS + 1);

// Words of shared memory: the address of a lane, and what is the same for all of them as the offset.
FYB_DEV void lds(unsigned (&x)[4], unsigned at, unsigned off) { asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at + off)); }
FYB_DEV void lds(unsigned (&x)[2], unsigned at, unsigned off) { asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(at + off)); }
FYB_DEV void lds(unsigned (&x)[1], unsigned at, unsigned off) { asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x[0]) : "r"(at + off)); }
FYB_DEV unsigned pack2(float lo, float hi)  // fp16 pair
{
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned *>(&p);
}
FYB_DEV float2 unpack2(unsigned p) { return __half22float2(*reinterpret_cast<const __half2 *>(&p)); }

// The lower (upper) numbers of two bytes of a word, 16 bits apart, less 8: a number under the bits of 1024 (of 64) is that
// much more, taken off exactly.
FYB_DEV unsigned lower8(unsigned x)
{
    const unsigned y = (x & 0x000f000fu) | 0x64006400u;
    const __half2 n = __hadd2(*reinterpret_cast<const __half2 *>(&y), __float2half2_rn(-1032.f));
    return *reinterpret_cast<const unsigned *>(&n);
}
FYB_DEV unsigned upper8(unsigned x)
{
    const unsigned y = (x & 0x00f000f0u) | 0x54005400u;
    const __half2 n = __hadd2(*reinterpret_cast<const __half2 *>(&y), __float2half2_rn(-72.f));
    return *reinterpret_cast<const unsigned *>(&n);
}

template <int HD> struct K4Shape {
    static constexpr int ROW = HD / 2, SCALES = HD / 64 * 4;               // bytes of a token's row, of its scales
    static constexpr int OFF_V = K4_TILE * ROW, OFF_KS = 2 * OFF_V, OFF_VS = OFF_KS + K4_TILE * SCALES,
                         STAGE = OFF_VS + K4_TILE * SCALES, STAGES = 3 * (128 / HD);
};

// W: rows a thread holds scores of (1: up to four query rows, 2: up to eight). LO: whether q and the weights have low
// halves at W = 2 (at W = 1 they are columns that cost nothing).
template <int HD, int W, bool LO>
__global__ void __launch_bounds__(K4_THREADS, K4_CTAS) kv4_decode_kernel(const __grid_constant__ Kv4Attention A, const __grid_constant__ CUtensorMap kmap,
    const __grid_constant__ CUtensorMap vmap)
{
    using S = K4Shape<HD>;
    constexpr int R = 4 * W, G = HD / 64, NW = HD / 32, J = W == 1 ? 2 : 1;  // NW: words of K a thread takes of a token
    extern __shared__ unsigned char k4_smem[];
    unsigned char *ring = k4_smem + ((1024u - (smem_u32(k4_smem) & 1023u)) & 1023u);
    float *o_s = reinterpret_cast<float *>(ring + S::STAGES * S::STAGE);    // [warps][R][HD], then weights of a join
    float2 *ml_s = reinterpret_cast<float2 *>(o_s + K4_WARPS * R * HD);     // [warps][R], then [R]
    uint64_t *full = reinterpret_cast<uint64_t *>(ml_s + K4_WARPS * R), *empty = full + S::STAGES;
    unsigned *here = reinterpret_cast<unsigned *>(empty + S::STAGES);       // [stages] which groups of 16 positions are loaded
    unsigned *flag = here + S::STAGES;
    volatile unsigned *dead = flag + 1;   // a wait ran out: nobody waits any more, the error word is set
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kv = A.c.kv_heads / A.split;
    if (tid == 0) {
        for (int i = 0; i < S::STAGES; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, K4_WARPS); }
        *dead = 0;
        fence_barrier_init();
    }
    const Kv8Place place = kv8_place<K4_TILE, K4_THREADS, 5, K4_COST>(A);  // a CTA barrier inside
    Kv8Walk<K4_TILE, K4_COST> walk(A, place);
    Kv8Segment s;
    unsigned stage = 0, phase = 0;
    auto advance = [&] { if (++stage == S::STAGES) { stage = 0; phase ^= 1; } };
    auto wait = [&](uint64_t *bar, unsigned ph) {
        if (*dead || mbar_wait_bounded(bar, ph)) return;
        *dead = 1;
        if (lane == 0) raise_error(A.error, ERR_TIMEOUT);
    };

    if (warp == K4_WARPS) {
        // ---- producer: block ids 32 at a time, tiles and scales by bulk copies
        const unsigned size = 1u << A.shift, box = min(size, (unsigned)K4_TILE), per = K4_TILE / box;
        unsigned issued = 0;
        while (walk.next(s)) {
            const int blocks = (kv8_attended(A, s.q, s.row_tile) + (int)size - 1) >> A.shift;
            const int *ids = A.table + (size_t)s.request * A.table_stride;
            int have = -1, id = 0;    // lane holds block 32 * have + lane
            for (int t = s.t0; t < s.t1; ++t) {
                const int b0 = t * K4_TILE >> A.shift;   // first block of the tile; `per` of them, or a part of one
                if (b0 / 32 != have) {
                    have = b0 / 32;
                    const int b = have * 32 + (int)lane;
                    id = b < blocks ? ids[b] : -1;
                    if (b < blocks && (unsigned)id >= A.c.blocks) {  // negative ones too
                        raise_error(A.error, ERR_BOUNDS);
                        id = -1;
                    }
                }
                wait(empty + stage, phase ^ 1);
                const int block = __shfl_sync(0xffffffffu, id, (b0 & 31) + (int)(lane % per));
                const bool load = lane < per && block >= 0;
                const unsigned boxes = __ballot_sync(0xffffffffu, load);
                // groups of 16 positions whose block is among the loaded ones
                const unsigned groups = __ballot_sync(0xffffffffu, lane < K4_TILE / 16 && (boxes >> (lane * 16 / box) & 1));
                if (lane == 0) {
                    here[stage] = groups;
                    if (boxes) mbar_expect_tx(full + stage, __popc(boxes) * 2 * box * (S::ROW + S::SCALES)); else mbar_arrive(full + stage);
                }
                __syncwarp();
                if (load && !*dead) {
                    const unsigned row = (((unsigned)block * kv + s.head / A.split) << A.shift) + ((unsigned)(t * K4_TILE) & (size - 1));  // a token
                    const unsigned dst = smem_u32(ring + stage * S::STAGE), at = lane * box, bar = smem_u32(full + stage);
                    k4_load_rows(dst + at * S::ROW, &kmap, (int)(row / (128 / S::ROW)), bar);
                    k4_load_rows(dst + S::OFF_V + at * S::ROW, &vmap, (int)(row / (128 / S::ROW)), bar);
                    k4_copy(dst + S::OFF_KS + at * S::SCALES, A.ks + (size_t)row * G, box * S::SCALES, bar);
                    k4_copy(dst + S::OFF_VS + at * S::SCALES, A.vs + (size_t)row * G, box * S::SCALES, bar);
                }
                __syncwarp();
                ++issued;
                advance();
            }
        }
        if (*dead) {  // copies in flight land before the CTA leaves its shared memory
            for (unsigned i = 0; i < min(issued, (unsigned)S::STAGES); ++i) mbar_wait_bounded(full + i, (issued - 1 - i) / S::STAGES & 1);
        }
        return;
    }

    // ---- consumers
    const unsigned g = lane >> 2, t4 = lane & 3;
    // Positions of a tile's 16 in the order of the MMAs: a thread has, of K, rows tau and tau + 8, of V rows ta, ta ^ X
    // and both + 8 (the same as k indexes 2 t4, 2 t4 + 1 and both + 8). Chosen so that what one phase of a load reads lies
    // in different banks.
    constexpr unsigned X = HD == 128 ? 3 : 7;
    auto order = [](unsigned t) { return HD == 128 ? (t & 1) + 4 * (t >> 1) : t; };
    const unsigned ta = order(t4), tau = order(g >> 1) ^ (g & 1 ? X : 0u);
    // this lane's place in a tile: of K, of V (two rows), of scales; eight rows further on it is `ahead` away
    const unsigned mine = smem_u32(ring) + warp * K4_SHARE * 16 * S::ROW;
    const unsigned k_at = mine + kv4_at<HD>(tau, 4 * NW * t4), v_at0 = mine + S::OFF_V + kv4_at<HD>(ta, 4 * G * g), v_at1 = mine + S::OFF_V + kv4_at<HD>(ta ^ X, 4 * G * g);
    auto ahead = [](unsigned at, unsigned tile, unsigned eights) {  // rows of 128 bytes move by 8 ROW / 128 each, and the swizzle with them
        return (at ^ (eights * (8 * S::ROW / 128) % 8 << 4)) + eights * 8 * S::ROW + tile;
    };
    const unsigned s_at = smem_u32(ring) + S::OFF_KS + (warp * K4_SHARE * 16 + tau) * S::SCALES;
    // Weights are up to 2^LAG, and P_SCALE times themselves in fp16, so below 2^15. What both halves lose is 2^-25 of that at
    // the most, 2^-38 of the largest weight: there are many of the smallest in a long row.
    constexpr float LAG = 2.f, P_SCALE = 8192.f;
    constexpr int FLUSH = 8;
    const unsigned minus8[4] = {0x80208020u, 0x82008200u, 0x80208020u, 0x82008200u};  // as numbers lie in the operands
    constexpr bool SUMS = W == 1 || LO;
    auto bar = [] { asm volatile("bar.sync 1, %0;" :: "n"(32 * K4_WARPS) : "memory"); };

    while (walk.next(s)) {
        const unsigned GR = A.group;
        const int j0 = s.row_tile * (int)A.row_tile, nrows = min((int)A.row_tile, s.q.rows - j0) * (int)GR;
        auto row_of = [&](unsigned rho, size_t &row, unsigned &head) {
            row = (size_t)(s.q.first + j0 + (int)(rho / GR));
            head = s.head * GR + rho % GR;
        };
        // ---- q: column g of the B fragments, normalized by a power of two and split in halves
        unsigned qh[2 * NW][2], ql[LO ? 2 * NW : 1][2];
        float fn[W], fq[W][G];  // score factors of this thread's rows, and times the sums of q
        int limit[W];           // positions they attend
        {
            const unsigned rho = W == 1 ? g >> 1 : g;
            float x[NW][8];
            float top = 0.f, sum[G] = {};
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
                if ((int)rho < nrows) {
                    size_t row;
                    unsigned head;
                    row_of(rho, row, head);
                    const size_t at = row * A.q_stride + (size_t)head * HD + 64 * (i % G) + 16 * t4 + 8 * (i / G);
                    a = kv8_load4(A.q, A.type, at);
                    b = kv8_load4(A.q, A.type, at + 4);
                }
                x[i][0] = a.x; x[i][1] = a.y; x[i][2] = a.z; x[i][3] = a.w;
                x[i][4] = b.x; x[i][5] = b.y; x[i][6] = b.z; x[i][7] = b.w;
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[i][j]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // largest magnitude to [2^12, 2^13): the low halves stay normal numbers of fp16
            const int e = 12 - exponent_of(top);
            const float up = power_of_two(min(e, 127)), up2 = power_of_two(e - min(e, 127));
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                __half h[8], l[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = x[i][j] * up * up2;
                    sum[i % G] += y;
                    split_half(j & 1 ? y * 0.0625f : y, h[j], l[j]);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const unsigned h0 = pack(h[2 * j], h[2 * j + 4]), h1 = pack(h[2 * j + 1], h[2 * j + 5]);
                    const unsigned l0 = pack(l[2 * j], l[2 * j + 4]), l1 = pack(l[2 * j + 1], l[2 * j + 5]);
                    const bool low = W == 1 && (g & 1);
                    qh[2 * i + j][0] = low ? l0 : h0;
                    qh[2 * i + j][1] = low ? l1 : h1;
                    if constexpr (LO) { ql[2 * i + j][0] = l0; ql[2 * i + j][1] = l1; }
                }
            }
#pragma unroll
            for (int h = 0; h < G; ++h) {
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                // the lane group that holds query row W t4 + w as its column
                const int from = (int)((W == 1 ? 2 * t4 : 2 * t4 + w) * 4);
                const unsigned mine = W * t4 + w;
                fn[w] = ldexpf(A.scale, -__shfl_sync(0xffffffffu, e, from));
#pragma unroll
                for (int h = 0; h < G; ++h) fq[w][h] = fn[w] * __shfl_sync(0xffffffffu, sum[h], from);
                limit[w] = (int)mine < nrows ? s.q.len - s.q.n + j0 + (int)(mine / GR) + 1 : 0;
            }
        }
        const int any = kv8_attended(A, s.q, s.row_tile);                   // positions some row attends
        const int all = max(0, s.q.len - s.q.n + j0 + 1);                    // positions every row attends
        float acc[G][4][4], m[W], l[W], zero[W][G], vref = 0.f;              // zero: sums of p low
        int vexp = -200;  // v scales are relative to 2^vexp
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[h][k][0] = acc[h][k][1] = acc[h][k][2] = acc[h][k][3] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            m[w] = -3.4e38f;
            l[w] = 0.f;
#pragma unroll
            for (int h = 0; h < G; ++h) zero[w][h] = 0.f;
        }

        // The accumulators go to this thread's sums in shared memory: every FLUSH tiles, as they round towards zero (once a
        // segment ragged 32 was 6.2e-6 off when it was 3.7e-6 so, for 4 us of 162); with five to eight rows of 16 bits once, at
        // the segment's end.
        auto sum_of = [&](int h, int k, int w) {
            return reinterpret_cast<float2 *>(o_s + (warp * R + W * t4 + w) * HD + 64 * h + 8 * g + 2 * k);
        };
        auto flush = [&](bool first) {
            const float back = vexp < -126 ? 0.f : power_of_two(vexp) * ((LO ? 1.f : 4194304.f) / P_SCALE), back16 = LO ? back : back * 0.0625f;
#pragma unroll
            for (int h = 0; h < G; ++h)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float (&a)[4] = acc[h][k];
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const float even = W == 1 ? a[0] + a[1] : a[w], odd = W == 1 ? a[2] + a[3] : a[2 + w];
                        float2 *o = sum_of(h, k, w);
                        const float2 y = first ? make_float2(0.f, 0.f) : *o;
                        *o = make_float2(fmaf(even, back, y.x), fmaf(odd, back16, y.y));
                    }
                    a[0] = a[1] = a[2] = a[3] = 0.f;
                }
        };
        if (SUMS) flush(true);
        for (int t = s.t0, left = FLUSH; t < s.t1; ++t, --left) {
            if (SUMS && left == 0) {
                flush(false);
                left = FLUSH;
            }
            wait(full + stage, phase);
            const unsigned tile = stage * S::STAGE;
            const unsigned loaded = here[stage];
#pragma unroll 1
            for (int u0 = 0; u0 < K4_SHARE; u0 += J) {
                // J groups of 16 positions at a time, from position `first`
                const unsigned in_tile = (warp * K4_SHARE + (unsigned)u0) * 16, use = loaded >> (in_tile / 16) & ((1u << J) - 1);
                const int first = t * K4_TILE + (int)in_tile;
                if (first >= any || !use) continue;
                // up to four rows: every other 16 positions count down from 15, with negative weights; else from 8
                auto down = [](int u) { return W == 1 && u == 1; };
                auto base = [&](int u) { return W == 2 ? 8.f : down(u) ? 15.f : 0.f; };
                // ---- scores
                float c[J][G][4];
#pragma unroll
                for (int u = 0; u < J; ++u) {
#pragma unroll
                    for (int h = 0; h < G; ++h) c[u][h][0] = c[u][h][1] = c[u][h][2] = c[u][h][3] = 0.f;
                    unsigned ka[NW], kb[NW];
                    lds(ka, ahead(k_at, tile, (u0 + u) * 2), 0);
                    lds(kb, ahead(k_at, tile, (u0 + u) * 2 + 1), 0);
#pragma unroll
                    for (int i = 0; i < NW; ++i) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const unsigned x = j ? ka[i] >> 6 : ka[i] * 4, y = j ? kb[i] >> 6 : kb[i] * 4;
                            const unsigned a[4] = {x & 0x003c003cu, y & 0x003c003cu, x & 0x03c003c0u, y & 0x03c003c0u};
                            mma_f16(c[u][i % G], a, qh[2 * i + j][0], qh[2 * i + j][1]);
                            if constexpr (LO) mma_f16(c[u][i % G], a, ql[2 * i + j][0], ql[2 * i + j][1]);
                        }
                    }
                }
                // ---- scales and lows of this thread's positions; what is not attended may hold anything
                float2 ks[J][2][G], vs[J][2][G];
#pragma unroll
                for (int u = 0; u < J; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        unsigned kw[G], vw[G];
                        lds(kw, s_at + tile, ((u0 + u) * 16 + 8 * h) * S::SCALES);
                        lds(vw, s_at + tile, ((u0 + u) * 16 + 8 * h) * S::SCALES + S::OFF_VS - S::OFF_KS);
#pragma unroll
                        for (int i = 0; i < G; ++i) {
                            ks[u][h][i] = __half22float2(*reinterpret_cast<const __half2 *>(&kw[i]));
                            vs[u][h][i] = __half22float2(*reinterpret_cast<const __half2 *>(&vw[i]));
                            vs[u][h][i].y = fmaf(base(u), vs[u][h][i].x, vs[u][h][i].y);  // the value of that number
                        }
                    }
                float x[J][2][W];  // [group of 16][position tau, tau + 8][row], in units of log2
#pragma unroll
                for (int u = 0; u < J; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int w = 0; w < W; ++w) {
                            float dot = 0.f, low = 0.f;
#pragma unroll
                            for (int i = 0; i < G; ++i) {
                                const float n = W == 1 ? c[u][i][2 * h] + c[u][i][2 * h + 1] : c[u][i][2 * h + w];
                                dot = fmaf(n, ks[u][h][i].x, dot);
                                low = fmaf(ks[u][h][i].y, fq[w][i], low);
                            }
                            x[u][h][w] = fmaf(dot * 4194304.f, fn[w], low);  // n was 2^22 too small
                        }
                if (first + 16 * J > all || use != (1u << J) - 1) {
#pragma unroll
                    for (int u = 0; u < J; ++u)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int pos = first + 16 * u + (int)tau + 8 * h;
                            const bool is = use >> u & 1;
#pragma unroll
                            for (int w = 0; w < W; ++w)
                                if (pos >= limit[w] || !is) x[u][h][w] = -INFINITY;
                            if (pos >= any || !is) {
#pragma unroll
                                for (int i = 0; i < G; ++i) vs[u][h][i] = make_float2(0.f, 0.f);
                            }
                        }
                }
                // ---- running maximum: moved only when a weight is 2^LAG. The scores' difference says so: it is exact where
                // they are near, and m + LAG is not (from 2^25 on it can round to m + 4, a weight of 2^4)
                bool over = false;
                float top[W];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    top[w] = fmaxf(x[0][0][w], x[0][1][w]);
                    if constexpr (J == 2) top[w] = fmaxf(top[w], fmaxf(x[J - 1][0][w], x[J - 1][1][w]));
                    over = over || top[w] - m[w] > LAG;
                }
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int w = 0; w < W; ++w) {
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], o));
                        if (top[w] - m[w] > LAG) {  // each row by its own scores: the same on all lanes that hold it
                            const float alpha = ex2(m[w] - top[w]);
                            m[w] = top[w];
                            l[w] *= alpha;
#pragma unroll
                            for (int h = 0; h < G; ++h) {
                                zero[w][h] *= alpha;
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    if (SUMS) {
                                        float2 *o = sum_of(h, k, w);
                                        *o = make_float2(o->x * alpha, o->y * alpha);
                                    }
                                    if constexpr (W == 1) { acc[h][k][0] *= alpha; acc[h][k][1] *= alpha; acc[h][k][2] *= alpha; acc[h][k][3] *= alpha; }
                                    else { acc[h][k][w] *= alpha; acc[h][k][2 + w] *= alpha; }
                                }
                            }
                        }
                    }
                }
                // ---- value scales relative to the largest power of two so far (they are not negative: ordered as integers)
                float most = 0.f;
#pragma unroll
                for (int u = 0; u < J; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < G; ++i) most = fmaxf(most, vs[u][h][i].x);
                most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
                const int e = exponent_of(most) + 1;
                if (e > vexp && most > 0.f) {
                    const float down = vexp < -126 ? 0.f : power_of_two(vexp - e);
#pragma unroll
                    for (int h = 0; h < G; ++h)
#pragma unroll
                        for (int k = 0; k < 4; ++k) { acc[h][k][0] *= down; acc[h][k][1] *= down; acc[h][k][2] *= down; acc[h][k][3] *= down; }
                    vexp = e;
                    vref = power_of_two(-e) * P_SCALE;
                }
                // ---- weights and values
#pragma unroll
                for (int u = 0; u < J; ++u) {
                    unsigned b[G][2], bl[G][2];
                    float p[2][W];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int w = 0; w < W; ++w) {
                            p[h][w] = ex2(x[u][h][w] - m[w]);
                            l[w] += p[h][w];
                        }
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        float wt[2][W];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float unit = vs[u][h][i].x * (down(u) ? -vref : vref);
#pragma unroll
                            for (int w = 0; w < W; ++w) {
                                zero[w][i] = fmaf(p[h][w], vs[u][h][i].y, zero[w][i]);
                                wt[h][w] = p[h][w] * unit;
                            }
                        }
                        if constexpr (W == 1) {  // columns: high and low half of a row
                            const unsigned hi = pack2(wt[0][0], wt[1][0]);
                            const float2 back = unpack2(hi);
                            const unsigned lo = pack2(wt[0][0] - back.x, wt[1][0] - back.y);
                            b[i][0] = movmatrix(__byte_perm(hi, lo, 0x5410));
                            b[i][1] = movmatrix(__byte_perm(hi, lo, 0x7632));
                        } else {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const unsigned hi = pack2(wt[h][0], wt[h][W - 1]);
                                b[i][h] = movmatrix(hi);
                                if constexpr (LO) {
                                    const float2 back = unpack2(hi);
                                    bl[i][h] = movmatrix(pack2(wt[h][0] - back.x, wt[h][W - 1] - back.y));
                                }
                            }
                        }
                    }
                    unsigned v[4][G];  // eight numbers of each group of positions ta, ta ^ X, and both + 8
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        lds(v[i], ahead(i & 1 ? v_at1 : v_at0, tile, (u0 + u) * 2 + (i >> 1)), 0);
#pragma unroll
                    for (int i = 0; i < G; ++i)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const unsigned ab = __byte_perm(v[0][i], v[1][i], half ? 0x7632 : 0x5410);
                            const unsigned cd = __byte_perm(v[2][i], v[3][i], half ? 0x7632 : 0x5410);
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                float (&o)[4] = acc[i][2 * half + j];
                                if constexpr (LO) {
                                    const unsigned y = ab >> (8 * j), z = cd >> (8 * j);
                                    const unsigned a[4] = {lower8(y), upper8(y), lower8(z), upper8(z)};
                                    mma_f16(o, a, b[i][0], b[i][1]);
                                    mma_f16(o, a, bl[i][0], bl[i][1]);
                                } else {
                                    const unsigned y = j ? ab >> 6 : ab * 4, z = j ? cd >> 6 : cd * 4, turn = down(u) ? ~0u : 0u;
                                    const unsigned a[4] = {(y ^ turn) & 0x003c003cu, (y ^ turn) & 0x03c003c0u, (z ^ turn) & 0x003c003cu, (z ^ turn) & 0x03c003c0u};
                                    if constexpr (W == 2) mma_f16(o, minus8, b[i][0], b[i][1]);
                                    mma_f16(o, a, b[i][0], b[i][1]);
                                }
                            }
                        }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + stage);
            advance();
        }
        // ---- the warps' parts: sums over the lanes of a row, then over the warps
        flush(!SUMS);
#pragma unroll
        for (int w = 0; w < W; ++w) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                l[w] += __shfl_xor_sync(0xffffffffu, l[w], o);
#pragma unroll
                for (int h = 0; h < G; ++h) zero[w][h] += __shfl_xor_sync(0xffffffffu, zero[w][h], o);
            }
            if (g == 0) ml_s[warp * R + W * t4 + w] = make_float2(m[w], l[w]);
        }
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    float2 *o = sum_of(h, k, w);
                    *o = make_float2(o->x + zero[w][h], o->y + zero[w][h]);
                }
        bar();
        kv8_join_warps<R, HD, K4_WARPS>(tid, ml_s, o_s, bar);
        kv8_finish<R, HD, 32 * K4_WARPS>(A, s, place, tid, ml_s, o_s, (unsigned)nrows, o_s + R * HD,
            (K4_WARPS - 1) * R * HD, flag, bar, [&](unsigned rho, unsigned chunk, float4 v) {
                size_t row;
                unsigned head;
                row_of(rho, row, head);
                kv8_store4(A.out, A.type, row * A.out_stride + (size_t)head * HD + 4 * chunk, v);
            });
        bar();
    }
}

template <int HD, int W, bool LO> static int decode_launch(const Kv4Attention &A, const CUtensorMap &k, const CUtensorMap &v,
    unsigned grid, cudaStream_t s)
{
    using S = K4Shape<HD>;
    constexpr int R = 4 * W;
    constexpr size_t smem = 1024 + (size_t)S::STAGES * S::STAGE + K4_WARPS * R * HD * 4 + K4_WARPS * R * 8 + S::STAGES * 20 + 16;
    static_assert(smem <= 227 * 1024 / K4_CTAS - 1024, "CTAs of an SM");
    static std::atomic<unsigned> allowed{0};
    if (allow_shared((const void *)kv4_decode_kernel<HD, W, LO>, smem, allowed)) return -2;
    kv4_decode_kernel<HD, W, LO><<<grid, K4_THREADS, smem, s>>>(A, k, v);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

template <int HD> static int decode_rows(const Kv4Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned grid, cudaStream_t s)
{
    if (A.row_tile * A.group <= 4) return decode_launch<HD, 1, false>(A, k, v, grid, s);
    return A.type == T_F32 ? decode_launch<HD, 2, true>(A, k, v, grid, s) : decode_launch<HD, 2, false>(A, k, v, grid, s);
}

int launch_kv4_decode(const Kv4Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned grid, cudaStream_t s)
{
    return A.c.head_dim == 128 ? decode_rows<128>(A, k, v, grid, s) : decode_rows<64>(A, k, v, grid, s);
}

}  // namespace fyb
