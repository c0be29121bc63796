// kv8_decode.cu - attention over the paged 8-bit cache for up to eight query
// rows per KV head: single tokens of grouped heads, short drafts.
//
//   S^T = K Q^T        16 positions x 8 columns per mma.sync m16n8k16
//   O^T = V^T P^T      16 head dimensions x 8 columns
//
// with K and V converted from 8 bits to fp16 in registers (exact) and q and p
// as two halves each, hi + lo, 22 bits: with up to four rows the eight columns
// are the hi and lo halves of the rows, one MMA for both; with up to eight they
// are the rows, two MMAs into one accumulator. Sums are F32.
//
// Bound by HBM: 2 head_dim bytes per position and KV head, read once for all
// rows. A position's 256 bytes (head_dim 128) pass an SM in 11.6 cycles at the
// measured copy rate, 46 warp instructions; the loop below issues about 15.
// Ragged batch of 32 (128 to 32768 positions, 32/8 heads, 1.05 GB): 173 us, 6.1
// TB/s, 0.94 of a measured copy; 16 requests of 8100 with eight rows: 60 us, 4.4
// TB/s, where the two passes of the low halves and the joins show.
// A producer warp keeps the TMA ring full across segments while four warps take
// 16 positions of every 64-position tile each.
#include "kv8_attention.cuh"

namespace fyb {

constexpr int KD_TILE = 64, KD_WARPS = 4, KD_THREADS = 32 * (KD_WARPS + 1);

template <int HD, int W> struct KdShape {
    static constexpr int STAGE = 2 * KD_TILE * HD;             // K and V bytes
    static constexpr int STAGES = (W == 1 ? 4 : 3) * (128 / HD);  // with the sums of the rows, three CTAs per SM
};
struct KdMeta { float ks[KD_TILE / 16], vs[KD_TILE / 16]; };   // scales of the tile's blocks; ks NaN: block not loaded

FYB_DEV void mma_f16(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two 16 x 16 byte matrices (row addresses from lanes 0..15 and 16..31),
// transposed: lane 4g + t gets column g (r0, r2) and g + 8 (r1, r3) of rows 4t..4t+3.
FYB_DEV void ldmatrix_trans_b8(unsigned (&r)[4], unsigned addr)
{
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
FYB_DEV void ldmatrix_b16(unsigned (&r)[4], unsigned addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
FYB_DEV unsigned movmatrix(unsigned x)
{
    unsigned y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// hi = fp16(w), lo = fp16(w - hi)
FYB_DEV void split_half(float w, __half &hi, __half &lo)
{
    hi = __float2half_rn(w);
    lo = __float2half_rn(w - __half2float(hi));
}
FYB_DEV unsigned pack(__half lo, __half hi)
{
    const __half2 p = __halves2half2(lo, hi);
    return *reinterpret_cast<const unsigned *>(&p);
}
// 2^-(exponent of x) and its inverse for a positive finite x (1 for 0).
FYB_DEV int exponent_of(float x) { return x > 0.f ? max(-126, (int)(__float_as_uint(x) >> 23) - 127) : 0; }
FYB_DEV float power_of_two(int e) { return e < -126 ? __uint_as_float(1u << max(0, e + 149)) : __uint_as_float((unsigned)(min(e, 127) + 127) << 23); }

// W: rows a thread holds scores of (1: up to four query rows, 2: up to eight).
// QL: whether q has low halves of its own (F32 rows at W = 2; 16-bit rows fit
// the high half, and at W = 1 the low halves are columns that cost nothing).
template <int HD, unsigned FMT, int W, bool QL>
__global__ void __launch_bounds__(KD_THREADS, 3) kv8_decode_kernel(const __grid_constant__ Kv8Attention A, const __grid_constant__ CUtensorMap kmap,
    const __grid_constant__ CUtensorMap vmap)
{
    constexpr int R = 4 * W, STAGES = KdShape<HD, W>::STAGES, STAGE = KdShape<HD, W>::STAGE, MT = HD / 16;
    extern __shared__ unsigned char kd_smem[];
    unsigned char *ring = kd_smem + ((1024u - (smem_u32(kd_smem) & 1023u)) & 1023u);
    float *o_s = reinterpret_cast<float *>(ring + STAGES * STAGE);          // [warps][R][HD], then weights of a join
    KdMeta *meta = reinterpret_cast<KdMeta *>(o_s + KD_WARPS * R * HD);     // [stages]
    float2 *ml_s = reinterpret_cast<float2 *>(meta + STAGES);               // [warps][R], then [R]
    uint64_t *full = reinterpret_cast<uint64_t *>(ml_s + KD_WARPS * R), *empty = full + STAGES;
    unsigned *flag = reinterpret_cast<unsigned *>(empty + STAGES);
    volatile unsigned *dead = flag + 1;   // a wait ran out: nobody waits any more, the error word is set
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kv = A.c.kv_heads;
    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(full + i, 2); mbar_init(empty + i, KD_WARPS); }
        *dead = 0;
        fence_barrier_init();
    }
    const Kv8Place place = kv8_place<KD_TILE, KD_THREADS, 5>(A);  // a CTA barrier inside
    Kv8Walk<KD_TILE> walk(A, place);
    Kv8Segment s;
    unsigned stage = 0, phase = 0;
    auto advance = [&] { if (++stage == STAGES) { stage = 0; phase ^= 1; } };
    auto wait = [&](uint64_t *bar, unsigned ph) {
        if (*dead || mbar_wait_bounded(bar, ph)) return;
        *dead = 1;
        if (lane == 0) raise_error(A.error, ERR_TIMEOUT);
    };

    if (warp == KD_WARPS) {
        // ---- producer: block ids and scales 32 blocks at a time, tiles by TMA
        const unsigned size = 1u << A.shift, box = min(size, (unsigned)KD_TILE), per = KD_TILE / box;
        unsigned issued = 0;
        while (walk.next(s)) {
            const int blocks = (kv8_attended(A, s.q, s.row_tile) + (int)size - 1) >> A.shift;
            const int *ids = A.table + (size_t)s.request * A.table_stride;
            int have = -1, id = 0;    // lane holds block 32 * have + lane
            float ks = 0.f, vs = 0.f;
            for (int t = s.t0; t < s.t1; ++t) {
                const int b0 = t * KD_TILE >> A.shift;   // first block of the tile; per of them, or a part of one
                const bool fetch = b0 / 32 != have;
                if (fetch) {
                    have = b0 / 32;
                    const int b = have * 32 + (int)lane;
                    id = b < blocks ? ids[b] : -1;
                    if (b < blocks && (unsigned)id >= A.c.blocks) {  // negative ones too
                        raise_error(A.error, ERR_BOUNDS);
                        id = -1;
                    }
                }
                wait(empty + stage, phase ^ 1);
                const int mine = __shfl_sync(0xffffffffu, id, (b0 & 31) + (int)(lane % per));
                const bool load = lane < per && mine >= 0;
                const unsigned boxes = __popc(__ballot_sync(0xffffffffu, load));
                __syncwarp();
                if (lane == 0) {
                    if (boxes) mbar_expect_tx(full + stage, boxes * 2 * box * HD); else mbar_arrive(full + stage);
                }
                __syncwarp();
                if (load && !*dead) {
                    const int row = (int)((((unsigned)mine * kv + s.head) << A.shift) + ((unsigned)(t * KD_TILE) & (size - 1)));
                    unsigned char *dst = ring + stage * STAGE + lane * box * HD;
                    tma_load_rows(dst, &kmap, row, full + stage);
                    tma_load_rows(dst + KD_TILE * HD, &vmap, row, full + stage);
                }
                // the scales come while the tile does
                if (fetch) {
                    ks = id >= 0 ? A.c.k_scale[(size_t)id * kv + s.head] : NAN;
                    vs = id >= 0 ? A.c.v_scale[(size_t)id * kv + s.head] : 0.f;
                }
                // groups of 16 positions and the blocks they lie in
                const unsigned group_block = (unsigned)(b0 & 31) + (lane % (KD_TILE / 16) * 16 >> min(A.shift, 6u));
                const float gk = __shfl_sync(0xffffffffu, ks, group_block), gv = __shfl_sync(0xffffffffu, vs, group_block);
                if (lane < KD_TILE / 16) { meta[stage].ks[lane] = gk; meta[stage].vs[lane] = gv; }
                __syncwarp();
                if (lane == 0) mbar_arrive(full + stage);
                ++issued;
                advance();
            }
        }
        if (*dead) {  // copies in flight land before the CTA leaves its shared memory
            for (unsigned i = 0; i < min(issued, (unsigned)STAGES); ++i) mbar_wait_bounded(full + i, (issued - 1 - i) / STAGES & 1);
        }
        return;
    }

    // ---- consumers
    const unsigned g = lane >> 2, t4 = lane & 3;
    // matrix row r of the first eight is position r + 8 (r >= 4), of the second r + 4, of a tile's 16: eight
    // different positions modulo 8 in every group of rows that ldmatrix fetches together, for K and for V
    const unsigned posA = warp * 16 + g + (g >= 4 ? 8 : 0), posB = warp * 16 + g + 4;
    const unsigned kr = lane & 7, kpos = warp * 16 + ((lane & 8) ? kr + 4 : kr + (kr >= 4 ? 8 : 0));
    const unsigned k_addr = kpos * HD + ((((lane >> 4) & 1) ^ kv8_swizzle<HD>(kpos)) << 4);
    const unsigned vi = lane & 15, vr = 2 * (vi >> 2) + (vi & 1);
    const unsigned vpos = warp * 16 + ((vi & 2) ? vr + 4 : vr + (vr >= 4 ? 8 : 0));
    const unsigned v_addr = KD_TILE * HD + vpos * HD + (((lane >> 4) ^ kv8_swizzle<HD>(vpos)) << 4);
    constexpr float P_SCALE = 32.f;  // keeps small weights clear of fp16's smallest numbers; the largest is 2^14
    auto bar = [] { asm volatile("bar.sync 1, %0;" :: "n"(32 * KD_WARPS) : "memory"); };

    while (walk.next(s)) {
        const unsigned G = A.group;
        const int j0 = s.row_tile * (int)A.row_tile, nrows = min((int)A.row_tile, s.q.rows - j0) * (int)G;
        auto row_of = [&](unsigned rho, size_t &row, unsigned &head) {
            row = (size_t)(s.q.first + j0 + (int)(rho / G));
            head = s.head * G + rho % G;
        };
        // ---- q: column g of the B fragments, normalized by a power of two and split in halves
        unsigned qh[MT][2], ql[QL ? MT : 1][2];
        float factor[W];  // score factor of this thread's rows
        int limit[W];     // positions they attend
        {
            const unsigned rho = W == 1 ? g >> 1 : g;
            float4 x[MT];
            float top = 0.f;
            if ((int)rho < nrows) {
                size_t row;
                unsigned head;
                row_of(rho, row, head);
#pragma unroll
                for (int k = 0; k < MT; ++k) {
                    x[k] = kv8_load4(A.q, A.type, row * A.q_stride + (size_t)head * HD + 16 * k + 4 * t4);
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w))));
                }
            } else {
#pragma unroll
                for (int k = 0; k < MT; ++k) x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // largest magnitude to [2^12, 2^13): the low halves stay normal numbers of fp16
            const int e = 12 - exponent_of(top);
            const float up = power_of_two(min(e, 127)), up2 = power_of_two(e - min(e, 127));
#pragma unroll
            for (int k = 0; k < MT; ++k) {
                __half h[4], l[4];
                split_half(x[k].x * up * up2, h[0], l[0]);
                split_half(x[k].y * up * up2, h[1], l[1]);
                split_half(x[k].z * up * up2, h[2], l[2]);
                split_half(x[k].w * up * up2, h[3], l[3]);
                if constexpr (W == 1) {
                    const bool low = g & 1;
                    qh[k][0] = low ? pack(l[0], l[1]) : pack(h[0], h[1]);
                    qh[k][1] = low ? pack(l[2], l[3]) : pack(h[2], h[3]);
                } else {
                    qh[k][0] = pack(h[0], h[1]); qh[k][1] = pack(h[2], h[3]);
                    if constexpr (QL) { ql[k][0] = pack(l[0], l[1]); ql[k][1] = pack(l[2], l[3]); }
                }
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                // the lane group that holds query row W t4 + w as its column
                const int er = __shfl_sync(0xffffffffu, e, (int)((W == 1 ? 2 * t4 : 2 * t4 + w) * 4));
                const unsigned mine = W * t4 + w;
                factor[w] = ldexpf(A.scale, -er);
                limit[w] = (int)mine < nrows ? s.q.len - s.q.n + j0 + (int)(mine / G) + 1 : 0;
            }
        }
        const int any = kv8_attended(A, s.q, s.row_tile);                   // positions some row attends
        const int all = max(0, s.q.len - s.q.n + j0 + 1);                    // positions every row attends
        float acc[MT][4], m[W], l[W], vref = 0.f;
        int vexp = -200;  // v scales are relative to 2^vexp
#pragma unroll
        for (int k = 0; k < MT; ++k) acc[k][0] = acc[k][1] = acc[k][2] = acc[k][3] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) { m[w] = -3.4e38f; l[w] = 0.f; }

        for (int t = s.t0; t < s.t1; ++t) {
            wait(full + stage, phase);
            const int base = t * KD_TILE, first = base + (int)warp * 16;
            const float ks = meta[stage].ks[warp], vs = meta[stage].vs[warp];
            if (first < any && !isnan(ks)) {
                const unsigned tile = smem_u32(ring + stage * STAGE);
                // ---- scores
                float c[2][4] = {};  // two chains
#pragma unroll
                for (int k = 0; k < MT; k += 2) {
                    unsigned r[4], a[4], b[4];
                    ldmatrix_b16(r, tile + (k_addr ^ (unsigned)(k / 2) << 5));
                    kv8_halves<FMT>(r[0], a[0], a[2]);
                    kv8_halves<FMT>(r[1], a[1], a[3]);
                    kv8_halves<FMT>(r[2], b[0], b[2]);
                    kv8_halves<FMT>(r[3], b[1], b[3]);
                    mma_f16(c[0], a, qh[k][0], qh[k][1]);
                    mma_f16(c[1], b, qh[k + 1][0], qh[k + 1][1]);
                    if constexpr (QL) {
                        mma_f16(c[0], a, ql[k][0], ql[k][1]);
                        mma_f16(c[1], b, ql[k + 1][0], ql[k + 1][1]);
                    }
                }
                float x[2][W];  // [position A, B][row], in units of log2
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float u = c[0][2 * h] + c[1][2 * h], v = c[0][2 * h + 1] + c[1][2 * h + 1];
                    if constexpr (W == 1) x[h][0] = (u + v) * (factor[0] * ks);
                    else { x[h][0] = u * (factor[0] * ks); x[h][1] = v * (factor[1] * ks); }
                }
                if (first + 16 > all) {
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        if (base + (int)posA >= limit[w]) x[0][w] = -INFINITY;
                        if (base + (int)posB >= limit[w]) x[1][w] = -INFINITY;
                    }
                }
                // ---- running maximum: moved only when a score is 2^8 above it. Their difference says so: it is exact
                // where they are near, and m + 8 is not (from 2^27 on it can round to m + 16, a weight of 2^16)
                bool over = false;
#pragma unroll
                for (int w = 0; w < W; ++w) over = over || fmaxf(x[0][w], x[1][w]) - m[w] > 8.f;
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        float top = fmaxf(x[0][w], x[1][w]);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                        if (top - m[w] > 8.f) {  // each row by its own scores: the same on all lanes that hold it
                            const float alpha = ex2(m[w] - top);
                            m[w] = top;
                            l[w] *= alpha;
#pragma unroll
                            for (int k = 0; k < MT; ++k) {
                                if constexpr (W == 1) { acc[k][0] *= alpha; acc[k][1] *= alpha; acc[k][2] *= alpha; acc[k][3] *= alpha; }
                                else { acc[k][w] *= alpha; acc[k][2 + w] *= alpha; }
                            }
                        }
                    }
                }
                // ---- value scales relative to the largest power of two so far
                const int e = max(exponent_of(vs) + 1, -100);
                if (e > vexp && vs > 0.f) {
                    const float down = vexp < -126 ? 0.f : power_of_two(vexp - e);
#pragma unroll
                    for (int k = 0; k < MT; ++k) { acc[k][0] *= down; acc[k][1] *= down; acc[k][2] *= down; acc[k][3] *= down; }
                    vexp = e;
                    vref = power_of_two(-e) * P_SCALE;
                }
                const float wv = vs * vref;
                unsigned b[2], bl[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    __half ph[W], pl[W];
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const float p = ex2(x[h][w] - m[w]);
                        l[w] += p;
                        split_half(p * wv, ph[w], pl[w]);
                    }
                    if constexpr (W == 1) b[h] = movmatrix(pack(ph[0], pl[0]));
                    else { b[h] = movmatrix(pack(ph[0], ph[1])); bl[h] = movmatrix(pack(pl[0], pl[1])); }
                }
                // ---- values; e4m3 bytes past the last position may be NaN, which 0 x would keep
                unsigned keep = 0xffffffffu;
                if (FMT == FYB_KV8_E4M3 && first + 16 > any) {
                    keep = 0;
                    const int pA = first + 2 * (int)t4 + (t4 >= 2 ? 8 : 0), pB = first + 2 * (int)t4 + 4;
                    if (pA < any) keep |= 0xffu;
                    if (pA + 1 < any) keep |= 0xff00u;
                    if (pB < any) keep |= 0xff0000u;
                    if (pB + 1 < any) keep |= 0xff000000u;
                }
#pragma unroll
                for (int k = 0; k < MT; k += 2) {
                    unsigned r[4], a[4], d[4];
                    ldmatrix_trans_b8(r, tile + (v_addr ^ (unsigned)(k / 2) << 5));
                    if (FMT == FYB_KV8_E4M3) { r[0] &= keep; r[1] &= keep; r[2] &= keep; r[3] &= keep; }
                    kv8_halves<FMT>(r[0], a[0], a[2]);
                    kv8_halves<FMT>(r[1], a[1], a[3]);
                    kv8_halves<FMT>(r[2], d[0], d[2]);
                    kv8_halves<FMT>(r[3], d[1], d[3]);
                    mma_f16(acc[k], a, b[0], b[1]);
                    mma_f16(acc[k + 1], d, b[0], b[1]);
                    if constexpr (W == 2) {
                        mma_f16(acc[k], a, bl[0], bl[1]);
                        mma_f16(acc[k + 1], d, bl[0], bl[1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + stage);
            advance();
        }
        // ---- the four warps' parts: sums over the lanes of a row, then over the warps
        const float back = vexp < -126 ? 0.f : power_of_two(vexp) / P_SCALE;
#pragma unroll
        for (int w = 0; w < W; ++w) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[w] += __shfl_xor_sync(0xffffffffu, l[w], o);
            if (g == 0) ml_s[warp * R + W * t4 + w] = make_float2(m[w], l[w]);
        }
#pragma unroll
        for (int k = 0; k < MT; ++k) {
            if constexpr (W == 1) {
                o_s[(warp * R + t4) * HD + 16 * k + g] = (acc[k][0] + acc[k][1]) * back;
                o_s[(warp * R + t4) * HD + 16 * k + g + 8] = (acc[k][2] + acc[k][3]) * back;
            } else {
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    o_s[(warp * R + 2 * t4 + w) * HD + 16 * k + g] = acc[k][w] * back;
                    o_s[(warp * R + 2 * t4 + w) * HD + 16 * k + g + 8] = acc[k][2 + w] * back;
                }
            }
        }
        bar();
        float2 joined[(R * HD / 4 + 127) / 128];
#pragma unroll
        for (int i = 0; i < (R * HD / 4 + 127) / 128; ++i) {
            const unsigned at = tid + 128 * i, row = at / (HD / 4);
            if (at >= R * HD / 4) break;
            float mm = ml_s[row].x, ll = 0.f;
#pragma unroll
            for (int w = 1; w < KD_WARPS; ++w) mm = fmaxf(mm, ml_s[w * R + row].x);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < KD_WARPS; ++w) {
                const float f = ex2(ml_s[w * R + row].x - mm);
                const float4 y = reinterpret_cast<const float4 *>(o_s)[w * R * HD / 4 + at];
                ll = fmaf(ml_s[w * R + row].y, f, ll);
                v.x = fmaf(y.x, f, v.x); v.y = fmaf(y.y, f, v.y); v.z = fmaf(y.z, f, v.z); v.w = fmaf(y.w, f, v.w);
            }
            reinterpret_cast<float4 *>(o_s)[at] = v;  // this thread alone reads and writes element `at` of warp 0's part
            joined[i] = make_float2(mm, ll);
        }
        bar();
#pragma unroll
        for (int i = 0; i < (R * HD / 4 + 127) / 128; ++i) {
            const unsigned at = tid + 128 * i;
            if (at < R * HD / 4 && at % (HD / 4) == 0) ml_s[at / (HD / 4)] = joined[i];
        }
        bar();
        kv8_finish<R, HD, 32 * KD_WARPS>(A, s, place, tid, ml_s, o_s, (unsigned)nrows, o_s + R * HD,
            (KD_WARPS - 1) * R * HD, flag, bar, [&](unsigned rho, unsigned chunk, float4 v) {
                size_t row;
                unsigned head;
                row_of(rho, row, head);
                kv8_store4(A.out, A.type, row * A.out_stride + (size_t)head * HD + 4 * chunk, v);
            });
        bar();
    }
}

template <int HD, unsigned FMT, int W, bool QL> static int decode_launch(const Kv8Attention &A, const CUtensorMap &k,
    const CUtensorMap &v, unsigned grid, cudaStream_t s)
{
    constexpr int R = 4 * W, STAGES = KdShape<HD, W>::STAGES;
    constexpr size_t smem = 1024 + (size_t)STAGES * KdShape<HD, W>::STAGE + KD_WARPS * R * HD * 4 + STAGES * sizeof(KdMeta) +
                            KD_WARPS * R * 8 + 2 * STAGES * 8 + 16;
    static_assert(smem <= 75 * 1024, "three CTAs per SM");
    static std::atomic<unsigned> allowed{0};
    if (allow_shared((const void *)kv8_decode_kernel<HD, FMT, W, QL>, smem, allowed)) return -2;
    kv8_decode_kernel<HD, FMT, W, QL><<<grid, KD_THREADS, smem, s>>>(A, k, v);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

template <int HD, unsigned FMT> static int decode_rows(const Kv8Attention &A, const CUtensorMap &k, const CUtensorMap &v,
    unsigned grid, cudaStream_t s)
{
    if (A.max_rows * A.group <= 4) return decode_launch<HD, FMT, 1, false>(A, k, v, grid, s);
    return A.type == T_F32 ? decode_launch<HD, FMT, 2, true>(A, k, v, grid, s)
                           : decode_launch<HD, FMT, 2, false>(A, k, v, grid, s);
}

int launch_kv8_decode(const Kv8Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned grid, cudaStream_t s)
{
    const bool e4m3 = A.c.format == FYB_KV8_E4M3;
    if (A.c.head_dim == 128) return e4m3 ? decode_rows<128, FYB_KV8_E4M3>(A, k, v, grid, s) : decode_rows<128, FYB_KV8_INT8>(A, k, v, grid, s);
    return e4m3 ? decode_rows<64, FYB_KV8_E4M3>(A, k, v, grid, s) : decode_rows<64, FYB_KV8_INT8>(A, k, v, grid, s);
}

}  // namespace fyb
