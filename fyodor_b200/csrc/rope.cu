// rope.cu - rotary positions of q and k rows, and the frequencies and tables
// they are turned by.
//
// A pair (a, b) of a head becomes (a cos t - b sin t, a sin t + b cos t) with
// t = position * freq[pair], the engine's rotation (llm_cpu.c:298-327) for
// interleaved pairs, for half pairs (j, j + dims / 2) and for heads of which
// only the first dims are rotated. Three flops a value: bound by memory, q and
// k read and written once; cosines and sines come from tables [position][pair]
// (one row of them serves every head of a token and stays in L1).
#include "rope.cuh"
#include "fyodor_b200.h"
#include <cmath>

namespace fyb {

constexpr unsigned ROPE_THREADS = 256;

// Grid (rows, items of a row / 256): thread = one item of up to HU heads of q or k.
template <typename T, int V, bool VEC, int HU>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(RopeTable tab, const int *positions, RopeRows q, RopeRows k,
    unsigned hd, RopeWork work, unsigned *error)
{
    const size_t row = blockIdx.x;
    const unsigned i = blockIdx.y * ROPE_THREADS + threadIdx.x;
    const int pos = positions[row];
    const unsigned q_groups = (q.heads + HU - 1) / HU, k_groups = (k.heads + HU - 1) / HU;
    unsigned group, item;
    if (!rope_place(work, q_groups + k_groups, i, group, item)) return;
    const bool is_q = group < q_groups;
    const RopeRows &r = is_q ? q : k;
    if (!is_q) group -= q_groups;
    const unsigned head = group, groups = is_q ? q_groups : k_groups;  // heads group, group + groups, ...
    const T *in = static_cast<const T *>(r.in) + row * r.in_stride + (size_t)head * hd;
    T *out = static_cast<T *>(r.out) + row * r.out_stride + (size_t)head * hd;
    rope_item<T, V, VEC, HU>(in, out, (size_t)groups * hd, (r.heads - head + groups - 1) / groups, tab.dims, tab.layout,
        item, [&](const float *&c, const float *&s) {
            if (pos < 0 || (unsigned)pos >= tab.rows) {
                if (i == 0) raise_error(error, ERR_BOUNDS);
                return false;
            }
            const size_t t = (size_t)pos * (tab.dims / 2);
            c = tab.cos + t;
            s = tab.sin + t;
            return true;
        });
}

// Many rows: a CTA takes row after row through shared memory, whole rows of q
// and k and their two table rows in and out by bulk copies (ROPE_STAGES rows at
// a time), and turns the pairs where they lie. Parts of a head that are only
// copied cost no instruction, and the loads do not wait for the threads: 64 / 8
// heads of 128, 8191 bf16 rows, 52 us against 78 us of rope_kernel.
constexpr int ROPE_STAGES = 4;
struct RopeStage {
    unsigned q_bytes, k_bytes, t_bytes, bytes;  // of a row of q, of k, of a table; of a stage
};
template <typename T, int V>
__global__ void __launch_bounds__(ROPE_THREADS) rope_rows_kernel(RopeTable tab, const int *positions, size_t rows,
    RopeRows q, RopeRows k, unsigned hd, RopeWork work, RopeStage st, unsigned *error)
{
    extern __shared__ __align__(128) unsigned char rope_smem[];
    __shared__ uint64_t full[ROPE_STAGES];
    __shared__ int pos_s[ROPE_STAGES];
    __shared__ unsigned dead;
    const unsigned tid = threadIdx.x, heads = q.heads + k.heads;
    const size_t mine = blockIdx.x < rows ? (rows - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
    auto row_of = [&](size_t i) { return blockIdx.x + i * gridDim.x; };
    if (tid == 0) {
        for (int i = 0; i < ROPE_STAGES; ++i) mbar_init(full + i, 1);
        dead = 0;
        fence_barrier_init();
    }
    __syncthreads();
    // thread 0: row i into its stage
    auto load = [&](size_t i, int pos) {
        const unsigned s = (unsigned)(i % ROPE_STAGES);
        unsigned char *base = rope_smem + (size_t)s * st.bytes;
        const size_t row = row_of(i);
        const bool turns = pos >= 0 && (unsigned)pos < tab.rows;
        pos_s[s] = turns ? pos : -1;
        if (!turns) raise_error(error, ERR_BOUNDS);
        mbar_expect_tx(full + s, st.q_bytes + st.k_bytes + (turns ? 2 * st.t_bytes : 0));
        if (q.heads) bulk_copy_g2s(base, static_cast<const T *>(q.in) + row * q.in_stride, st.q_bytes, full + s);
        if (k.heads) bulk_copy_g2s(base + st.q_bytes, static_cast<const T *>(k.in) + row * k.in_stride, st.k_bytes, full + s);
        if (turns) {
            const size_t t = (size_t)pos * (tab.dims / 2);
            bulk_copy_g2s(base + st.q_bytes + st.k_bytes, tab.cos + t, st.t_bytes, full + s);
            bulk_copy_g2s(base + st.q_bytes + st.k_bytes + st.t_bytes, tab.sin + t, st.t_bytes, full + s);
        }
    };
    int ahead = 0;  // position of the row that is loaded next
    if (tid == 0) {
        for (size_t i = 0; i + 1 < ROPE_STAGES && i < mine; ++i) load(i, positions[row_of(i)]);
        if (ROPE_STAGES - 1 < mine) ahead = positions[row_of(ROPE_STAGES - 1)];
    }
    const unsigned per_row = heads * work.turned;
    size_t i = 0;
    for (; i < mine; ++i) {
        const unsigned s = (unsigned)(i % ROPE_STAGES);
        unsigned char *base = rope_smem + (size_t)s * st.bytes;
        const bool here = mbar_wait_bounded(full + s, (unsigned)(i / ROPE_STAGES) & 1);
        if (!here) dead = 1;
        const bool turns = pos_s[s] >= 0;
        if (turns) {
            const float *c = reinterpret_cast<const float *>(base + st.q_bytes + st.k_bytes);
            const float *sn = reinterpret_cast<const float *>(base + st.q_bytes + st.k_bytes + st.t_bytes);
            T *values = reinterpret_cast<T *>(base);  // q's heads, then k's
            for (unsigned j = tid; j < per_row; j += ROPE_THREADS) {
                T *head = values + (size_t)(j / work.turned) * hd;
                rope_item<T, V, true, 1>(head, head, 0, 1, tab.dims, tab.layout, j % work.turned,
                    [&](const float *&a, const float *&b) { a = c; b = sn; return true; });
            }
        }
        fence_proxy_async();
        if (__syncthreads_or(dead != 0)) break;
        if (tid == 0) {
            if (turns) {
                const size_t row = row_of(i);
                if (q.heads) bulk_copy_s2g(static_cast<T *>(q.out) + row * q.out_stride, base, st.q_bytes);
                if (k.heads) bulk_copy_s2g(static_cast<T *>(k.out) + row * k.out_stride, base + st.q_bytes, st.k_bytes);
            }
            bulk_commit();
            // the row before has left its stage: the next row but two goes there
            bulk_read<1>();
            const size_t next = i + ROPE_STAGES - 1;
            if (next < mine) {
                load(next, ahead);
                if (next + 1 < mine) ahead = positions[row_of(next + 1)];
            }
        }
    }
    if (tid == 0) {
        if (i < mine) {  // a wait ran out: the copies in flight land before the CTA leaves its shared memory
            raise_error(error, ERR_TIMEOUT);
            for (size_t n = i + 1; n < mine && n < i + ROPE_STAGES - 1; ++n)
                mbar_wait_bounded(full + n % ROPE_STAGES, (unsigned)(n / ROPE_STAGES) & 1);
        }
        bulk_drain();
    }
}

// cos / sin of (float)(first + row) * freq[j], the engine's F32 angle.
__global__ void rope_table_kernel(const float *freq, unsigned pairs, float magnitude, unsigned first, size_t count,
    float *c, float *s)
{
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (size_t)gridDim.x * blockDim.x) {
        const float angle = __fmul_rn((float)(first + (unsigned)(i / pairs)), freq[i % pairs]);
        c[i] = __fmul_rn(cosf(angle), magnitude);
        s[i] = __fmul_rn(sinf(angle), magnitude);
    }
}

int rope_table_of(const fyb_rope_desc *d, RopeTable *t)
{
    if (!d || !d->cos_table || !d->sin_table || d->table_rows == 0 || d->table_rows > 0x7fffffffu || d->dims < 2 ||
        d->dims % 2 || d->layout > FYB_ROPE_HALF)
        return -1;
    t->cos = d->cos_table; t->sin = d->sin_table;
    t->rows = d->table_rows; t->dims = d->dims; t->layout = d->layout;
    return 0;
}

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// 16-byte accesses when every address allows them: pointers, strides, heads
// and both halves of the rotated part.
bool rope_vectors(const RopeTable &t, unsigned hd, size_t width, const RopeRows &r)
{
    if (!r.heads) return true;
    const size_t v = 16 / width;
    return aligned16(r.in) && aligned16(r.out) && r.in_stride % v == 0 && r.out_stride % v == 0 && hd % v == 0 &&
           t.dims % v == 0 && (t.layout == 0 || t.dims / 2 % v == 0) && (t.dims / 2) % 4 == 0 && aligned16(t.cos) &&
           aligned16(t.sin);
}

template <typename T>
int rope_launch(const RopeTable &t, const int *positions, size_t rows, unsigned hd, const RopeRows &q,
    const RopeRows &k, unsigned *error, cudaStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    const bool vec = rope_vectors(t, hd, sizeof(T), q) && rope_vectors(t, hd, sizeof(T), k);
    const unsigned step = vec ? V : t.layout == 0 ? 2 : 1;
    const bool in_place = q.in == q.out && (!k.heads || k.in == k.out);
    const RopeWork work = rope_work(hd, t.dims, t.layout, step, in_place);
    const bool many = vec && rope_many(rows, q.heads + k.heads, work);
    const size_t hu = many ? ROPE_HEADS : 1;
    const size_t per_row = ((q.heads + hu - 1) / hu + (k.heads + hu - 1) / hu) * (work.turned + work.copied);
    RopeStage st{(unsigned)(q.heads * hd * sizeof(T)), (unsigned)(k.heads * hd * sizeof(T)), t.dims / 2 * 4, 0};
    st.bytes = (st.q_bytes + st.k_bytes + 2 * st.t_bytes + 127) / 128 * 128;
    // through shared memory once that is 8 MB, 4 rows and more a CTA (below, the copies' latency is what counts), if two
    // CTAs' stages fit an SM
    const size_t smem = (size_t)ROPE_STAGES * st.bytes;
    if (vec && rows * (st.q_bytes + st.k_bytes) >= 8u << 20 && rows >= 4 * 2 * 148 && smem <= 110 * 1024) {
        static std::atomic<unsigned> allowed{0};
        if (allow_shared((const void *)rope_rows_kernel<T, V>, 110 * 1024, allowed)) return -2;
        const unsigned ctas = (unsigned)std::min<size_t>(3, 220 * 1024 / smem) * 148;
        rope_rows_kernel<T, V><<<ctas, ROPE_THREADS, smem, s>>>(t, positions, rows, q, k, hd, work, st, error);
        return cudaGetLastError() == cudaSuccess ? 0 : -2;
    }
    const size_t y = (per_row + ROPE_THREADS - 1) / ROPE_THREADS;
    if (y > 65535) return -1;
    const dim3 grid((unsigned)rows, (unsigned)y);
    if (many) rope_kernel<T, V, true, ROPE_HEADS><<<grid, ROPE_THREADS, 0, s>>>(t, positions, q, k, hd, work, error);
    else if (vec) rope_kernel<T, V, true, 1><<<grid, ROPE_THREADS, 0, s>>>(t, positions, q, k, hd, work, error);
    else if (t.layout == 0) rope_kernel<T, 2, false, 1><<<grid, ROPE_THREADS, 0, s>>>(t, positions, q, k, hd, work, error);
    else rope_kernel<T, 1, false, 1><<<grid, ROPE_THREADS, 0, s>>>(t, positions, q, k, hd, work, error);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

int rope_run(unsigned type, const RopeTable &t, const int *positions, size_t rows, unsigned hd, const RopeRows &q,
    const RopeRows &k, unsigned *error, cudaStream_t s)
{
    if (type == T_F32) return rope_launch<float>(t, positions, rows, hd, q, k, error, s);
    if (type == T_F16) return rope_launch<__half>(t, positions, rows, hd, q, k, error, s);
    return rope_launch<__nv_bfloat16>(t, positions, rows, hd, q, k, error, s);
}

}  // namespace fyb

using namespace fyb;

extern "C" int fyb_rope_frequencies(uint32_t dims, float base, const fyb_rope_scaling *sc, const float *factors,
    float *freq, float *magnitude)
{
    if (!freq || !magnitude || dims < 2 || dims % 2 || !(base > 0.f) || !std::isfinite(base)) return -1;
    const unsigned kind = sc ? sc->kind : FYB_ROPE_PLAIN, pairs = dims / 2;
    if (kind > FYB_ROPE_BANDS) return -1;
    const double factor = sc ? sc->factor : 1.0;
    if (kind != FYB_ROPE_PLAIN && !(factor >= 1.0 && std::isfinite(factor))) return -1;
    if ((kind == FYB_ROPE_YARN || kind == FYB_ROPE_BANDS) && !(sc->original_context > 0.f)) return -1;
    if (kind == FYB_ROPE_NTK && dims == 2) return -1;
    if (factors)
        for (unsigned j = 0; j < pairs; ++j) if (!(factors[j] > 0.f)) return -1;
    *magnitude = kind == FYB_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.f;
    const double turn = 2.0 * 3.14159265358979323846;
    double b = base;
    if (kind == FYB_ROPE_NTK) b *= std::pow(factor, (double)dims / (dims - 2.0));
    // the pair index at which a dimension makes `turns` turns over the original context
    auto pair_of = [&](double turns) { return pairs * std::log(sc->original_context / (turns * turn)) / std::log(b); };
    double lo = 0, hi = 0;
    if (kind == FYB_ROPE_YARN) {
        lo = std::max(0.0, std::floor(pair_of(sc->beta_fast > 0.f ? sc->beta_fast : 32.0)));
        // past the last pair where every dimension makes more turns than beta_slow: the ramp is then cut off by the
        // pairs there are, and not made steeper
        hi = std::min(dims - 1.0, std::ceil(pair_of(sc->beta_slow > 0.f ? sc->beta_slow : 1.0)));
        if (hi - lo < 1e-3) hi = lo + 1e-3;
    }
    for (unsigned j = 0; j < pairs; ++j) {
        // the engine's own F32 formula where nothing but factors changes it
        double f = kind == FYB_ROPE_PLAIN || kind == FYB_ROPE_LINEAR ? (double)powf(base, -(float)j / (float)pairs)
                                                                     : std::pow(b, -(double)j / pairs);
        if (kind == FYB_ROPE_LINEAR) f /= factor;
        if (kind == FYB_ROPE_YARN) {
            const double ramp = std::min(1.0, std::max(0.0, (j - lo) / (hi - lo)));
            f = f / factor * ramp + f * (1.0 - ramp);
        }
        if (kind == FYB_ROPE_BANDS) {
            const double low = sc->low_freq > 0.f ? sc->low_freq : 1.0, high = sc->high_freq > 0.f ? sc->high_freq : 4.0;
            if (!(high > low)) return -1;
            const double turns = sc->original_context * f / turn;
            const double keep = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
            f = f / factor * (1.0 - keep) + f * keep;
        }
        freq[j] = (float)(factors ? f / factors[j] : f);
    }
    return 0;
}

extern "C" int fyb_rope_tables(const float *freq, uint32_t dims, float magnitude, uint32_t first, uint32_t rows,
    float *c, float *s, void *stream)
{
    if (!freq || !c || !s || dims < 2 || dims % 2 || first > 0x7fffffffu || rows > 0x7fffffffu - first) return -1;
    const size_t count = (size_t)rows * (dims / 2);
    if (!count) return 0;
    const unsigned grid = (unsigned)std::min<size_t>((count + 255) / 256, 148 * 8);
    rope_table_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(freq, dims / 2, magnitude, first, count, c, s);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int fyb_rope(const fyb_rope_desc *rope, const int32_t *positions, size_t rows, uint32_t hd, uint32_t type,
    const void *q, size_t q_stride, void *q_out, size_t q_out_stride, uint32_t heads, const void *k, size_t k_stride,
    void *k_out, size_t k_out_stride, uint32_t kv_heads, uint32_t *error, void *stream)
{
    RopeTable t;
    if (rope_table_of(rope, &t) || hd < t.dims || hd % 2 || hd > 65536 || heads > 65536 || kv_heads > 65536 ||
        rows > 0x7fffffffu || heads + kv_heads == 0 || (rows && heads && (!q || !q_out)) || (rows && kv_heads && (!k || !k_out)) ||
        q_stride < (size_t)heads * hd || q_out_stride < (size_t)heads * hd || k_stride < (size_t)kv_heads * hd ||
        k_out_stride < (size_t)kv_heads * hd || (heads && q == q_out && q_stride != q_out_stride) ||
        (kv_heads && k == k_out && k_stride != k_out_stride))
        return -1;
    if (type != T_F32 && type != T_F16 && type != T_BF16) return -1;
    if (!rows) return 0;
    const size_t width = type == T_F32 ? 4 : 2;
    if (!positions || (heads && off_element(width, q, q_out)) || (kv_heads && off_element(width, k, k_out))) return -1;
    const RopeRows rq{q, q_out, q_stride, q_out_stride, heads}, rk{k, k_out, k_stride, k_out_stride, kv_heads};
    return rope_run(type, t, positions, rows, hd, rq, rk, error, (cudaStream_t)stream);
}
