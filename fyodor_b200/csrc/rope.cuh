// rope.cuh - rotary positions of one run of a head's values, shared by the
// stand-alone kernel (rope.cu) and the cache appends (kv8.cu, kv4.cu).
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace fyb {

// (a, b) turned by the angle whose cosine and sine are c and s, each product
// and sum rounded on its own (llm_cpu.c:298-327).
FYB_DEV void rope_turn(float &a, float &b, float c, float s)
{
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
    a = x;
}

// V values of a row, as one access when VEC (aligned to V * sizeof(T), 16 bytes at most).
template <typename T, int V, bool VEC> FYB_DEV void row_load(const T *p, float (&x)[V])
{
    if constexpr (VEC) {
        struct alignas(V * sizeof(T)) Pack { T t[V]; };
        const Pack u = *reinterpret_cast<const Pack *>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = row_value(u.t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = row_value(p[i]);
    }
}
// One operand of a rotation: rows of `heads` heads, strides in elements.
struct RopeRows {
    const void *in = nullptr;
    void *out = nullptr;
    size_t in_stride = 0, out_stride = 0;
    unsigned heads = 0;
};
struct RopeTable {
    const float *cos = nullptr, *sin = nullptr;
    unsigned rows = 0, dims = 0, layout = 0;
};

// V floats of a table row, 16-byte accesses where V and VEC allow.
template <int V, bool VEC> FYB_DEV void rope_row(const float *p, float (&x)[V])
{
    if constexpr (VEC && V % 4 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(p + i);
            x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
        }
    } else {
        row_load<float, V, VEC>(p, x);
    }
}

// Work items of one head: interleaved pairs, one per V values; half pairs,
// one per V pairs (both halves) and one per V values that are only copied.
// V divides the rotated part (both halves of it) and the head, or is 2
// (interleaved) or 1 (half).
//
// A row's work, rotated items of all head groups before copied ones: the lanes of a warp then do the same, and
// neighbouring lanes work on neighbouring memory.
struct RopeWork {
    unsigned turned = 0, copied = 0;  // items of a head
};
FYB_HOST_DEV RopeWork rope_work(unsigned hd, unsigned dims, unsigned layout, unsigned V, bool in_place)
{
    RopeWork w;
    w.turned = (layout == 0 ? dims : dims / 2) / V;
    w.copied = in_place ? 0 : (hd - dims) / V;
    return w;
}
// Index i of a row with `groups` head groups: its group and item; false past the row's end.
FYB_DEV bool rope_place(const RopeWork &w, unsigned groups, unsigned i, unsigned &group, unsigned &item)
{
    const unsigned first = groups * w.turned;
    if (i < first) {
        group = i / w.turned;
        item = i % w.turned;
        return true;
    }
    i -= first;
    if (i >= groups * w.copied) return false;
    group = i / w.copied;
    item = w.turned + i % w.copied;
    return true;
}

// V values of a row as loaded: one access when VEC.
template <typename T, int V> struct alignas(V * sizeof(T)) RopePack { T t[V]; };
template <typename T, int V, bool VEC> FYB_DEV RopePack<T, V> rope_get(const T *p)
{
    if constexpr (VEC) {
        return *reinterpret_cast<const RopePack<T, V> *>(p);
    } else {
        RopePack<T, V> u;
#pragma unroll
        for (int i = 0; i < V; ++i) u.t[i] = p[i];
        return u;
    }
}
template <typename T, int V, bool VEC> FYB_DEV void rope_put(T *p, const RopePack<T, V> &u)
{
    if constexpr (VEC) {
        *reinterpret_cast<RopePack<T, V> *>(p) = u;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = u.t[i];
    }
}

// Item `item` of `count` (<= HU) heads, `apart` elements from one to the next: they share the row's cosines and
// sines. at(&c, &s) gives the row's table, or false for a row that stays as it is; it is asked after the values have
// been asked for, so the position's latency and theirs pass together.
template <typename T, int V, bool VEC, int HU, typename At>
FYB_DEV void rope_item(const T *in, T *out, size_t apart, unsigned count, unsigned dims, unsigned layout, unsigned item, At at)
{
    const unsigned pairs = dims / 2;
    const bool two = layout != 0 && item * V < pairs;      // both halves of V pairs
    const unsigned e = layout == 0 || two ? item * V : dims + (item * V - pairs);
    const bool turn = layout == 0 ? e < dims : two;
    RopePack<T, V> a[HU], b[HU];
#pragma unroll
    for (int h = 0; h < HU; ++h)
        if (h < count) {
            a[h] = rope_get<T, V, VEC>(in + h * apart + e);
            if (two) b[h] = rope_get<T, V, VEC>(in + h * apart + e + pairs);
        }
    const float *c, *s;
    if (!at(c, s)) return;
    if (two) {
        float cv[V], sv[V];
        rope_row<V, VEC>(c + e, cv);
        rope_row<V, VEC>(s + e, sv);
#pragma unroll
        for (int h = 0; h < HU; ++h)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float x = row_value(a[h].t[i]), y = row_value(b[h].t[i]);
                rope_turn(x, y, cv[i], sv[i]);
                a[h].t[i] = row_round<T>(x);
                b[h].t[i] = row_round<T>(y);
            }
    } else if (turn) {
        if constexpr (V > 1) {
            float cv[V / 2], sv[V / 2];
            rope_row<V / 2, VEC>(c + e / 2, cv);
            rope_row<V / 2, VEC>(s + e / 2, sv);
#pragma unroll
            for (int h = 0; h < HU; ++h)
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    float x = row_value(a[h].t[2 * i]), y = row_value(a[h].t[2 * i + 1]);
                    rope_turn(x, y, cv[i], sv[i]);
                    a[h].t[2 * i] = row_round<T>(x);
                    a[h].t[2 * i + 1] = row_round<T>(y);
                }
        }
    }
#pragma unroll
    for (int h = 0; h < HU; ++h)
        if (h < count) {
            rope_put<T, V, VEC>(out + h * apart + e, a[h]);
            if (two) rope_put<T, V, VEC>(out + h * apart + e + pairs, b[h]);
        }
}

// Heads that a thread takes: two (they share the cosines and sines) once that leaves two full waves of threads, one
// below, where the length of a thread is the time of the call.
constexpr int ROPE_HEADS = 2;
inline bool rope_many(size_t rows, unsigned heads, const RopeWork &w)
{
    return rows * (heads / ROPE_HEADS) * (w.turned + w.copied) >= (size_t)2 * 148 * 2048;
}

// A row of q beside a cache append (kv8.cu, kv4.cu), whose arguments A are: CTA `cta` takes THREADS items of it.
template <typename T, int HD, unsigned THREADS, typename Append> FYB_DEV void rope_row_of_q(const Append &A, unsigned cta)
{
    const size_t r = cta / A.q_rows;
    const unsigned i = cta % A.q_rows * THREADS + threadIdx.x;
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

}  // namespace fyb
