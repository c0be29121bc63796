// rope.cuh - rotary positions of one run of a head's values, shared by the
// stand-alone kernel (rope.cu) and the cache append (kv8.cu).
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

// V values of a row, as one access when VEC (aligned to V * sizeof(T)).
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
template <typename T, int V, bool VEC> FYB_DEV void row_store(T *p, const float (&x)[V])
{
    if constexpr (VEC) {
        struct alignas(V * sizeof(T)) Pack { T t[V]; };
        Pack u;
#pragma unroll
        for (int i = 0; i < V; ++i) u.t[i] = row_round<T>(x[i]);
        *reinterpret_cast<Pack *>(p) = u;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = row_round<T>(x[i]);
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

// Work items of one head: interleaved pairs, one per V values; half pairs,
// one per V pairs (both halves) and one per V values that are only copied.
// V divides the rotated part (both halves of it) and the head, or is 2
// (interleaved) or 1 (half).
FYB_HOST_DEV unsigned rope_items(unsigned hd, unsigned dims, unsigned layout, unsigned V)
{
    return layout == 0 ? hd / V : dims / 2 / V + (hd - dims) / V;
}

template <typename T, int V, bool VEC>
FYB_DEV void rope_item(const T *in, T *out, const float *c, const float *s, unsigned dims, unsigned layout, unsigned item)
{
    if (layout == 0) {
        const unsigned e = item * V;
        float x[V];
        row_load<T, V, VEC>(in + e, x);
        if (e < dims) {
            if constexpr (V > 1) {
                float cv[V / 2], sv[V / 2];
                row_load<float, V / 2, VEC>(c + e / 2, cv);
                row_load<float, V / 2, VEC>(s + e / 2, sv);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) rope_turn(x[2 * i], x[2 * i + 1], cv[i], sv[i]);
            }
        } else if (in == out) {
            return;
        }
        row_store<T, V, VEC>(out + e, x);
        return;
    }
    const unsigned pairs = dims / 2;
    if (item * V < pairs) {
        const unsigned e = item * V;
        float a[V], b[V], cv[V], sv[V];
        row_load<T, V, VEC>(in + e, a);
        row_load<T, V, VEC>(in + e + pairs, b);
        row_load<float, V, VEC && V <= 4>(c + e, cv);
        row_load<float, V, VEC && V <= 4>(s + e, sv);
#pragma unroll
        for (int i = 0; i < V; ++i) rope_turn(a[i], b[i], cv[i], sv[i]);
        row_store<T, V, VEC>(out + e, a);
        row_store<T, V, VEC>(out + e + pairs, b);
    } else if (in != out) {
        const unsigned e = dims + (item * V - pairs);
        float x[V];
        row_load<T, V, VEC>(in + e, x);
        row_store<T, V, VEC>(out + e, x);
    }
}

}  // namespace fyb
