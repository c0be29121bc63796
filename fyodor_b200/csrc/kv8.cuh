// kv8.cuh - the paged 8-bit KV cache: formats, geometry and argument checks
// shared by the append / read kernels (kv8.cu) and the attention kernels
// (kv8_attention.cu).
#pragma once
#include "common.cuh"
#include "kernels.h"
#include "fyodor_b200.h"
#include <cuda_fp8.h>

namespace fyb {

// Largest stored magnitude of a format.
FYB_HOST_DEV float kv8_top(unsigned format) { return format == FYB_KV8_INT8 ? 127.f : 448.f; }
// The scale that holds magnitudes up to peak: peak times the F32 reciprocal.
FYB_DEV float kv8_scale(unsigned format, float peak)
{
    return __fmul_rn(peak, format == FYB_KV8_INT8 ? 1.f / 127.f : 1.f / 448.f);
}

// x / scale (already divided) to its stored byte: nearest, ties to even; the
// magnitude is at most the format's largest value but for the rounding of the
// scale, which the clamp (int8) and the saturating conversion (e4m3) take back.
template <unsigned FMT> FYB_DEV unsigned kv8_store(float y)
{
    if constexpr (FMT == FYB_KV8_INT8) return (unsigned)max(-127, min(127, __float2int_rn(y))) & 0xffu;
    else return (unsigned)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}
// The number a stored byte stands for, before its scale (exact).
template <unsigned FMT> FYB_DEV float kv8_number(unsigned byte)
{
    if constexpr (FMT == FYB_KV8_INT8) return (float)(signed char)byte;
    else return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

// Geometry checks of a cache handle: 0, or -1. Token rows are indexed in 31
// bits, byte offsets in size_t.
inline int kv8_check(const fyb_kv8_cache *c)
{
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || ((uintptr_t)c->k | (uintptr_t)c->v) % 16 ||
        c->blocks == 0 || c->kv_heads == 0 || (c->head_dim != 64 && c->head_dim != 128) || c->format > FYB_KV8_E4M3 ||
        c->block_size < 16 || c->block_size > 256 || (c->block_size & (c->block_size - 1)))
        return -1;
    return (unsigned long long)c->blocks * c->kv_heads * c->block_size > 0x7fffffffull ? -1 : 0;
}
inline unsigned kv8_shift(const fyb_kv8_cache *c)
{
    unsigned s = 4;
    while (1u << s < c->block_size) ++s;
    return s;
}

}  // namespace fyb
