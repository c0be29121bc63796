// kv4.cuh - the paged 4-bit KV cache: its format, geometry and argument checks,
// shared by the append / read kernels (kv4.cu) and the attention kernels.
//
// A group of 64 values of one head of one token is held as low + scale n, n =
// 0..15, scale and low F16. A token's row of a head is packed eight values to a
// 32-bit word, the first in the lowest bits; with two groups (head_dim 128)
// their words take turns: word 2j holds dimensions 8j.., word 2j + 1 64 + 8j...
// So 16 bytes hold 16 consecutive dimensions of each group, 8 bytes eight of
// each: what a thread of the attention takes of a token lies together.
#pragma once
#include "common.cuh"
#include "kernels.h"
#include "fyodor_b200.h"

namespace fyb {

constexpr int KV4_GROUP = 64;
constexpr float KV4_MOST = 61440.f;  // largest magnitude held: low + 15 scale stays a finite half however scale rounds

// Geometry checks of a cache handle: 0, or -1. Token rows are indexed in 31
// bits, byte offsets in size_t.
inline int kv4_check(const fyb_kv4_cache *c)
{
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale ||
        ((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scale | (uintptr_t)c->v_scale) % 16 || c->blocks == 0 ||
        c->kv_heads == 0 || c->kv_heads > 65536 || (c->head_dim != 64 && c->head_dim != 128) || c->block_size < 16 || c->block_size > 256 ||
        (c->block_size & (c->block_size - 1)))
        return -1;
    return (unsigned long long)c->blocks * c->kv_heads * c->block_size > 0x7fffffffull ? -1 : 0;
}
inline unsigned kv4_shift(const fyb_kv4_cache *c)
{
    unsigned s = 4;
    while (1u << s < c->block_size) ++s;
    return s;
}

// First dimension of word w of a token's row.
template <int HD> FYB_HOST_DEV unsigned kv4_first(unsigned w)
{
    return HD == 64 ? 8 * w : (w & 1) * KV4_GROUP + (w >> 1) * 8;
}
FYB_DEV float kv4_value(unsigned word, int i, float2 scale_low)
{
    return __fmaf_rn((float)(word >> (4 * i) & 15u), scale_low.x, scale_low.y);
}

}  // namespace fyb
