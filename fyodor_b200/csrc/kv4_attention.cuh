// kv4_attention.cuh - what the kernels of attention over the paged 4-bit cache
// share: their arguments and the loads of the cache. The work is split over the
// GPU as the 8-bit cache's is (kv8_attention.cuh).
#pragma once
#include "kv8_attention.cuh"
#include "kv4.cuh"

namespace fyb {

struct Kv4Attention : Kv8Attention {
    const __half2 *ks, *vs;  // scale and low of each group
    unsigned split;          // parts of a KV head's group of query heads, each counted as a head (c.kv_heads, group)
    bool vec, vec_out;       // rows of 16 bits of q, of out begin on 16 bytes
};

int launch_kv4_decode(const Kv4Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned grid, cudaStream_t s);
constexpr int K4_TILE = 128;  // positions of a unit
constexpr unsigned K4_CTAS = 3, K4_GRID = K4_CTAS * 148;  // of the few-row kernel: CTAs per SM, largest grid
constexpr size_t K4_COUNTER_BYTES = (K4_GRID * 4 + 255) / 256 * 256;

}  // namespace fyb
