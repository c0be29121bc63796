// kv4_attention.cuh - what the kernels of attention over the paged 4-bit cache
// share: their arguments and the loads of the cache. The work is split over the
// GPU as the 8-bit cache's is (kv8_attention.cuh).
#pragma once
#include "kv8_attention.cuh"
#include "kv4.cuh"

namespace fyb {

// The segment that begins in a CTA of the many-row kernel and goes on in others: its last CTA, its query rows (0: there is
// none), the first of its call's rows, its head.
struct K4tJoin {
    unsigned last, rows, first_row, head;
};
struct Kv4Attention : Kv8Attention {
    K4tJoin *join;
    const __half2 *ks, *vs;  // scale and low of each group
    unsigned split;          // parts of a KV head's group of query heads, each counted as a head (c.kv_heads, group)
    bool vec, vec_out;       // rows of 16 bits of q, of out begin on 16 bytes
};

// Byte `byte` of token `pos` of a tile of K or V in shared memory: rows of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7).
template <int HD> FYB_HOST_DEV unsigned kv4_at(unsigned pos, unsigned byte)
{
    constexpr unsigned ROW = HD / 2, TOKENS = 128 / ROW;
    const unsigned row = pos / TOKENS;
    return row * 128 + ((pos % TOKENS * ROW + byte) ^ ((row & 7) << 4));
}
FYB_DEV void k4_copy(unsigned dst, const void *src, unsigned bytes, unsigned bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
FYB_DEV void k4_load_rows(unsigned dst, const CUtensorMap *map, int row, unsigned bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(dst), "l"(map), "r"(0), "r"(row), "r"(bar) : "memory");
}

int launch_kv4_decode(const Kv4Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned grid, cudaStream_t s);
constexpr int K4_TILE = 128;  // positions of a unit
constexpr unsigned K4_CTAS = 3, K4_GRID = K4_CTAS * 148;  // of the few-row kernel: CTAs per SM, largest grid
constexpr unsigned K4T_GRID = 148;                        // of the many-row kernel: one CTA per SM
constexpr size_t K4_COUNTER_BYTES = (K4_GRID * 4 + 255) / 256 * 256, K4_JOIN_BYTES = (K4T_GRID * sizeof(K4tJoin) + 255) / 256 * 256;

}  // namespace fyb
