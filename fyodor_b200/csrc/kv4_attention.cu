// kv4_attention.cu - the entry point of attention over the paged 4-bit cache:
// argument checks, the workspace, and which kernel runs.
//
// Up to eight query rows per KV head (rows of a request x heads of a group), and
// rows of F32 whatever their number, run on kv4_decode.cu, many rows in row tiles of
// eight; many rows of 16 bits on kv4_tiles.cuh, in row tiles of 32, 64 or 256. Both
// kernels, us, with that many bf16 rows per KV head (four heads a group, 8 KV heads):
//
//                                    8 rows     16 rows    32 rows
//   16 requests at 8100              57 /  73   97 /  73   175 /  74
//   32 of 128 to 8192 (145 MB)       57 /  75   99 /  77   179 /  78
//   32 of 128 to 32768 (649 MB)     185 / 248  353 / 255
//   4 of 500                                  13.7 / 15.4  15.6 / 16.3
//
// F32 rows pay for each eight of them (16 requests at 8100: 8 rows 76 us, 16 131, 32
// 241; a chunk of 2000 rows of one of 16000 1703, in bf16 161): the tiles round K, V and
// the weights to 16 bits, which is not enough for them.
#include "kv4_attention.cuh"

namespace fyb {

using TilesLaunch = int(const Kv4Attention &, const CUtensorMap &, const CUtensorMap &, unsigned, cudaStream_t);
TilesLaunch kv4_tiles_128_32, kv4_tiles_128_64, kv4_tiles_128_256, kv4_tiles_64_32, kv4_tiles_64_64, kv4_tiles_64_256;

// K or V as rows of 128 bytes (two tokens of 64, or four of 32 bytes), boxes of one block (128 tokens at most), in the
// swizzle of 128 bytes (kv4_at). With a row for each token drafts of 8 took 345 us instead of 337, single tokens the same.
static int kv4_tensor_map(CUtensorMap *map, const fyb_kv4_cache &c, const void *pool)
{
    const unsigned tokens = 256 / c.head_dim;
    return kv8_tensor_map(map, pool, 128, (size_t)c.blocks * c.kv_heads * c.block_size / tokens,
                          std::min(c.block_size, (unsigned)K4_TILE) / tokens, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Row tile of the many-row kernel. 128 rows of a request are two tiles of 64 (one of 16000 tokens: 40 us, in tiles of 256
// 52; four of them 77 and 90); 256 rows of one of 16000 would still be quicker so (51 and 59), of one of 64000 not (127
// and 111), 500 rows at 16000 not either (76 and 70), 2000 rows far from it (234 and 165).
static unsigned tile_rows(unsigned long long group_rows) { return group_rows <= 32 ? 32 : group_rows <= 128 ? 64 : 256; }
// Query rows of a call's partials, two for each CTA of its kernel (F32 rows need 2 K4_GRID of eight: fewer than tiles do).
static size_t part_rows(unsigned long long group_rows)
{
    static_assert(2 * K4_GRID * KV8_DECODE_ROWS <= 2 * K4T_GRID * 32, "");
    return group_rows <= KV8_DECODE_ROWS ? 2 * K4_GRID * KV8_DECODE_ROWS : 2 * K4T_GRID * tile_rows(group_rows);
}

}  // namespace fyb

using namespace fyb;

extern "C" size_t fyb_kv4_attention_workspace(uint32_t requests, uint32_t max_rows, uint32_t heads, uint32_t kv_heads,
    uint32_t head_dim)
{
    if (!requests || !max_rows || !kv_heads || heads < kv_heads || heads % kv_heads || heads / kv_heads > 64 ||
        (head_dim != 64 && head_dim != 128))
        return 0;
    return K4_COUNTER_BYTES + K4_JOIN_BYTES + part_rows((unsigned long long)max_rows * (heads / kv_heads)) * (head_dim + 2) * sizeof(float);
}

extern "C" int fyb_kv4_attention(const fyb_kv4_cache *cache, const int32_t *lengths, const int32_t *row_start,
    uint32_t requests, uint32_t max_rows, size_t rows, const int32_t *table, size_t table_stride, uint32_t type,
    const void *q, size_t q_stride, void *out, size_t out_stride, uint32_t heads, float scale, void *workspace,
    size_t workspace_bytes, uint32_t *error, void *stream)
{
    if (kv4_check(cache) || (type != T_F32 && type != T_F16 && type != T_BF16) || table_stride == 0 ||
        table_stride > 0x7fffffffu || rows > 0x7fffffffu || max_rows > 0x7fffffffu)
        return -1;
    const size_t need = fyb_kv4_attention_workspace(requests, max_rows, heads, cache->kv_heads, cache->head_dim);
    const size_t row = (size_t)heads * cache->head_dim;
    if (!need || !lengths || !table || (rows && (!q || !out)) || q_stride < row || out_stride < row || !workspace ||
        (uintptr_t)workspace % 16 || workspace_bytes < need || (!row_start && rows != requests))
        return -1;
    if (!rows) return 0;
    if (off_element(type == T_F32 ? 4 : 2, q, out)) return -1;
    Kv4Attention A{};
    A.c.blocks = cache->blocks; A.c.kv_heads = cache->kv_heads; A.c.block_size = cache->block_size;
    A.c.head_dim = cache->head_dim;
    A.ks = static_cast<const __half2 *>(cache->k_scale); A.vs = static_cast<const __half2 *>(cache->v_scale);
    A.lengths = lengths; A.row_start = row_start; A.table = table; A.table_stride = table_stride;
    A.rows = (unsigned)rows; A.q = q; A.q_stride = q_stride; A.out = out; A.out_stride = out_stride;
    A.requests = requests; A.max_rows = max_rows; A.heads = heads; A.group = heads / cache->kv_heads; A.split = 1;
    A.shift = kv4_shift(cache); A.type = type; A.scale = scale * 1.44269504f; A.error = error;
    const unsigned long long group_rows = (unsigned long long)max_rows * A.group;
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    A.counters = reinterpret_cast<unsigned *>(ws);
    A.join = reinterpret_cast<K4tJoin *>(ws + K4_COUNTER_BYTES);
    A.part_ml = reinterpret_cast<float2 *>(ws + K4_COUNTER_BYTES + K4_JOIN_BYTES);
    A.part_o = reinterpret_cast<float *>(A.part_ml + part_rows(group_rows));
    CUtensorMap k, v;
    if (kv4_tensor_map(&k, *cache, cache->k) || kv4_tensor_map(&v, *cache, cache->v)) return -2;
    // no more CTAs than the most units the tables can hold
    const unsigned long long holds = (unsigned long long)table_stride << A.shift;
    const unsigned long long tiles = std::min<unsigned long long>((holds + K4_TILE - 1) / K4_TILE * requests, 1u << 20);
    cudaStream_t s = (cudaStream_t)stream;
    if (group_rows <= KV8_DECODE_ROWS || type == T_F32) {
        // more heads than a row tile holds: parts of a group, each as a KV head of its own over the same cache
        while (A.group > KV8_DECODE_ROWS || cache->kv_heads * A.split * A.group != heads) {
            ++A.split;
            A.group = heads / cache->kv_heads / A.split;
        }
        A.c.kv_heads = cache->kv_heads * A.split;
        A.row_tile = std::min(max_rows, KV8_DECODE_ROWS / A.group);
        const unsigned long long units = tiles * A.c.kv_heads * std::min<unsigned long long>((max_rows + A.row_tile - 1) / A.row_tile, 1u << 20);
        return launch_kv4_decode(A, k, v, (unsigned)std::min<unsigned long long>(K4_GRID, units), s);
    }
    const unsigned n = tile_rows(group_rows);
    A.vec = (uintptr_t)q % 16 == 0 && q_stride % 8 == 0;
    A.vec_out = (uintptr_t)out % 16 == 0 && out_stride % 8 == 0;
    A.row_tile = n / A.group;
    const unsigned long long units = tiles * A.c.kv_heads * std::min<unsigned long long>((max_rows + A.row_tile - 1) / A.row_tile, 1u << 20);
    const unsigned grid = (unsigned)std::min<unsigned long long>(K4T_GRID, units);
    TilesLaunch *go = cache->head_dim == 128 ? (n == 32 ? kv4_tiles_128_32 : n == 64 ? kv4_tiles_128_64 : kv4_tiles_128_256)
                                             : (n == 32 ? kv4_tiles_64_32 : n == 64 ? kv4_tiles_64_64 : kv4_tiles_64_256);
    return go(A, k, v, grid, s);
}
