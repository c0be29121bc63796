// kv8_attention.cu - the entry point of attention over the paged 8-bit cache:
// argument checks, the workspace, and which kernel runs.
//
// Up to eight query rows per KV head (rows of a request x heads of a group) run
// on kv8_decode.cu, more on kv8_tiles.cuh in row tiles of 32 rows, or of 64
// where a request can bring more. Both sides, head_dim 128, int8 (us):
//
//   eight rows    16 requests of 8100   decode  62   tiles of 32   97
//                  1 request of 300             10                 16
//   32 rows       32 requests of 8100   of 32  184   of 64        235
//   64 rows       32 requests of 8100          266                247
//   512 rows       1 request of 16000          166                131
//
// (Below a wave of segments tiles of 32 also win at 64 rows, 19 against 31 us
// for one request of 512, but the lengths that decide it are on the device.)
#include "kv8_attention.cuh"

namespace fyb {

using TilesLaunch = int(const Kv8Attention &, const CUtensorMap &, const CUtensorMap &, unsigned, unsigned, cudaStream_t);
TilesLaunch kv8_tiles_128_0, kv8_tiles_128_1, kv8_tiles_64_0, kv8_tiles_64_1;

constexpr unsigned KT_GRID = 148, KT_ROWS = 64;  // one CTA per SM; most query rows of a row tile

int kv8_tensor_map(CUtensorMap *map, const void *pool, unsigned row_bytes, size_t rows, unsigned box_rows, CUtensorMapSwizzle swizzle)
{
    using Encode = decltype(&cuTensorMapEncodeTiled);
    static const Encode encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            f = nullptr;
        }
        return (Encode)f;
    }();
    if (!encode) return -2;
    const cuuint64_t dims[2] = {row_bytes, rows}, strides[1] = {row_bytes};
    const cuuint32_t box[2] = {row_bytes, box_rows}, step[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(pool), dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -2;
}
int kv8_tensor_map(CUtensorMap *map, const fyb_kv8_cache &c, const void *pool)
{
    return kv8_tensor_map(map, pool, c.head_dim, (size_t)c.blocks * c.kv_heads * c.block_size, std::min(c.block_size, 64u),
                          c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

// Partials of a call: two per CTA of its kernel, `rows` query rows each.
static size_t part_slots(bool few) { return few ? 2 * KA_GRID * KV8_DECODE_ROWS : 2 * KT_GRID * KT_ROWS; }

}  // namespace fyb

using namespace fyb;

extern "C" size_t fyb_kv8_attention_workspace(uint32_t requests, uint32_t max_rows, uint32_t heads, uint32_t kv_heads,
    uint32_t head_dim)
{
    if (!requests || !max_rows || !kv_heads || heads < kv_heads || heads % kv_heads || heads / kv_heads > KT_ROWS ||
        (head_dim != 64 && head_dim != 128))
        return 0;
    const bool few = (unsigned long long)max_rows * (heads / kv_heads) <= KV8_DECODE_ROWS;
    return KA_COUNTER_BYTES + part_slots(few) * (head_dim + 2) * sizeof(float);
}

extern "C" int fyb_kv8_attention(const fyb_kv8_cache *cache, const int32_t *lengths, const int32_t *row_start,
    uint32_t requests, uint32_t max_rows, size_t rows, const int32_t *table, size_t table_stride, uint32_t type,
    const void *q, size_t q_stride, void *out, size_t out_stride, uint32_t heads, float scale, void *workspace,
    size_t workspace_bytes, uint32_t *error, void *stream)
{
    if (kv8_check(cache) || (type != T_F32 && type != T_F16 && type != T_BF16) || table_stride == 0 ||
        table_stride > 0x7fffffffu || rows > 0x7fffffffu || max_rows > 0x7fffffffu)
        return -1;
    const size_t need = fyb_kv8_attention_workspace(requests, max_rows, heads, cache->kv_heads, cache->head_dim);
    const size_t row = (size_t)heads * cache->head_dim;
    if (!need || !lengths || !table || (rows && (!q || !out)) || q_stride < row || out_stride < row || !workspace ||
        (uintptr_t)workspace % 16 || workspace_bytes < need || (!row_start && rows != requests))
        return -1;
    if (!rows) return 0;
    if (off_element(type == T_F32 ? 4 : 2, q, out)) return -1;
    Kv8Attention A{};
    A.c = *cache;
    A.lengths = lengths; A.row_start = row_start; A.table = table; A.table_stride = table_stride;
    A.rows = (unsigned)rows; A.q = q; A.q_stride = q_stride; A.out = out; A.out_stride = out_stride;
    A.requests = requests; A.max_rows = max_rows; A.heads = heads; A.group = heads / cache->kv_heads;
    A.shift = kv8_shift(cache); A.type = type; A.scale = scale * 1.44269504f; A.error = error;
    const unsigned long long group_rows = (unsigned long long)max_rows * A.group;
    const bool few = group_rows <= KV8_DECODE_ROWS;
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    A.counters = reinterpret_cast<unsigned *>(ws);
    A.part_ml = reinterpret_cast<float2 *>(ws + KA_COUNTER_BYTES);
    A.part_o = reinterpret_cast<float *>(A.part_ml + part_slots(few));
    CUtensorMap k, v;
    if (kv8_tensor_map(&k, A.c, A.c.k) || kv8_tensor_map(&v, A.c, A.c.v)) return -2;
    // no more CTAs than the most units the tables can hold
    const unsigned long long holds = (unsigned long long)table_stride << A.shift;
    cudaStream_t s = (cudaStream_t)stream;
    if (few) {
        A.row_tile = max_rows;
        const unsigned long long units = (holds + 63) / 64 * requests * cache->kv_heads;
        return launch_kv8_decode(A, k, v, (unsigned)std::min<unsigned long long>(KA_GRID, units), s);
    }
    const unsigned n = group_rows <= 32 ? 32 : KT_ROWS;
    A.row_tile = n / A.group;
    const unsigned long long tiles = std::min<unsigned long long>((max_rows + A.row_tile - 1) / A.row_tile, 1u << 20);
    const unsigned long long units = std::min<unsigned long long>((holds + 127) / 128 * requests, 1u << 20) * tiles * cache->kv_heads;
    const unsigned grid = (unsigned)std::min<unsigned long long>(KT_GRID, units);
    TilesLaunch *go = cache->head_dim == 128 ? (cache->format == FYB_KV8_INT8 ? kv8_tiles_128_0 : kv8_tiles_128_1)
                                             : (cache->format == FYB_KV8_INT8 ? kv8_tiles_64_0 : kv8_tiles_64_1);
    return go(A, k, v, n, grid, s);
}
