// kv8_tiles_inst.cu - one head dimension and format of the many-row attention
// kernel (kv8_tiles.cuh); the build compiles this file once for each pair.
#include "kv8_tiles.cuh"

#ifndef FYB_KT_HD
#define FYB_KT_HD 128
#define FYB_KT_FMT 0
#endif
#define FYB_KT_NAME2(hd, fmt) kv8_tiles_##hd##_##fmt
#define FYB_KT_NAME(hd, fmt) FYB_KT_NAME2(hd, fmt)

namespace fyb {

int FYB_KT_NAME(FYB_KT_HD, FYB_KT_FMT)(const Kv8Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned rows,
    unsigned grid, cudaStream_t s)
{
    const bool f32 = A.type == T_F32;
    if (rows == 32)
        return f32 ? kv8_tiles_go<FYB_KT_HD, FYB_KT_FMT, 32, 2>(A, k, v, grid, s)
                   : kv8_tiles_go<FYB_KT_HD, FYB_KT_FMT, 32, 1>(A, k, v, grid, s);
    return f32 ? kv8_tiles_go<FYB_KT_HD, FYB_KT_FMT, 64, 2>(A, k, v, grid, s)
               : kv8_tiles_go<FYB_KT_HD, FYB_KT_FMT, 64, 1>(A, k, v, grid, s);
}

}  // namespace fyb
