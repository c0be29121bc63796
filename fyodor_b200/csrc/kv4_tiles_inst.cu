// kv4_tiles_inst.cu - one head dimension and row tile of the many-row attention
// kernel over the 4-bit cache (kv4_tiles.cuh); the build compiles this file once
// for each pair.
#include "kv4_tiles.cuh"

#ifndef FYB_K4_HD
#define FYB_K4_HD 128
#define FYB_K4_NR 256
#endif
#define FYB_K4_NAME2(hd, nr) kv4_tiles_##hd##_##nr
#define FYB_K4_NAME(hd, nr) FYB_K4_NAME2(hd, nr)

namespace fyb {

int FYB_K4_NAME(FYB_K4_HD, FYB_K4_NR)(const Kv4Attention &A, const CUtensorMap &k, const CUtensorMap &v, unsigned grid,
    cudaStream_t s)
{
    return kv4_tiles_go<FYB_K4_HD, FYB_K4_NR>(A, k, v, grid, s);
}

}  // namespace fyb
