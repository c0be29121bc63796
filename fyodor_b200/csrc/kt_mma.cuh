// kt_mma.cuh - tcgen05 matrix products, tensor memory and bounded waits of the
// many-row attention kernels (kv8_tiles.cuh, kv4_tiles.cuh).
#pragma once
#include "common.cuh"

namespace fyb {

// ---- tcgen05 -------------------------------------------------------------------
// Operand in 128-byte swizzled rows, eight-row groups 1024 bytes apart. K-major:
// a row is 64 K values of one M/N index. M/N-major: a row is 64 M/N values of one
// K index, `lead` bytes to the next 64.
FYB_DEV uint64_t kt_desc(unsigned addr, unsigned lead)
{
    return (uint64_t)(addr >> 4 & 0x3FFFu) | (uint64_t)(lead >> 4) << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61;
}
// F32 accumulator, fp16 operands, M = 128; mn: B is N-major
FYB_HOST_DEV constexpr uint32_t kt_idesc(unsigned N, bool mn)
{
    return 1u << 4 | (mn ? 1u << 16 : 0u) | N >> 3 << 17 | 128u >> 4 << 24;
}
// D (tensor memory) (+)= A (tensor memory: row m in lane m, 16 K values in 8 columns) x B (shared memory)
FYB_DEV void kt_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
// the same with A in shared memory
FYB_DEV void kt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
FYB_DEV void kt_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 :: "r"(smem_u32(bar)) : "memory");
}
FYB_DEV bool kt_elect()
{
    unsigned one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}
FYB_DEV void kt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
FYB_DEV void kt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 16 consecutive columns of this thread's TMEM lane
FYB_DEV void kt_ld16(uint32_t addr, float *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
                   "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
                 : "r"(addr) : "memory");
}
FYB_DEV void kt_ld32(uint32_t addr, float *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
                   "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
                   "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
                   "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
                 : "r"(addr) : "memory");
}
FYB_DEV void kt_ld4(uint32_t addr, float *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]) : "r"(addr) : "memory");
}
FYB_DEV void kt_st4(uint32_t addr, const float *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};"
                 :: "r"(addr), "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]) : "memory");
}
FYB_DEV void kt_st16(uint32_t addr, const float *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 :: "r"(addr), "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]),
                    "f"(r[8]), "f"(r[9]), "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15])
                 : "memory");
}
// 16 lanes x 32 columns: registers 4j, 4j + 1 of lane 4g + t go to TMEM lane g, columns 8j + 2t and + 1; 4j + 2, 4j + 3
// to TMEM lane g + 8
FYB_DEV void kt_st256(uint32_t addr, const unsigned *r)
{
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                    "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
FYB_DEV void kt_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
FYB_DEV void kt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A bounded wait that gives up when it, or another of the CTA (*dead), has run out; the kernel's end raises the error
// word for it. Kept to a few instructions: the roles' loops together have to stay in the instruction cache (with
// everything inlined a tile took 7000 cycles, half of them waiting for instructions).
FYB_DEV void kt_wait(uint64_t *bar, unsigned parity, volatile unsigned *dead)
{
    if (__builtin_expect(mbar_try_wait(bar, parity & 1), 1)) return;
    for (unsigned i = 0; !mbar_try_wait(bar, parity & 1); ++i)
        if (__builtin_expect(i >= 1u << 22 || *dead, 0)) {
            *dead = 1;
            break;
        }
}
FYB_DEV unsigned kt_pack(float lo, float hi)  // fp16 pair
{
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned *>(&p);
}
FYB_DEV float2 kt_unpack(unsigned p) { return __half22float2(*reinterpret_cast<const __half2 *>(&p)); }
FYB_DEV int kt_exponent(float x) { return x > 0.f ? max(-126, (int)(__float_as_uint(x) >> 23) - 127) : 0; }
FYB_DEV float kt_power(int e) { return e < -126 ? __uint_as_float(1u << max(0, e + 149)) : __uint_as_float((unsigned)(min(e, 127) + 127) << 23); }

}  // namespace fyb
