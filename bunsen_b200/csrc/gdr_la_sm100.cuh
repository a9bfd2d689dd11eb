// What the chunked linear attention kernels on the 5th-generation tensor cores
// share: waits with a limit, TMEM access by pairs of columns, bf16 conversions.
#pragma once

#include "gdr_f32x2.cuh"
#include "gdr_sm100.cuh"

namespace gdr {
namespace sm100 {

constexpr int kWaitRounds = 1 << 20;  // of two tries of 90 cycles or more: a tenth of a second

// Waits for a phase; false once the tries ran out. A try suspends the warp for
// some 90 cycles (one with a time of its own becomes a loop of sleeps). One lane's answer:
// a role leaves its loop as a warp, so it asks warp_wait.
__device__ __forceinline__ bool lane_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b32 i;\n\t"
        "mov.b32 i, %3;\n\t"
        "LA_TRY:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra LA_DONE;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra LA_DONE;\n\t"
        "sub.s32 i, i, 1;\n\tsetp.ne.s32 q, i, 0;\n\t@q bra LA_TRY;\n\t"
        "LA_DONE:\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "n"(kWaitRounds)
        : "memory");
    return ok != 0;
}
// The same for a whole warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, lane_wait(bar, parity));
}
// One lane of a converged warp. (The compiler knows it: behind `lane == 0` it
// wraps every product, commit and copy in an election of its own, 15
// instructions each.)
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
        : "memory");
}
// 32 lanes x 8 columns, as pairs of columns, arrived.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint64_t (&v)[4]) {
    asm volatile(
        "{\n\t.reg .b32 r<8>;\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {r0, r1, r2, r3, r4, r5, r6, r7}, [%4];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t"
        "mov.b64 %0, {r0, r1};\n\tmov.b64 %1, {r2, r3};\n\t"
        "mov.b64 %2, {r4, r5};\n\tmov.b64 %3, {r6, r7};\n\t}"
        : "=l"(v[0]), "=l"(v[1]), "=l"(v[2]), "=l"(v[3])
        : "r"(taddr)
        : "memory");
}
// 32 lanes x 16 columns, as pairs of columns, arrived. (The loads take some 30
// cycles; several in flight gained nothing.)
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint64_t (&v)[8]) {
    asm volatile(
        "{\n\t.reg .b32 r<16>;\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32"
        " {r0, r1, r2, r3, r4, r5, r6, r7, r8, r9, r10, r11, r12, r13, r14, r15}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t"
        "mov.b64 %0, {r0, r1};\n\tmov.b64 %1, {r2, r3};\n\t"
        "mov.b64 %2, {r4, r5};\n\tmov.b64 %3, {r6, r7};\n\t"
        "mov.b64 %4, {r8, r9};\n\tmov.b64 %5, {r10, r11};\n\t"
        "mov.b64 %6, {r12, r13};\n\tmov.b64 %7, {r14, r15};\n\t}"
        : "=l"(v[0]), "=l"(v[1]), "=l"(v[2]), "=l"(v[3]), "=l"(v[4]), "=l"(v[5]), "=l"(v[6]),
          "=l"(v[7])
        : "r"(taddr)
        : "memory");
}

// Two f32 as bf16, x in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
__device__ __forceinline__ float low_f32(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high_f32(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

__device__ __forceinline__ uint32_t pack_bf16(uint64_t p) {
    float x, y;
    unpair(p, x, y);
    return pack_bf16(x, y);
}
__device__ __forceinline__ uint64_t widen(uint32_t p) { return pair(low_f32(p), high_f32(p)); }

}  // namespace sm100
}  // namespace gdr
