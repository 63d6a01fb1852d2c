// PTX wrappers that only the training-loss kernels use, beside sm100_ptx.cuh: bf16 operands, a
// shared-memory operand read along its rows (MN-major), 16-column TMEM accesses, the register
// split between warpgroups and the programmatic launch order of a chain of kernels.
#pragma once
#include "sm100_ptx.cuh"

namespace rh {

// Instruction descriptor, kind::f16: D f32, A and B both f16 or both bf16, A K-major; B K-major,
// or MN-major (b_mn: the contraction runs along the image's rows).
__host__ __device__ constexpr uint32_t idesc_16b(bool bf16, bool b_mn, uint32_t M, uint32_t N) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           ((N >> 3) << 17) | ((M >> 4) << 24);
}

// Descriptor of the same 128-byte-swizzled image (two halves of 64 K slots, 16 KB apart, rows of
// 128 bytes) read MN-major: N runs along the row, 64 elements per half (leading offset 16 KB),
// the contraction along the rows, 8 of them per 1024 bytes (stride offset).
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t addr) {
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3FFFu);
    d |= (uint64_t)(16384u >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}

// 16 columns of the warp's 32 lanes, in flight until tmem_ld_wait16 (which ties the registers, so no
// use can move above the wait).
__device__ __forceinline__ void tmem_ld32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_st32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Scores of a tile, f32: the products lo.hi, hi.lo and hi.hi of up to 8 K steps each. K runs along
// the image's rows' bytes (32 bytes a step, the second four steps in the image's other half; the low
// image 32 KB further); A in TMEM, 8 columns a step, the low part 64 columns further. One elect.sync
// and immediate offsets: the tensor core queues only a few instructions, so what the issuing warp
// spends between them is time it stands still.
__device__ __forceinline__ void mma_scores_f32_warp(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                                    int steps) {
    asm volatile(
        "{\n\t.reg .pred e, pf, pt, q1, q2, q3, q4, q5, q6, q7;\n\t.reg .b64 b<8>, c<8>;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 pf, 0, 0;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "setp.gt.and.s32 q1, %4, 1, e;\n\t"
        "add.s64 b1, %2, 2;\n\t"
        "setp.gt.and.s32 q2, %4, 2, e;\n\t"
        "add.s64 b2, %2, 4;\n\t"
        "setp.gt.and.s32 q3, %4, 3, e;\n\t"
        "add.s64 b3, %2, 6;\n\t"
        "setp.gt.and.s32 q4, %4, 4, e;\n\t"
        "add.s64 b4, %2, 1024;\n\t"
        "setp.gt.and.s32 q5, %4, 5, e;\n\t"
        "add.s64 b5, %2, 1026;\n\t"
        "setp.gt.and.s32 q6, %4, 6, e;\n\t"
        "add.s64 b6, %2, 1028;\n\t"
        "setp.gt.and.s32 q7, %4, 7, e;\n\t"
        "add.s64 b7, %2, 1030;\n\t"
        "add.s64 c0, %2, 2048;\n\t"
        "add.s64 c1, %2, 2050;\n\t"
        "add.s64 c2, %2, 2052;\n\t"
        "add.s64 c3, %2, 2054;\n\t"
        "add.s64 c4, %2, 3072;\n\t"
        "add.s64 c5, %2, 3074;\n\t"
        "add.s64 c6, %2, 3076;\n\t"
        "add.s64 c7, %2, 3078;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+64], %2, %3, pf;\n\t"
        "@q1 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+72], b1, %3, pt;\n\t"
        "@q2 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+80], b2, %3, pt;\n\t"
        "@q3 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+88], b3, %3, pt;\n\t"
        "@q4 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+96], b4, %3, pt;\n\t"
        "@q5 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+104], b5, %3, pt;\n\t"
        "@q6 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+112], b6, %3, pt;\n\t"
        "@q7 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+120], b7, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+0], c0, %3, pt;\n\t"
        "@q1 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+8], c1, %3, pt;\n\t"
        "@q2 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+16], c2, %3, pt;\n\t"
        "@q3 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+24], c3, %3, pt;\n\t"
        "@q4 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+32], c4, %3, pt;\n\t"
        "@q5 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+40], c5, %3, pt;\n\t"
        "@q6 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+48], c6, %3, pt;\n\t"
        "@q7 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+56], c7, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+0], %2, %3, pt;\n\t"
        "@q1 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+8], b1, %3, pt;\n\t"
        "@q2 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+16], b2, %3, pt;\n\t"
        "@q3 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+24], b3, %3, pt;\n\t"
        "@q4 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+32], b4, %3, pt;\n\t"
        "@q5 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+40], b5, %3, pt;\n\t"
        "@q6 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+48], b6, %3, pt;\n\t"
        "@q7 tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+56], b7, %3, pt;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(steps)
        : "memory");
}

// Scores of a tile, bf16: up to 8 K steps, A in shared memory, an image like B's.
__device__ __forceinline__ void mma_scores_bf16_warp(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                     int steps) {
    asm volatile(
        "{\n\t.reg .pred e, pf, pt, q1, q2, q3, q4, q5, q6, q7;\n\t.reg .b64 a<8>, b<8>;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 pf, 0, 0;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "setp.gt.and.s32 q1, %4, 1, e;\n\t"
        "add.s64 b1, %2, 2;\n\t"
        "add.s64 a1, %1, 2;\n\t"
        "setp.gt.and.s32 q2, %4, 2, e;\n\t"
        "add.s64 b2, %2, 4;\n\t"
        "add.s64 a2, %1, 4;\n\t"
        "setp.gt.and.s32 q3, %4, 3, e;\n\t"
        "add.s64 b3, %2, 6;\n\t"
        "add.s64 a3, %1, 6;\n\t"
        "setp.gt.and.s32 q4, %4, 4, e;\n\t"
        "add.s64 b4, %2, 1024;\n\t"
        "add.s64 a4, %1, 1024;\n\t"
        "setp.gt.and.s32 q5, %4, 5, e;\n\t"
        "add.s64 b5, %2, 1026;\n\t"
        "add.s64 a5, %1, 1026;\n\t"
        "setp.gt.and.s32 q6, %4, 6, e;\n\t"
        "add.s64 b6, %2, 1028;\n\t"
        "add.s64 a6, %1, 1028;\n\t"
        "setp.gt.and.s32 q7, %4, 7, e;\n\t"
        "add.s64 b7, %2, 1030;\n\t"
        "add.s64 a7, %1, 1030;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, pf;\n\t"
        "@q1 tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, pt;\n\t"
        "@q2 tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, pt;\n\t"
        "@q3 tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, pt;\n\t"
        "@q4 tcgen05.mma.cta_group::1.kind::f16 [%0], a4, b4, %3, pt;\n\t"
        "@q5 tcgen05.mma.cta_group::1.kind::f16 [%0], a5, b5, %3, pt;\n\t"
        "@q6 tcgen05.mma.cta_group::1.kind::f16 [%0], a6, b6, %3, pt;\n\t"
        "@q7 tcgen05.mma.cta_group::1.kind::f16 [%0], a7, b7, %3, pt;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(steps)
        : "memory");
}

// The second product of a tile, f32 (lo.hi, hi.lo, hi.hi): the contraction runs along the image's 128
// rows (2 KB a step); A in TMEM, 16 columns a step: 8 of the high part, then 8 of the low part.
__device__ __forceinline__ void mma_rows_f32_warp(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred e, pf, pt;\n\t.reg .b64 b<8>, c<8>;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 pf, 0, 0;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "add.s64 b1, %2, 128;\n\t"
        "add.s64 b2, %2, 256;\n\t"
        "add.s64 b3, %2, 384;\n\t"
        "add.s64 b4, %2, 512;\n\t"
        "add.s64 b5, %2, 640;\n\t"
        "add.s64 b6, %2, 768;\n\t"
        "add.s64 b7, %2, 896;\n\t"
        "add.s64 c0, %2, 2048;\n\t"
        "add.s64 c1, %2, 2176;\n\t"
        "add.s64 c2, %2, 2304;\n\t"
        "add.s64 c3, %2, 2432;\n\t"
        "add.s64 c4, %2, 2560;\n\t"
        "add.s64 c5, %2, 2688;\n\t"
        "add.s64 c6, %2, 2816;\n\t"
        "add.s64 c7, %2, 2944;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+8], %2, %3, pf;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+24], b1, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+40], b2, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+56], b3, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+72], b4, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+88], b5, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+104], b6, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+120], b7, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+0], c0, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+16], c1, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+32], c2, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+48], c3, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+64], c4, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+80], c5, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+96], c6, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+112], c7, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+0], %2, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+16], b1, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+32], b2, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+48], b3, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+64], b4, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+80], b5, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+96], b6, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+112], b7, %3, pt;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc)
        : "memory");
}

// The same in bf16 (8 of a step's 16 columns), added to the accumulator where `accumulate` is set.
__device__ __forceinline__ void mma_rows_bf16_warp(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                                   uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, pf, pt;\n\t.reg .b64 b<8>;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 pf, %4, 0;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "add.s64 b1, %2, 128;\n\t"
        "add.s64 b2, %2, 256;\n\t"
        "add.s64 b3, %2, 384;\n\t"
        "add.s64 b4, %2, 512;\n\t"
        "add.s64 b5, %2, 640;\n\t"
        "add.s64 b6, %2, 768;\n\t"
        "add.s64 b7, %2, 896;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+0], %2, %3, pf;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+16], b1, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+32], b2, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+48], b3, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+64], b4, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+80], b5, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+96], b6, %3, pt;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1+112], b7, %3, pt;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// All phases complete? The try_waits issue back to back, so their latencies overlap.
__device__ __forceinline__ bool mbar_try_wait3(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1,
                                               uint32_t bar2, uint32_t parity2) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p0, p1, p2;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p0, [%1], %2;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p1, [%3], %4;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p2, [%5], %6;\n\t"
        "and.pred p0, p0, p1;\n\t"
        "and.pred p0, p0, p2;\n\t"
        "selp.u32 %0, 1, 0, p0;\n\t}"
        : "=r"(ok)
        : "r"(bar0), "r"(parity0), "r"(bar1), "r"(parity1), "r"(bar2), "r"(parity2)
        : "memory");
    return ok != 0;
}

// Programmatic launch order: the next kernel of the chain may start its own set-up now; nothing of
// the one before may be read or overwritten before the wait, which sees it complete.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void setmaxnreg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void setmaxnreg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

}  // namespace rh
