// tcgen05 steps of the kernels whose products follow one another through tensor memory: operands read from it,
// 32-column loads and stores, and bounded waits that poll.
#pragma once
#include "common.cuh"

namespace db {
namespace chain {

// One lane of a converged warp.  MMAs are issued under this and not under a test of the lane's number: only then does the
// compiler keep their operands in uniform registers (B200, from one warp: 17 / 38 / 67 cycles per MMA of N = 16 / 64
// / 128 with A in tensor memory, against 93 for each).
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }

// D[tmem] (+)= A[tmem] * B[smem]^T, kind::f16, one CTA.  A: 128 lanes, two f16 of consecutive K per column.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 32 lanes x 32 consecutive 32-bit columns from registers into tensor memory.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
        "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
        "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// Makes every later use of r depend on this point (placed after tcgen05.wait::ld, so the compiler cannot hoist a use
// of registers loaded by tcgen05.ld above the wait).
__device__ __forceinline__ void tie32(uint32_t (&r)[32]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}

// Bounded wait of a whole warp, without suspending it (a suspended one resumes up to a microsecond late, which a chain of
// hand-offs cannot absorb).  Every lane looks: one that looked for the others cost the warp a divergence and a
// hand-over, 250 cycles even for a wait that was over.  The loop stands out of line, so that the code between two waits
// is short (B200: delta walk over 8192 tokens 812 -> 705 us, 1000 rows of cache attention 213 -> 149 us, both of these
// together).  False: the CTA was aborted, here or elsewhere, and the error word says so.
static __device__ __noinline__ bool warp_wait_on(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
    const uint64_t start = globaltimer();
    for (uint32_t i = 1;; ++i) {
        if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
        if ((i & 63u) == 0) {
            if (__any_sync(0xffffffffu, *abort_flag)) return false;
            if (__any_sync(0xffffffffu, globaltimer() - start > DB_WAIT_LIMIT_NS)) {
                *abort_flag = 1;
                if (err && (threadIdx.x & 31) == 0) atomicOr(err, code);
                return false;
            }
        }
    }
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
    if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
    return warp_wait_on(bar, parity, abort_flag, err, code);
}

}  // namespace chain
}  // namespace db
