// f8blk_tc5.cuh - what the two tensor-core kernels of block-scaled e4m3 products share.
//
// The scales of a block are arbitrary f32, so the tensor core cannot apply them: it sums one 128-element block of K at a time into
// tensor memory (kind::f8f6f4, f32), and the epilogue warps, which keep the product in registers, add it on with the block's
// two scales while the tensor core does the next block.  The two are multiplied first, which is one number a token or column; a product of
// theirs outside f32 takes the term with it, though the sum might have brought it back.  That costs one fused multiply-add per element and block, and reading every
// element of tensor memory once per block.
#pragma once
#include "f8blk.cuh"
#include "tc5.cuh"

namespace f8blk {

// One plane or, for the gated front, two; y = f32 / bf16 product, or hq with hs.
struct Call {
    const void *w[2], *ws[2], *xq, *xs;
    void *y, *hs;
    uint32_t in_dim, out_dim, batch;
};

// tc5::mbar_wait that reads the global timer only after some failed attempts: these waits are short and one per block of K.
__device__ __forceinline__ bool wait_soon(uint64_t* bar, uint32_t parity, const tc5::WaitCtx& ctx, unsigned int code, unsigned int detail,
                                          unsigned long long budget_ns = tc5::kWaitBudgetNs) {
    for (uint32_t i = 0; i < 64u; ++i)
        if (tc5::mbar_try_wait(bar, parity)) return true;
    return tc5::mbar_wait(bar, parity, ctx, code, detail, budget_ns);
}

// One arrival of a converged warp (tc5.cuh has why not from a branch of one lane).
__device__ __forceinline__ void mbar_arrive_elect(uint64_t* bar) {
    asm volatile(TC5_ELECT "@e mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(tc5::smem_u32(bar)) : "memory");
}

// For a CTA in which a wait ran out, every role past its loop: boxes that were requested, and MMAs that read them, may still be on their way
// into memory that the next CTA gets.  64 us are far more than they take.
__device__ __forceinline__ void wait_for_copies() {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
}

// The wait for this warp's loads, as what hands their registers on: nothing that uses them can be moved in front of it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                   "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                   "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// silu(g) * u, g / (1 + exp(-g)) * u.  The quotient is the hardware's (2 units): an IEEE one has a rare path that is branched to, which keeps
// neighbouring elements from overlapping.  It is 0 for divisors beyond 2^126, which a negative gate has from -87.34 on: there the divisor comes
// down by 4 and the quotient with it.  Both are exact, and a divisor that is a number stays below 2^126.  A positive gate's divisor is at most 2, and
// its quotient would pass f32 for gates beyond 2^126.
__device__ __forceinline__ float gated(float g, float u) {
    const float c = g < 0.0f ? 0.25f : 1.0f;
    return __fdividef(g, c * (1.0f + expf(-g))) * c * u;
}

}  // namespace f8blk

// f8blk_split.cu, f8blk_wide.cu: 0 or a cudaError_t
int pdk_f8blk_split_clusters(int planes, const uint32_t* resident[2]);
int pdk_f8blk_split(const f8blk::Call& c, int planes, bool bf16, uint32_t cols, uint32_t split, cudaStream_t st);
int pdk_f8blk_wide(const f8blk::Call& c, int planes, bool bf16, uint32_t cols, cudaStream_t st);
