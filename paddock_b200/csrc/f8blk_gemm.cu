// f8blk_gemm.cu - products of block-scaled e4m3 operands (f8blk.cuh): entry points.
//
//   y[t][n] = sum_b xs[t][b] * ws[n / 128][b] * ( sum_{k in block b} xq[t][k] * wq[n][k] )
//   h[t][f] = silu(g) * u of two such products, left quantized in blocks of 128 f per token
#include "cluster_caps.cuh"
#include "f8blk_plan.cuh"
#include "f8blk_tc5.cuh"

namespace {

bool operands_ok(const void* w, const void* ws, const void* xq, const void* xs, uint32_t in_dim, uint32_t out_dim, uint32_t batch) {
    constexpr uint32_t kMost = 0x7fffff00u;   // coordinates of a box are signed
    return w && ws && xq && xs && in_dim != 0u && (in_dim & 15u) == 0u && in_dim <= kMost && out_dim <= kMost && batch <= kMost &&
           pdk_aligned(w, 16) && pdk_aligned(xq, 16) && pdk_aligned(ws, 4) && pdk_aligned(xs, 4);
}

int plan_of(int planes, uint32_t in_dim, uint32_t out_dim, uint32_t batch, f8blk::Plan* plan) {
    const uint32_t* resident[2] = {nullptr, nullptr};
    if (int rc = pdk_f8blk_split_clusters(planes, resident)) return rc;
    *plan = f8blk::choose(planes, in_dim, out_dim, batch, resident, kPdkMaxCluster, (uint32_t)pdk_sm_count());
    return 0;
}
int launch(const f8blk::Call& c, int planes, bool bf16, cudaStream_t st) {
    f8blk::Plan p;
    if (int rc = plan_of(planes, c.in_dim, c.out_dim, c.batch, &p)) return rc;
    return p.kernel == 2u ? pdk_f8blk_wide(c, planes, bf16, p.cols, st) : pdk_f8blk_split(c, planes, bf16, p.cols, p.split, st);
}

int gemm(const void* w, const void* ws, const void* xq, const void* xs, void* y, uint32_t in_dim, uint32_t out_dim, uint32_t batch, bool bf16,
         cudaStream_t st) {
    if (out_dim == 0u || batch == 0u) return 0;
    if (!operands_ok(w, ws, xq, xs, in_dim, out_dim, batch) || !y || !pdk_aligned(y, bf16 ? 2 : 4)) return cudaErrorInvalidValue;
    const f8blk::Call c{{w, nullptr}, {ws, nullptr}, xq, xs, y, nullptr, in_dim, out_dim, batch};
    return launch(c, 1, bf16, st);
}

// Two warps wait on barriers that nothing arrives on.  The first gives up after `budget_ns`, the second, whose own limit is the kernels', by the
// first one's flag.  Each vote is the whole warp's, as behind every wait of the products.
__global__ void wait_selftest_kernel(unsigned long long budget_ns, unsigned int* err_word, unsigned int* left) {
    __shared__ uint64_t bar[2];
    __shared__ int abort_flag;
    const uint32_t warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        tc5::mbar_init(&bar[0], 1);
        tc5::mbar_init(&bar[1], 1);
        abort_flag = 0;
        tc5::mbar_fence_init();
    }
    __syncthreads();
    const tc5::WaitCtx ctx{&abort_flag, err_word};
    const bool ok = __all_sync(0xffffffffu, f8blk::wait_soon(&bar[warp], 0u, ctx, tc5::kErrTestWait, 8u + warp, warp == 0u ? budget_ns : tc5::kWaitBudgetNs));
    if ((threadIdx.x & 31u) == 0u) left[warp] = ok ? 2u : 1u;      // 1 = gave up as designed
}

}  // namespace

PDK_EXPORT int pdk_f8blk_gemm(const void* data, const void* w_scale, const void* xq, const void* x_scale, void* y, uint32_t in_dim,
                              uint32_t out_dim, uint32_t batch, void* stream) {
    return gemm(data, w_scale, xq, x_scale, y, in_dim, out_dim, batch, false, (cudaStream_t)stream);
}
PDK_EXPORT int pdk_f8blk_gemm_bf16(const void* data, const void* w_scale, const void* xq, const void* x_scale, void* y, uint32_t in_dim,
                                   uint32_t out_dim, uint32_t batch, void* stream) {
    return gemm(data, w_scale, xq, x_scale, y, in_dim, out_dim, batch, true, (cudaStream_t)stream);
}
PDK_EXPORT int pdk_f8blk_gate_up(const void* gate_data, const void* gate_scale, const void* up_data, const void* up_scale, const void* xq,
                                 const void* x_scale, void* hq, void* h_scale, uint32_t in_dim, uint32_t ff, uint32_t batch, void* stream) {
    if (ff == 0u || batch == 0u) return 0;
    if (!operands_ok(gate_data, gate_scale, xq, x_scale, in_dim, ff, batch) || !operands_ok(up_data, up_scale, xq, x_scale, in_dim, ff, batch) ||
        !hq || !h_scale || (ff & 15u) != 0u || !pdk_aligned(hq, 16) || !pdk_aligned(h_scale, 4))
        return cudaErrorInvalidValue;
    const f8blk::Call c{{gate_data, up_data}, {gate_scale, up_scale}, xq, x_scale, hq, h_scale, in_dim, ff, batch};
    return launch(c, 2, false, (cudaStream_t)stream);
}

// Diagnostics: the plan of a product (planes 1) or gated front (planes 2) on the current device
PDK_EXPORT int pdk_f8blk_plan(uint32_t planes, uint32_t in_dim, uint32_t out_dim, uint32_t batch, uint32_t* plan) {
    if (planes < 1u || planes > 2u || in_dim == 0u || out_dim == 0u || batch == 0u || !plan) return cudaErrorInvalidValue;
    f8blk::Plan p;
    if (int rc = plan_of((int)planes, in_dim, out_dim, batch, &p)) return rc;
    plan[0] = p.kernel; plan[1] = p.cols; plan[2] = p.split;
    return 0;
}

// Runs the timed-out path of these kernels' waits (one of two waits with a limit of budget_us, 1..100000): 0 when both gave up and the kernel
// exited; pdk_device_error() then reads kErrTestWait << 8 | 8.  `scratch` is 8 bytes of device memory.  Synchronizes.
PDK_EXPORT int pdk_selftest_f8blk_wait(uint32_t budget_us, void* scratch, void* stream) {
    if (budget_us == 0u || budget_us > 100000u || !scratch || !pdk_aligned(scratch, 4)) return cudaErrorInvalidValue;
    const cudaStream_t st = (cudaStream_t)stream;
    if (cudaError_t e = cudaMemsetAsync(scratch, 0, 8, st); e != cudaSuccess) return (int)e;
    wait_selftest_kernel<<<1, 64, 0, st>>>((unsigned long long)budget_us * 1000ull, pdk_error_word(), (unsigned int*)scratch);
    if (int rc = pdk_launch_status()) return rc;
    if (cudaError_t e = cudaStreamSynchronize(st); e != cudaSuccess) return (int)e;
    unsigned int left[2] = {0u, 0u};
    if (cudaError_t e = cudaMemcpy(left, scratch, 8, cudaMemcpyDeviceToHost); e != cudaSuccess) return (int)e;
    return left[0] == 1u && left[1] == 1u ? 0 : cudaErrorUnknown;
}
