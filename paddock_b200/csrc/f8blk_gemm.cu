// f8blk_gemm.cu - products of block-scaled e4m3 operands (f8blk.cuh): entry points.
//
//   y[t][n] = sum_b xs[t][b] * ws[n / 128][b] * ( sum_{k in block b} xq[t][k] * wq[n][k] )
//   h[t][f] = silu(g) * u of two such products, left quantized in blocks of 128 f per token
#include "f8blk.cuh"

namespace {

using namespace f8blk;

// one warp: the product of a token's row and a channel's, 16 bytes a lane and turn
__device__ __forceinline__ float row_product(const uint8_t* __restrict__ w, const float* __restrict__ ws, const uint8_t* __restrict__ x,
                                             const float* __restrict__ xs, uint32_t in_dim) {
    float sum = 0.0f;
    for (uint32_t k = (threadIdx.x & 31u) * 16u; k < in_dim; k += 512u) {
        const uint4 a = *reinterpret_cast<const uint4*>(w + k), b = *reinterpret_cast<const uint4*>(x + k);
        const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
        float part = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const float2 a0 = values2(aw[i] & 0xffffu), a1 = values2(aw[i] >> 16), b0 = values2(bw[i] & 0xffffu), b1 = values2(bw[i] >> 16);
            part = fmaf(a0.x, b0.x, part); part = fmaf(a0.y, b0.y, part);
            part = fmaf(a1.x, b1.x, part); part = fmaf(a1.y, b1.y, part);
        }
        sum = fmaf(part, ws[k / kBlock] * xs[k / kBlock], sum);
    }
    return pdk_warp_sum(sum);
}
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// a CTA per token and 128 channels
template <typename TO>
__global__ void __launch_bounds__(256) gemm_kernel(const uint8_t* w, const float* ws, const uint8_t* x, const float* xs, TO* y, uint32_t in_dim,
                                                   uint32_t out_dim, uint32_t tiles) {
    const uint32_t t = blockIdx.x / tiles, tile = blockIdx.x % tiles, kb = blocks_of(in_dim);
    for (uint32_t n = tile * kBlock + (threadIdx.x >> 5); n < min(out_dim, (tile + 1u) * kBlock); n += 8u) {
        const float v = row_product(w + (size_t)n * in_dim, ws + (size_t)tile * kb, x + (size_t)t * in_dim, xs + (size_t)t * kb, in_dim);
        if ((threadIdx.x & 31u) == 0u) put(y + (size_t)t * out_dim + n, v);
    }
}
__global__ void __launch_bounds__(256) gate_up_kernel(const uint8_t* g, const float* gs, const uint8_t* u, const float* us, const uint8_t* x,
                                                      const float* xs, uint8_t* hq, float* hs, uint32_t in_dim, uint32_t ff, uint32_t tiles) {
    __shared__ float h[kBlock];
    const uint32_t t = blockIdx.x / tiles, tile = blockIdx.x % tiles, kb = blocks_of(in_dim);
    if (threadIdx.x < kBlock) h[threadIdx.x] = 0.0f;
    __syncthreads();
    for (uint32_t n = tile * kBlock + (threadIdx.x >> 5); n < min(ff, (tile + 1u) * kBlock); n += 8u) {
        const float a = row_product(g + (size_t)n * in_dim, gs + (size_t)tile * kb, x + (size_t)t * in_dim, xs + (size_t)t * kb, in_dim);
        const float b = row_product(u + (size_t)n * in_dim, us + (size_t)tile * kb, x + (size_t)t * in_dim, xs + (size_t)t * kb, in_dim);
        if ((threadIdx.x & 31u) == 0u) h[n % kBlock] = a / (1.0f + expf(-a)) * b;
    }
    __syncthreads();
    float a = 0.0f;
    for (uint32_t i = 0; i < kBlock; ++i) a = fmaxf(a, fabsf(h[i]));
    const float s = scale_of(a);
    const uint32_t n = tile * kBlock + threadIdx.x;
    if (threadIdx.x < kBlock && n < ff) hq[(size_t)t * ff + n] = code1(h[threadIdx.x], 1.0f / s);
    if (threadIdx.x == 0u) hs[(size_t)t * tiles + tile] = s;
}

bool operands_ok(const void* w, const void* ws, const void* xq, const void* xs, uint32_t in_dim, uint32_t out_dim, uint32_t batch) {
    constexpr uint32_t kMost = 0x7fffff00u;   // coordinates of a box are signed
    return w && ws && xq && xs && in_dim != 0u && (in_dim & 15u) == 0u && in_dim <= kMost && out_dim <= kMost && batch <= kMost &&
           pdk_aligned(w, 16) && pdk_aligned(xq, 16) && pdk_aligned(ws, 4) && pdk_aligned(xs, 4);
}

template <typename TO>
int gemm(const void* w, const void* ws, const void* xq, const void* xs, void* y, uint32_t in_dim, uint32_t out_dim, uint32_t batch,
         cudaStream_t st) {
    if (out_dim == 0u || batch == 0u) return 0;
    if (!operands_ok(w, ws, xq, xs, in_dim, out_dim, batch) || !y || !pdk_aligned(y, sizeof(TO))) return cudaErrorInvalidValue;
    const uint32_t tiles = blocks_of(out_dim);
    gemm_kernel<TO><<<batch * tiles, 256, 0, st>>>((const uint8_t*)w, (const float*)ws, (const uint8_t*)xq, (const float*)xs, (TO*)y, in_dim,
                                                   out_dim, tiles);
    return pdk_launch_status();
}

}  // namespace

PDK_EXPORT int pdk_f8blk_gemm(const void* data, const void* w_scale, const void* xq, const void* x_scale, void* y, uint32_t in_dim,
                              uint32_t out_dim, uint32_t batch, void* stream) {
    return gemm<float>(data, w_scale, xq, x_scale, y, in_dim, out_dim, batch, (cudaStream_t)stream);
}
PDK_EXPORT int pdk_f8blk_gemm_bf16(const void* data, const void* w_scale, const void* xq, const void* x_scale, void* y, uint32_t in_dim,
                                   uint32_t out_dim, uint32_t batch, void* stream) {
    return gemm<__nv_bfloat16>(data, w_scale, xq, x_scale, y, in_dim, out_dim, batch, (cudaStream_t)stream);
}
PDK_EXPORT int pdk_f8blk_gate_up(const void* gate_data, const void* gate_scale, const void* up_data, const void* up_scale, const void* xq,
                                 const void* x_scale, void* hq, void* h_scale, uint32_t in_dim, uint32_t ff, uint32_t batch, void* stream) {
    if (ff == 0u || batch == 0u) return 0;
    if (!operands_ok(gate_data, gate_scale, xq, x_scale, in_dim, ff, batch) || !operands_ok(up_data, up_scale, xq, x_scale, in_dim, ff, batch) ||
        !hq || !h_scale || (ff & 15u) != 0u || !pdk_aligned(hq, 16) || !pdk_aligned(h_scale, 4))
        return cudaErrorInvalidValue;
    const uint32_t tiles = f8blk::blocks_of(ff);
    gate_up_kernel<<<batch * tiles, 256, 0, (cudaStream_t)stream>>>((const uint8_t*)gate_data, (const float*)gate_scale, (const uint8_t*)up_data,
                                                                    (const float*)up_scale, (const uint8_t*)xq, (const float*)x_scale,
                                                                    (uint8_t*)hq, (float*)h_scale, in_dim, ff, tiles);
    return pdk_launch_status();
}
