// f8blk_quant.cu - what writes and reads block-scaled e4m3 operands (f8blk.cuh has the formats and the rule): the activation
// quantizer, its form behind residual add and RMSNorm, the weight quantizer and the way back to f32.
//
// All are bound by HBM; what each layout buys is one pass: a block's values stay in registers from the load to the store.
#include "f8blk.cuh"

namespace {

using namespace f8blk;

__device__ __forceinline__ float amax_of(const float4& v) {
    return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
}
template <uint32_t kLanes>
__device__ __forceinline__ float max_over(float a) {   // aligned groups of kLanes lanes
#pragma unroll
    for (uint32_t d = 1; d < kLanes; d <<= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
    return a;
}

// ---- activations --------------------------------------------------------------------------------------------
// 16 bytes a lane: a block is 32 lanes of f32 or 16 lanes of bf16, whose maximum takes five or four shuffles.
template <typename T>
struct Piece;
template <>
struct Piece<float> {
    static constexpr uint32_t kElems = 4, kLanes = 32;
    float4 v;
    __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void zero() { v = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ float amax() const { return amax_of(v); }
    __device__ __forceinline__ void store(uint8_t* q, float r) const { *reinterpret_cast<uint32_t*>(q) = codes4(v.x, v.y, v.z, v.w, r); }
};
template <>
struct Piece<__nv_bfloat16> {
    static constexpr uint32_t kElems = 8, kLanes = 16;
    uint4 v;
    static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void zero() { v = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ float amax() const {
        return fmaxf(amax_of(make_float4(lo(v.x), hi(v.x), lo(v.y), hi(v.y))), amax_of(make_float4(lo(v.z), hi(v.z), lo(v.w), hi(v.w))));
    }
    __device__ __forceinline__ uint2 codes(float r) const {
        return make_uint2(codes4(lo(v.x), hi(v.x), lo(v.y), hi(v.y), r), codes4(lo(v.z), hi(v.z), lo(v.w), hi(v.w), r));
    }
    __device__ __forceinline__ void store(uint8_t* q, float r) const { *reinterpret_cast<uint2*>(q) = codes(r); }
};

constexpr uint32_t kQuantThreads = 256;
constexpr uint32_t kMostElems = 0xffffff00u;   // of a row, so that the end of its last block is still a number of 32 bits

// kEach blocks per group of lanes, their loads in flight together.  Rows of whole pieces, aligned.  4096 rows of 5120 f32 17.6 us, 5.97 TB/s (24.5
// with one block each, 18.5 with two); 1000 rows of 17408 bf16 10.0 us, 5.2 TB/s; 64 rows of 5120 1.8 us, a launch.
template <typename T, uint32_t kEach>
__global__ void __launch_bounds__(kQuantThreads) quantize_blk_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                                     float* __restrict__ scale, uint32_t n, uint32_t per_row, uint32_t total) {
    using P = Piece<T>;
    constexpr uint32_t kGroups = kQuantThreads / P::kLanes;
    const uint32_t sub = threadIdx.x % P::kLanes, first = blockIdx.x * (kGroups * kEach) + threadIdx.x / P::kLanes;
    pdk_pdl_launch_dependents();
    pdk_pdl_wait();
    P piece[kEach];
    size_t at[kEach];
    bool live[kEach];
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t b = first + i * kGroups, row = b / per_row, col = (b - row * per_row) * kBlock + sub * P::kElems;
        live[i] = b < total && col < n;
        at[i] = (size_t)row * n + col;
        piece[i].zero();
        if (live[i]) piece[i].load(x + at[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t b = first + i * kGroups;
        const float s = scale_of(max_over<P::kLanes>(piece[i].amax()));
        if (live[i]) piece[i].store(q + at[i], 1.0f / s);
        if (sub == 0u && b < total) scale[b] = s;
    }
}

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// Any row length and alignment: a warp per block, element by element.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_blk_any_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                                         float* __restrict__ scale, uint32_t n, uint32_t per_row,
                                                                         uint32_t total) {
    const uint32_t lane = threadIdx.x & 31u, b = blockIdx.x * (kQuantThreads / 32u) + (threadIdx.x >> 5);
    pdk_pdl_launch_dependents();
    pdk_pdl_wait();
    if (b >= total) return;
    const uint32_t row = b / per_row, col0 = (b - row * per_row) * kBlock;
    const size_t at = (size_t)row * n;
    float v[4], a = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t col = col0 + i * 32u + lane;
        v[i] = col < n ? widen(x[at + col]) : 0.0f;
        a = fmaxf(a, fabsf(v[i]));
    }
    const float s = scale_of(max_over<32>(a)), r = 1.0f / s;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t col = col0 + i * 32u + lane;
        if (col < n) q[at + col] = code1(v[i], r);
    }
    if (lane == 0u) scale[b] = s;
}

template <typename T>
int quantize(const void* x, void* q, void* scale, uint32_t n, uint32_t batch, cudaStream_t st) {
    if (n == 0u || batch == 0u) return 0;
    if (!x || !q || !scale || !pdk_aligned(x, sizeof(T)) || !pdk_aligned(scale, 4)) return cudaErrorInvalidValue;
    const uint32_t per_row = blocks_of(n);
    if (n > kMostElems || (uint64_t)per_row * batch > 0xffff0000ull) return cudaErrorInvalidValue;   // columns and blocks are numbered in 32 bits
    const uint32_t total = per_row * batch;
    using P = Piece<T>;
    if (n % P::kElems != 0u || !pdk_aligned(x, 16) || !pdk_aligned(q, P::kElems)) {
        const uint32_t per = kQuantThreads / 32u;
        return pdk_launch_pdl(quantize_blk_any_kernel<T>, dim3(total / per + (total % per != 0u)), dim3(kQuantThreads), 0, st, (const T*)x,
                              (uint8_t*)q, (float*)scale, n, per_row, total);
    }
    constexpr uint32_t kGroups = kQuantThreads / P::kLanes;
    // four blocks a group of lanes once that still leaves every SM eight thread blocks
    const uint32_t each = total >= (uint32_t)pdk_sm_count() * 8u * kGroups * 4u ? 4u : 1u, per = kGroups * each;
    const dim3 grid(total / per + (total % per != 0u));
    if (each == 4u)
        return pdk_launch_pdl(quantize_blk_kernel<T, 4>, grid, dim3(kQuantThreads), 0, st, (const T*)x, (uint8_t*)q, (float*)scale, n, per_row,
                              total);
    return pdk_launch_pdl(quantize_blk_kernel<T, 1>, grid, dim3(kQuantThreads), 0, st, (const T*)x, (uint8_t*)q, (float*)scale, n, per_row, total);
}

// ---- residual add + RMSNorm + quantizer ------------------------------------------------------------------------
// One CTA per row, which stays in registers: thread t holds the row's float4 number t, t + T, t + 2T, ... (T threads, whole warps), so
// a warp's 32 pieces of one turn are 128 neighbouring elements on a 128-element boundary: exactly one block.  The mean square is an
// f32 tree (per thread, lanes, warps in warp order).  4096 rows of 5120 with residual and xn 55.2 us, 6.46 TB/s; 7 rows 2.8 us.  Rows beyond 32768
// elements hold 16 pieces a thread and spill some of them.
constexpr uint32_t kNormThreads = 1024;

template <uint32_t kChunks>
__global__ void __launch_bounds__(kNormThreads) add_rmsnorm_quant_blk_kernel(float* __restrict__ x, const float* __restrict__ proj,
                                                                             const float* __restrict__ w, float* __restrict__ xn,
                                                                             uint8_t* __restrict__ q, float* __restrict__ scale, uint32_t n,
                                                                             float eps) {
    __shared__ float warp_sq[32];
    const uint32_t t = threadIdx.x, width = blockDim.x, n4 = n >> 2, lane = t & 31u;
    const size_t row4 = (size_t)blockIdx.x * n4;
    float4* xr = reinterpret_cast<float4*>(x) + row4;
    pdk_pdl_launch_dependents();
    pdk_pdl_wait();
    float4 v[kChunks];
    float sq = 0.0f;
#pragma unroll
    for (uint32_t c = 0; c < kChunks; ++c) {
        const uint32_t at = c * width + t;
        v[c] = at < n4 ? xr[at] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    if (proj != nullptr) {
        const float4* pr = reinterpret_cast<const float4*>(proj) + row4;
#pragma unroll
        for (uint32_t c = 0; c < kChunks; ++c) {
            const uint32_t at = c * width + t;
            const float4 p = at < n4 ? pr[at] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            v[c].x += p.x; v[c].y += p.y; v[c].z += p.z; v[c].w += p.w;
            if (at < n4) xr[at] = v[c];
        }
    }
#pragma unroll
    for (uint32_t c = 0; c < kChunks; ++c) sq += (v[c].x * v[c].x + v[c].y * v[c].y) + (v[c].z * v[c].z + v[c].w * v[c].w);
    sq = pdk_warp_sum(sq);
    if (lane == 0u) warp_sq[t >> 5] = sq;
    __syncthreads();
    float sum = 0.0f;
    for (uint32_t i = 0; i < (width >> 5); ++i) sum += warp_sq[i];
    const float norm = 1.0f / sqrtf(sum / (float)n + eps);
    const uint32_t per_row = blocks_of(n);
#pragma unroll
    for (uint32_t c = 0; c < kChunks; ++c) {
        const uint32_t at = c * width + t;
        float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (at < n4) {
            const float4 g = reinterpret_cast<const float4*>(w)[at];
            r = make_float4(v[c].x * norm * g.x, v[c].y * norm * g.y, v[c].z * norm * g.z, v[c].w * norm * g.w);
            if (xn != nullptr) (reinterpret_cast<float4*>(xn) + row4)[at] = r;
        }
        const float s = scale_of(max_over<32>(amax_of(r)));
        if (at < n4) {
            reinterpret_cast<uint32_t*>(q)[row4 + at] = codes4(r.x, r.y, r.z, r.w, 1.0f / s);
            if (lane == 0u) scale[(size_t)blockIdx.x * per_row + (at >> 5)] = s;
        }
    }
}

// ---- weights -----------------------------------------------------------------------------------------------------
constexpr uint32_t kTileThreads = 256;

__device__ __forceinline__ float block_max(float a, float* per_warp) {
    a = max_over<32>(a);
    if ((threadIdx.x & 31u) == 0u) per_warp[threadIdx.x >> 5] = a;
    __syncthreads();
    float m = per_warp[0];
#pragma unroll
    for (uint32_t i = 1; i < kTileThreads / 32u; ++i) m = fmaxf(m, per_warp[i]);
    return m;
}

// A CTA per tile: 16 threads of 16 bytes span a tile's row, eight rows a thread, all its loads in flight before the maximum.  Four CTAs an
// SM: 5120 x 17408 40.6 us, 6.6 TB/s (48 with the 87 registers a thread that the compiler would take, which leave room for two).
__global__ void __launch_bounds__(kTileThreads, 4) bf16_to_f8blk_kernel(const __nv_bfloat16* __restrict__ w, uint8_t* __restrict__ q,
                                                                        float* __restrict__ scale, uint32_t in_dim, uint32_t out_dim,
                                                                        uint32_t per_row) {
    __shared__ float per_warp[kTileThreads / 32u];
    const uint32_t tile_n = blockIdx.x / per_row, tile_k = blockIdx.x - tile_n * per_row;
    const uint32_t col = tile_k * kBlock + (threadIdx.x & 15u) * 8u, row0 = tile_n * kBlock + (threadIdx.x >> 4);
    // this thread's rows of the tile, 16 apart
    const uint32_t rows = col < in_dim && row0 < out_dim ? (min(out_dim - row0, kBlock - (threadIdx.x >> 4)) + 15u) / 16u : 0u;
    const size_t at = (size_t)row0 * in_dim + col, step = (size_t)in_dim * 16u;
    Piece<__nv_bfloat16> piece[8];
    const __nv_bfloat16* from = w + at;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
        piece[i].zero();
        if (i < rows) piece[i].load(from);
        from += step;
    }
    float a = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) a = fmaxf(a, piece[i].amax());
    const float s = scale_of(block_max(a, per_warp)), r = 1.0f / s;
    if (threadIdx.x == 0u) scale[blockIdx.x] = s;
    uint8_t* to = q + at;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
        if (i < rows) piece[i].store(to, r);
        to += step;
    }
}

// Any row length and alignment, element by element: the tile is read twice.
__global__ void __launch_bounds__(kTileThreads) bf16_to_f8blk_any_kernel(const __nv_bfloat16* __restrict__ w, uint8_t* __restrict__ q,
                                                                         float* __restrict__ scale, uint32_t in_dim, uint32_t out_dim,
                                                                         uint32_t per_row) {
    __shared__ float per_warp[kTileThreads / 32u];
    const uint32_t tile_n = blockIdx.x / per_row, tile_k = blockIdx.x - tile_n * per_row;
    const uint32_t col = tile_k * kBlock + (threadIdx.x & 127u), row0 = tile_n * kBlock, row1 = min(out_dim - row0, kBlock) + row0;
    float a = 0.0f;
    for (uint32_t row = row0 + (threadIdx.x >> 7); row < row1; row += 2u)
        if (col < in_dim) a = fmaxf(a, fabsf(__bfloat162float(w[(size_t)row * in_dim + col])));
    const float s = scale_of(block_max(a, per_warp)), r = 1.0f / s;
    if (threadIdx.x == 0u) scale[blockIdx.x] = s;
    for (uint32_t row = row0 + (threadIdx.x >> 7); row < row1; row += 2u)
        if (col < in_dim) q[(size_t)row * in_dim + col] = code1(__bfloat162float(w[(size_t)row * in_dim + col]), r);
}

// A CTA per tile, 16 lanes a row of it: eight codes a lane in, 32 bytes out, eight rows' loads in flight.  One store of 32 bytes rather than
// two of 16 (`whole`: y is on a 32-byte boundary): 5120 x 5003 21.2 us, 6.05 TB/s, instead of 22.3.
__global__ void __launch_bounds__(kTileThreads) f8blk_dequant_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                                     float* __restrict__ y, uint32_t in_dim, uint32_t out_dim, uint32_t per_row,
                                                                     uint32_t whole) {
    const uint32_t tile_n = blockIdx.x / per_row, tile_k = blockIdx.x - tile_n * per_row;
    const uint32_t col = tile_k * kBlock + (threadIdx.x & 15u) * 8u, row0 = tile_n * kBlock + (threadIdx.x >> 4);
    pdk_pdl_launch_dependents();
    pdk_pdl_wait();
    const float s = scale[blockIdx.x];
    const uint32_t rows = col < in_dim && row0 < out_dim ? (min(out_dim - row0, kBlock - (threadIdx.x >> 4)) + 15u) / 16u : 0u;
    const size_t at = (size_t)row0 * in_dim + col, step = (size_t)in_dim * 16u;
    uint2 c[8];
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) c[i] = i < rows ? *reinterpret_cast<const uint2*>(q + at + i * step) : make_uint2(0u, 0u);
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
        const float2 v0 = values2(c[i].x & 0xffffu), v1 = values2(c[i].x >> 16), v2 = values2(c[i].y & 0xffffu), v3 = values2(c[i].y >> 16);
        if (i >= rows) continue;
        float* p = y + at + i * step;
        if (whole) {
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v0.x * s), "f"(v0.y * s), "f"(v1.x * s), "f"(v1.y * s),
                         "f"(v2.x * s), "f"(v2.y * s), "f"(v3.x * s), "f"(v3.y * s)
                         : "memory");
        } else {
            reinterpret_cast<float4*>(p)[0] = make_float4(v0.x * s, v0.y * s, v1.x * s, v1.y * s);
            reinterpret_cast<float4*>(p)[1] = make_float4(v2.x * s, v2.y * s, v3.x * s, v3.y * s);
        }
    }
}
__global__ void __launch_bounds__(kTileThreads) f8blk_dequant_any_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                                         float* __restrict__ y, uint32_t in_dim, uint32_t out_dim,
                                                                         uint32_t per_row) {
    const uint32_t tile_n = blockIdx.x / per_row, tile_k = blockIdx.x - tile_n * per_row;
    const uint32_t col = tile_k * kBlock + (threadIdx.x & 127u), row0 = tile_n * kBlock, row1 = min(out_dim - row0, kBlock) + row0;
    pdk_pdl_launch_dependents();
    pdk_pdl_wait();
    const float s = scale[blockIdx.x];
    for (uint32_t row = row0 + (threadIdx.x >> 7); row < row1; row += 2u)
        if (col < in_dim) y[(size_t)row * in_dim + col] = values2(q[(size_t)row * in_dim + col]).x * s;
}

}  // namespace

// No slot: activations f32 [batch][n] -> e4m3 and a scale per token and 128 elements
PDK_EXPORT int pdk_quantize_e4m3_blk(const void* x, void* q, void* scale, uint32_t n, uint32_t batch, void* stream) {
    return quantize<float>(x, q, scale, n, batch, (cudaStream_t)stream);
}
PDK_EXPORT int pdk_quantize_e4m3_blk_bf16(const void* x, void* q, void* scale, uint32_t n, uint32_t batch, void* stream) {
    return quantize<__nv_bfloat16>(x, q, scale, n, batch, (cudaStream_t)stream);
}

// No slot: slot 513's step in front of block-scaled operands
PDK_EXPORT int pdk_add_rmsnorm_quant_e4m3_blk(void* x, const void* proj, const void* w, void* xn, void* q, void* scale, uint32_t n, float eps,
                                              uint32_t batch, void* stream) {
    if (n == 0u || batch == 0u) return 0;
    if (!x || !w || !q || !scale || (n & 3u) != 0u || batch > 0x7fffffffu || !pdk_aligned(x, 16) || !pdk_aligned(proj, 16) || !pdk_aligned(w, 16) ||
        !pdk_aligned(xn, 16) || !pdk_aligned(q, 4) || !pdk_aligned(scale, 4))
        return cudaErrorInvalidValue;
    const uint32_t n4 = n >> 2;
    uint32_t chunks = 1;
    while (chunks < 16u && (n4 + chunks - 1u) / chunks > kNormThreads) chunks <<= 1;
    const uint32_t width = ((n4 + chunks - 1u) / chunks + 31u) & ~31u;
    if (width > kNormThreads) return cudaErrorNotSupported;   // rows beyond 65536 elements
#define PDK_NORM_CASE(C)                                                                                                          \
    case C:                                                                                                                       \
        return pdk_launch_pdl(add_rmsnorm_quant_blk_kernel<C>, dim3(batch), dim3(width), 0, (cudaStream_t)stream, (float*)x, (const float*)proj, \
                              (const float*)w, (float*)xn, (uint8_t*)q, (float*)scale, n, eps)
    switch (chunks) {
        PDK_NORM_CASE(1);
        PDK_NORM_CASE(2);
        PDK_NORM_CASE(4);
        PDK_NORM_CASE(8);
        PDK_NORM_CASE(16);
    }
#undef PDK_NORM_CASE
    return cudaErrorNotSupported;
}

static bool plane_ok(const void* p0, uintptr_t a0, const void* p1, const void* p2, uintptr_t a2, uint32_t in_dim, uint32_t out_dim) {
    return p0 && p1 && p2 && pdk_aligned(p0, a0) && pdk_aligned(p1, 4) && pdk_aligned(p2, a2) && in_dim <= kMostElems && out_dim <= kMostElems &&
           (uint64_t)f8blk::blocks_of(in_dim) * f8blk::blocks_of(out_dim) <= 0x7fffffffull;
}

// No slot: bf16 weights [out][in] -> block-scaled e4m3.  An ordinary launch: a plane's readers may start ahead of the launch before them.
PDK_EXPORT int pdk_bf16_to_f8blk(const void* bf16, void* data, void* scale, uint32_t in_dim, uint32_t out_dim, void* stream) {
    if (in_dim == 0u || out_dim == 0u) return 0;
    if (!plane_ok(bf16, 2, scale, data, 1, in_dim, out_dim)) return cudaErrorInvalidValue;
    const uint32_t per_row = f8blk::blocks_of(in_dim), tiles = per_row * f8blk::blocks_of(out_dim);
    auto kern = (in_dim & 7u) == 0u && pdk_aligned(bf16, 16) && pdk_aligned(data, 8) ? bf16_to_f8blk_kernel : bf16_to_f8blk_any_kernel;
    kern<<<tiles, kTileThreads, 0, (cudaStream_t)stream>>>((const __nv_bfloat16*)bf16, (uint8_t*)data, (float*)scale, in_dim, out_dim, per_row);
    return pdk_launch_status();
}

// No slot: y f32 [out][in] = code * scale, one f32 rounding
PDK_EXPORT int pdk_f8blk_dequant(const void* data, const void* scale, void* y, uint32_t in_dim, uint32_t out_dim, void* stream) {
    if (in_dim == 0u || out_dim == 0u) return 0;
    if (!plane_ok(data, 1, scale, y, 4, in_dim, out_dim)) return cudaErrorInvalidValue;
    const uint32_t per_row = f8blk::blocks_of(in_dim), tiles = per_row * f8blk::blocks_of(out_dim);
    if ((in_dim & 7u) == 0u && pdk_aligned(data, 8) && pdk_aligned(y, 16))
        return pdk_launch_pdl(f8blk_dequant_kernel, dim3(tiles), dim3(kTileThreads), 0, (cudaStream_t)stream, (const uint8_t*)data, (const float*)scale,
                              (float*)y, in_dim, out_dim, per_row, pdk_aligned(y, 32) ? 1u : 0u);
    return pdk_launch_pdl(f8blk_dequant_any_kernel, dim3(tiles), dim3(kTileThreads), 0, (cudaStream_t)stream, (const uint8_t*)data, (const float*)scale,
                          (float*)y, in_dim, out_dim, per_row);
}
