// f8blk_gemm.cu - products of block-scaled e4m3 operands (f8blk.cuh): entry points.
//
//   y[t][n] = sum_b xs[t][b] * ws[n / 128][b] * ( sum_{k in block b} xq[t][k] * wq[n][k] )
//   h[t][f] = silu(g) * u of two such products, left quantized in blocks of 128 f per token
#include <cstdlib>

#include "f8blk_tc5.cuh"

namespace {

bool operands_ok(const void* w, const void* ws, const void* xq, const void* xs, uint32_t in_dim, uint32_t out_dim, uint32_t batch) {
    constexpr uint32_t kMost = 0x7fffff00u;   // coordinates of a box are signed
    return w && ws && xq && xs && in_dim != 0u && (in_dim & 15u) == 0u && in_dim <= kMost && out_dim <= kMost && batch <= kMost &&
           pdk_aligned(w, 16) && pdk_aligned(xq, 16) && pdk_aligned(ws, 4) && pdk_aligned(xs, 4);
}

// PDK_F8BLK_ROUTE=1 or 2 keeps every call on the split or the wide kernel (A/B switch, read once).
bool prefer_pair(const f8blk::Call& c, int planes) {
    static const int force = [] { const char* e = getenv("PDK_F8BLK_ROUTE"); return e ? atoi(e) : 0; }();
    if (force) return force == 2;
    if (c.batch <= 128u) return false;
    const uint64_t small = (uint64_t)((c.batch + 127u) / 128u) * f8blk::blocks_of(c.out_dim) * planes, slabs = f8blk::blocks_of(c.in_dim);
    return small > 100u && (small - 100u) * slabs > 6000u;
}
int launch(const f8blk::Call& c, int planes, bool bf16, cudaStream_t st) {
    return prefer_pair(c, planes) ? pdk_f8blk_wide(c, planes, bf16, st) : pdk_f8blk_split(c, planes, bf16, st);
}

int gemm(const void* w, const void* ws, const void* xq, const void* xs, void* y, uint32_t in_dim, uint32_t out_dim, uint32_t batch, bool bf16,
         cudaStream_t st) {
    if (out_dim == 0u || batch == 0u) return 0;
    if (!operands_ok(w, ws, xq, xs, in_dim, out_dim, batch) || !y || !pdk_aligned(y, bf16 ? 2 : 4)) return cudaErrorInvalidValue;
    const f8blk::Call c{{w, nullptr}, {ws, nullptr}, xq, xs, y, nullptr, in_dim, out_dim, batch};
    return launch(c, 1, bf16, st);
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
