// f8blk_split.cu - products of block-scaled e4m3 operands at decode widths: a stream of weights.
//
// A tile is 128 channels (tensor-memory lanes, one weight scale per block of K) x BN tokens; a cluster of S CTAs shares it, each with
// every S-th part of K, because one CTA per tile would leave most SMs idle for the planes of a decode step.  Two CTAs share an SM: one
// streams while the other meets its cluster.  A stage is one block of K:
//   warp 0      producer: TMA boxes of the plane (or of gate and up) and of the tokens, 128-byte swizzle
//   warp 1      MMA issuer: four MMAs per plane and stage into one of the tensor-memory buffers, whose sum is one block's
//   warps 2..5  lane = channel: wait for a block's sums, hand the buffer back, and add them on in registers with the scales.  A column's
//               scale is the token's times the plane's; each warp keeps the BN products of a block in a row of shared memory of its own and
//               reads them back as broadcasts.
// The partial products meet through distributed shared memory and are added in rank order: the same bits whatever the timing.  A store
// that may be past the batch is predicated, not branched around (60 tokens through a gated 2880 x 2880 front 14.0 -> 9.8 us with tiles of 32).
// HBM bounds it: 1 token through 5120 x 17408 15.5 us, 5.7 TB/s; its gated front 28 us, 6.3 TB/s; 7 tokens through 17408 x 5003 16.2 us, 5.4 TB/s.  Below
// some MB of weights it is start-up and meeting: 1 token through 5120 x 1024 4.5 us, of which the stream takes 0.8.
// Gated front: gate and up of a channel are in one thread's registers.  They meet by token: the owner of a token has all 128
// channels of a block of h, which one warp sums, gates, scales and writes, 128 codes in one line.
#include "cluster_caps.cuh"
#include "f8blk_tc5.cuh"

namespace {

using namespace f8blk;
using tc5::cluster_addr;
using tc5::cluster_sync;

constexpr uint32_t BM = 128, BK = 128;
constexpr uint32_t kABytes = BM * BK;
constexpr uint32_t kThreads = 192;
constexpr uint32_t kMaxStages = 5, kMaxBufs = 4;
constexpr uint32_t kSmemHalf = 115712;   // what lets two CTAs share an SM: 228 KB / 2 - 1 KB reserved

template <uint32_t BN, int kPlanes>
struct Cfg {
    static constexpr uint32_t kBBytes = BN * BK, kStageBytes = kPlanes * kABytes + kBBytes;
    static constexpr uint32_t kScaleBytes = 4u * 2u * kPlanes * BN * 4u;   // four warps, two rows in turn, the columns' scales per plane
    static constexpr uint32_t kFit = (kSmemHalf - 256u - kScaleBytes) / kStageBytes;
    static constexpr uint32_t kStages = kFit < kMaxStages ? kFit : kMaxStages;
    static constexpr uint32_t kCols = kPlanes * BN;                         // tensor-memory columns of a buffer
    static constexpr uint32_t kBufs = 256u / kCols < kMaxBufs ? 256u / kCols : kMaxBufs;
    static constexpr uint32_t kTmemCols = kBufs * kCols;
    static constexpr uint32_t kIdesc = tc5::idesc_f32acc(0u, 0u, BM, BN);
    static constexpr uint32_t kSmemBytes = kStages * kStageBytes + kScaleBytes + 256u;
    static_assert(kStages >= 2u && kBufs >= 2u && (kTmemCols & (kTmemCols - 1u)) == 0u, "double buffers");
    // the partial products reuse the stages: by channel S x BN tokens x ceil(128 / S) channels rounded up to four, or by token
    // S x ceil(BN / S) tokens x 128 channels of two planes
    static_assert(kPlanes == 2 ? 2u * (BN + kPdkMaxCluster - 1u) * BM * 4u <= kStages * kStageBytes
                               : BN * (BM + 4u * kPdkMaxCluster) * 4u <= kStages * kStageBytes,
                  "partial products fit the stages");
};

struct Shared {
    uint64_t full[kMaxStages];
    uint64_t empty[kMaxStages];
    uint64_t acc_full[kMaxBufs];
    uint64_t acc_empty[kMaxBufs];
    uint32_t tmem_base;
    int abort_flag;
    int gave_up;      // some CTA of the cluster did not come to the end of its blocks
};
static_assert(sizeof(Shared) <= 256u, "control block");

struct Args {
    const float *ws0, *ws1, *xs;
    void* y;
    float* hs;
    uint32_t out_dim, batch, num_kb;
    uint32_t tile_t0, tile_w0;   // the launch's first token and channel tile
    uint32_t vec_store;          // y rows take 4-channel vector stores
    unsigned int* err;
};

// A store that may be past the batch: predicated, not branched around (a branch per store costs about 50 cycles each).
__device__ __forceinline__ void store_if(float* p, float v, bool on) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q st.global.f32 [%0], %1;\n\t}" ::"l"(p), "f"(v), "r"((uint32_t)on) : "memory");
}
__device__ __forceinline__ void store_if(__nv_bfloat16* p, float v, bool on) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q st.global.b16 [%0], %1;\n\t}" ::"l"(p),
                 "h"(__bfloat16_as_ushort(__float2bfloat16_rn(v))), "r"((uint32_t)on)
                 : "memory");
}
__device__ __forceinline__ void st_cluster_if(uint32_t addr, float v, bool on) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q st.shared::cluster.f32 [%0], %1;\n\t}" ::"r"(addr), "f"(v), "r"((uint32_t)on) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void store4(float* p, const float4& v) { __stcs(reinterpret_cast<float4*>(p), v); }
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float4& v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b)));
}

template <uint32_t BN, int kPlanes, typename TO>
__global__ void __launch_bounds__(kThreads, 2)
f8blk_split_kernel(const __grid_constant__ CUtensorMap tmap_w0, const __grid_constant__ CUtensorMap tmap_w1,
                   const __grid_constant__ CUtensorMap tmap_x, const Args a) {
    using C = Cfg<BN, kPlanes>;
    extern __shared__ __align__(1024) uint8_t smem[];
    float* scale_rows = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes);
    Shared* sh = reinterpret_cast<Shared*>(smem + C::kStages * C::kStageBytes + C::kScaleBytes);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t split = gridDim.x, rank = blockIdx.x;   // the cluster spans x
    const uint32_t tw = a.tile_w0 + blockIdx.z, t0 = (a.tile_t0 + blockIdx.y) * BN, n0 = tw * BM, n_tok = min(BN, a.batch - t0);
    const uint32_t kb_lo = rank * a.num_kb / split, kb_hi = (rank + 1u) * a.num_kb / split;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < C::kStages; ++s) {
            tc5::mbar_init(&sh->full[s], 1);
            tc5::mbar_init(&sh->empty[s], 1);
        }
        for (uint32_t b = 0; b < C::kBufs; ++b) {
            tc5::mbar_init(&sh->acc_full[b], 1);
            tc5::mbar_init(&sh->acc_empty[b], 4);
        }
        sh->abort_flag = 0;
        sh->gave_up = 0;
        tc5::mbar_fence_init();
        tc5::tma_prefetch_desc(&tmap_w0);
        if (kPlanes == 2) tc5::tma_prefetch_desc(&tmap_w1);
        tc5::tma_prefetch_desc(&tmap_x);
    }
    if (warp == 1) {
        tc5::tmem_alloc(&sh->tmem_base, C::kTmemCols);
        tc5::tmem_relinquish();
    }
    tc5::fence_before_sync();
    __syncthreads();
    tc5::fence_after_sync();
    const uint32_t tmem_base = sh->tmem_base;
    const tc5::WaitCtx ctx{&sh->abort_flag, a.err};
    pdk_pdl_launch_dependents();

    float acc[kPlanes][BN];
    bool ok = true;
    if (warp == 0) {
        // ------------------------------------------------------------ producer (whole warp, one lane issues)
        const uint64_t stream_once = tc5::l2_policy_evict_first();
        const bool reused = gridDim.y > 1u;    // several token tiles read the same weights: keep them in L2
        auto issue_w = [&](uint32_t stage, uint32_t kb) {
            uint8_t* s = smem + stage * C::kStageBytes;
            tc5::mbar_arrive_expect_tx_elect(&sh->full[stage], C::kStageBytes);
#pragma unroll
            for (int p = 0; p < kPlanes; ++p) {
                const CUtensorMap* m = p == 0 ? &tmap_w0 : &tmap_w1;
                if (reused) tc5::tma_load_2d_elect(s + p * kABytes, m, &sh->full[stage], (int32_t)(kb * BK), (int32_t)n0);
                else tc5::tma_load_2d_hint_elect(s + p * kABytes, m, &sh->full[stage], (int32_t)(kb * BK), (int32_t)n0, stream_once);
            }
        };
        // weights depend on nothing the previous kernel in the stream writes: the first stages go out before the wait for it
        const uint32_t pre = min(kb_hi - kb_lo, C::kStages);
        for (uint32_t i = 0; i < pre; ++i) issue_w(i, kb_lo + i);
        pdk_pdl_wait();
        uint32_t stage = 0, phase = 0;
        for (uint32_t kb = kb_lo; kb < kb_hi; ++kb) {
            if (kb - kb_lo >= pre) {
                ok = __all_sync(0xffffffffu, wait_soon(&sh->empty[stage], phase ^ 1u, ctx, tc5::kErrEmptyWait, stage));
                if (!ok) break;
                issue_w(stage, kb);
            }
            tc5::tma_load_2d_elect(smem + stage * C::kStageBytes + kPlanes * kABytes, &tmap_x, &sh->full[stage], (int32_t)(kb * BK), (int32_t)t0);
            if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (whole warp, one lane issues)
        uint32_t stage = 0, phase = 0, buf = 0, bphase = 0;
        pdk_pdl_wait();   // the tokens come behind it: a limit that started earlier would count the launch in front
        for (uint32_t kb = kb_lo; kb < kb_hi; ++kb) {
            ok = __all_sync(0xffffffffu, wait_soon(&sh->acc_empty[buf], bphase ^ 1u, ctx, tc5::kErrTmemEmptyWait, buf) &&
                                             wait_soon(&sh->full[stage], phase, ctx, tc5::kErrFullWait, stage));
            if (!ok) break;
            tc5::fence_after_sync();
            const uint32_t s_addr = tc5::smem_u32(smem + stage * C::kStageBytes);
            const uint64_t b_desc = tc5::smem_desc_sw128(s_addr + kPlanes * kABytes);
#pragma unroll
            for (int p = 0; p < kPlanes; ++p)
                tc5::mma_f8f6f4_x4_elect(tmem_base + buf * C::kCols + p * BN, tc5::smem_desc_sw128(s_addr + p * kABytes), b_desc, C::kIdesc, 0u);
            tc5::mma_commit_elect(&sh->empty[stage]);
            tc5::mma_commit_elect(&sh->acc_full[buf]);
            if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
            if (++buf == C::kBufs) { buf = 0; bphase ^= 1u; }
        }
    } else {
        // ------------------------------------------------------------ a block's sums, scaled, onto the product
        pdk_pdl_wait();   // scales and y may still be in use by the previous kernel
        float* row = scale_rows + (warp - 2u) * (2u * kPlanes * BN);
        const float* xs[BN / 32u];
#pragma unroll
        for (uint32_t c = 0; c < BN / 32u; ++c) xs[c] = a.xs + (size_t)min(t0 + c * 32u + lane, a.batch - 1u) * a.num_kb;
        const float *ws0 = a.ws0 + (size_t)tw * a.num_kb, *ws1 = kPlanes == 2 ? a.ws1 + (size_t)tw * a.num_kb : nullptr;
#pragma unroll
        for (int p = 0; p < kPlanes; ++p)
#pragma unroll
            for (uint32_t i = 0; i < BN; ++i) acc[p][i] = 0.0f;
        float next_x[BN / 32u], next_w[2] = {0.0f, 0.0f};
        auto fetch = [&](uint32_t kb) {
#pragma unroll
            for (uint32_t c = 0; c < BN / 32u; ++c) next_x[c] = xs[c][kb];
            next_w[0] = ws0[kb];
            if (kPlanes == 2) next_w[1] = ws1[kb];
        };
        fetch(kb_lo);
        const uint32_t lanes = tmem_base + (((warp & 3u) * 32u) << 16);
        uint32_t buf = 0, bphase = 0;
        for (uint32_t kb = kb_lo; kb < kb_hi; ++kb) {
            float* turn = row + ((kb - kb_lo) & 1u) * (kPlanes * BN);   // two rows in turn: a lane may still read the last block's
#pragma unroll
            for (uint32_t c = 0; c < BN / 32u; ++c) {
                turn[c * 32u + lane] = next_x[c] * next_w[0];
                if (kPlanes == 2) turn[BN + c * 32u + lane] = next_x[c] * next_w[1];
            }
            if (kb + 1u < kb_hi) fetch(kb + 1u);
            __syncwarp();
            ok = __all_sync(0xffffffffu, wait_soon(&sh->acc_full[buf], bphase, ctx, tc5::kErrTmemFullWait, buf));
            if (!ok) break;
            tc5::fence_after_sync();
            // two loads of 32 columns on their way, where a product of 128 columns leaves registers for that; plane p's columns are p * BN .. + BN - 1
            constexpr uint32_t kLoads = C::kCols / 32u, kAtOnce = C::kCols <= 64u ? 2u : 1u;
            uint32_t r[kAtOnce][32];
            const uint32_t from = lanes + buf * C::kCols;
            auto add = [&](uint32_t l) {
                const float4* s = reinterpret_cast<const float4*>(turn + l * 32u);
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) {
                    const float4 s4 = s[i];
                    float* to = acc[l * 32u / BN] + l * 32u % BN + 4u * i;
                    const uint32_t(&v)[32] = r[l % kAtOnce];
                    to[0] = fmaf(__uint_as_float(v[4u * i]), s4.x, to[0]);
                    to[1] = fmaf(__uint_as_float(v[4u * i + 1u]), s4.y, to[1]);
                    to[2] = fmaf(__uint_as_float(v[4u * i + 2u]), s4.z, to[2]);
                    to[3] = fmaf(__uint_as_float(v[4u * i + 3u]), s4.w, to[3]);
                }
            };
#pragma unroll
            for (uint32_t l = 0; l < kLoads; l += kAtOnce) {
#pragma unroll
                for (uint32_t i = 0; i < kAtOnce && l + i < kLoads; ++i) tc5::tmem_ld_32x32(from + (l + i) * 32u, r[i]);
#pragma unroll
                for (uint32_t i = 0; i < kAtOnce && l + i < kLoads; ++i) tmem_ld_wait(r[i]);
                if (l + kAtOnce >= kLoads) {   // the last columns are in registers: the buffer goes back
                    tc5::fence_before_sync();
                    __syncwarp();
                    if (lane == 0u) tc5::mbar_arrive(&sh->acc_empty[buf]);
                }
#pragma unroll
                for (uint32_t i = 0; i < kAtOnce && l + i < kLoads; ++i) add(l + i);
            }
            if (++buf == C::kBufs) { buf = 0; bphase ^= 1u; }
        }
    }
    tc5::fence_before_sync();
    __syncthreads();
    const bool gave_up = sh->abort_flag != 0;
    if (gave_up) wait_for_copies();
    // every CTA's stages are consumed from here on: they take the partial products
    if (split > 1u) cluster_sync();
    tc5::fence_after_sync();
    if (warp == 1) tc5::tmem_dealloc(tmem_base, C::kTmemCols);   // the last sums are in registers
    // Where a wait ran out blocks of K are missing: with the partial products every CTA of the cluster hears of it, and none stores a result.
    if (gave_up && threadIdx.x < split) st_cluster_u32(cluster_addr(tc5::smem_u32(&sh->gave_up), threadIdx.x), 1u);

    const uint32_t ch = (warp & 3u) * 32u + lane;
    TO* y = reinterpret_cast<TO*>(a.y);
    if (kPlanes == 1 && split == 1u) {
        if (warp >= 2u && !gave_up) {   // the tile is whole: 32 neighbouring channels per store
            const bool live = n0 + ch < a.out_dim;
            TO* out = y + (size_t)t0 * a.out_dim + n0 + ch;
#pragma unroll
            for (uint32_t i = 0; i < BN; ++i) {
                store_if(out, acc[0][i], live && i < n_tok);
                out += a.out_dim;
            }
        }
        return;
    }

    const uint32_t red = tc5::smem_u32(smem);
    if constexpr (kPlanes == 1) {
        // Rank r adds up and stores channels [r * cpr, (r + 1) * cpr): each CTA leaves its part in the owner's buffer
        // [rank][token][cpr channels].  A lane is a channel, so its owner and address are fixed.
        const uint32_t cpr = ((BM + split - 1u) / split + 3u) & ~3u;
        if (warp >= 2u) {
            const uint32_t dst = cluster_addr(red, ch / cpr) + (rank * n_tok * cpr + ch % cpr) * 4u;
#pragma unroll
            for (uint32_t i = 0; i < BN; ++i)
                st_cluster_if(dst + i * cpr * 4u, acc[0][i], i < n_tok);
        }
        cluster_sync();
        if (sh->gave_up) return;
        const uint32_t ch_lo = rank * cpr, groups = ch_lo < BM ? min(cpr, BM - ch_lo) / 4u : 0u;   // of four channels
        for (uint32_t i = threadIdx.x; i < groups * n_tok; i += kThreads) {
            const uint32_t tok = i / groups, g = (i - tok * groups) * 4u, n = n0 + ch_lo + g;
            if (n >= a.out_dim) continue;
            const float* part = reinterpret_cast<const float*>(smem) + tok * cpr + g;
            float4 sum = *reinterpret_cast<const float4*>(part);
            for (uint32_t s = 1; s < split; ++s) {
                const float4 p = *reinterpret_cast<const float4*>(part + s * n_tok * cpr);
                sum.x += p.x; sum.y += p.y; sum.z += p.z; sum.w += p.w;
            }
            TO* out = y + (size_t)(t0 + tok) * a.out_dim + n;
            if (a.vec_store) {          // out_dim % 4 == 0: the four channels are all there
                store4(out, sum);
            } else {
                store_if(out, sum.x, true);
                store_if(out + 1, sum.y, n + 1u < a.out_dim);
                store_if(out + 2, sum.z, n + 2u < a.out_dim);
                store_if(out + 3, sum.w, n + 3u < a.out_dim);
            }
        }
    } else {
        // Rank r owns tokens [r * tpr, (r + 1) * tpr): buffer [rank][plane][its tokens][128 channels].
        const uint32_t tpr = (n_tok + split - 1u) / split;
        if (warp >= 2u) {
            const uint32_t own = (rank * 2u * tpr * BM + ch) * 4u;
            uint32_t owner = 0u, tok = 0u;
#pragma unroll
            for (uint32_t i = 0; i < BN; ++i) {      // no branches: one per token costs more than the stores
                const uint32_t dst = cluster_addr(red, min(owner, split - 1u)) + own + tok * BM * 4u;
                st_cluster_if(dst, acc[0][i], i < n_tok);
                st_cluster_if(dst + tpr * BM * 4u, acc[kPlanes - 1][i], i < n_tok);
                const bool next = ++tok == tpr;
                owner += next ? 1u : 0u;
                tok = next ? 0u : tok;
            }
        }
        if (split > 1u) cluster_sync();
        else __syncthreads();
        if (sh->gave_up) return;
        const uint32_t tok_lo = rank * tpr, toks = tok_lo < n_tok ? min(tpr, n_tok - tok_lo) : 0u;
        const uint32_t n = n0 + lane * 4u, blocks = (a.out_dim + BM - 1u) / BM;
        for (uint32_t tok = warp; tok < toks; tok += kThreads / 32u) {
            float4 g = make_float4(0.0f, 0.0f, 0.0f, 0.0f), u = g;
            for (uint32_t s = 0; s < split; ++s) {
                const float4* part = reinterpret_cast<const float4*>(smem) + ((s * 2u * tpr + tok) * BM) / 4u + lane;
                const float4 pg = part[0], pu = part[tpr * BM / 4u];
                g.x += pg.x; g.y += pg.y; g.z += pg.z; g.w += pg.w;
                u.x += pu.x; u.y += pu.y; u.z += pu.z; u.w += pu.w;
            }
            const float4 h = make_float4(gated(g.x, u.x), gated(g.y, u.y), gated(g.z, u.z), gated(g.w, u.w));
            float m = fmaxf(fmaxf(fabsf(h.x), fabsf(h.y)), fmaxf(fabsf(h.z), fabsf(h.w)));
#pragma unroll
            for (uint32_t d = 1; d < 32u; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            const float sc = scale_of(m);
            const size_t t = t0 + tok_lo + tok;
            if (n < a.out_dim)    // ff % 16 == 0: the four channels are all there
                *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(a.y) + t * a.out_dim + n) = codes4(h.x, h.y, h.z, h.w, 1.0f / sc);
            if (lane == 0u) a.hs[t * blocks + tw] = sc;
        }
    }
}

template <uint32_t BN, int kPlanes, typename TO>
int clusters(const uint32_t** resident) {
    static PdkClusterCaps table;
    return pdk_cluster_caps(table, (const void*)f8blk_split_kernel<BN, kPlanes, TO>, kThreads, Cfg<BN, kPlanes>::kSmemBytes, resident);
}

template <uint32_t BN, int kPlanes, typename TO>
int launch_bn(const Call& c, uint32_t split, cudaStream_t st) {
    using C = Cfg<BN, kPlanes>;
    auto kern = f8blk_split_kernel<BN, kPlanes, TO>;
    const uint32_t* resident = nullptr;
    if (int rc = clusters<BN, kPlanes, TO>(&resident)) return rc;      // raises the kernel's shared memory limit on this device
    Args a{};
    a.ws0 = (const float*)c.ws[0]; a.ws1 = (const float*)c.ws[1]; a.xs = (const float*)c.xs; a.y = c.y; a.hs = (float*)c.hs;
    a.out_dim = c.out_dim; a.batch = c.batch; a.num_kb = blocks_of(c.in_dim);
    a.vec_store = (c.out_dim & 3u) == 0u && pdk_aligned(c.y, 4u * sizeof(TO)) ? 1u : 0u;
    a.err = pdk_error_word();
    const uint32_t tiles_t = c.batch / BN + (c.batch % BN != 0u), tiles_w = blocks_of(c.out_dim);

    CUtensorMap tw0, tw1, tx;
    if (int rc = pdk_make_tmap_2d(&tw0, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.w[0], c.in_dim, c.out_dim, c.in_dim, BK, BM)) return rc;
    tw1 = tw0;
    if (kPlanes == 2)
        if (int rc = pdk_make_tmap_2d(&tw1, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.w[1], c.in_dim, c.out_dim, c.in_dim, BK, BM)) return rc;
    if (int rc = pdk_make_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.xq, c.in_dim, c.batch, c.in_dim, BK, BN)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdk_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    constexpr uint32_t kAxis = 65535u;   // one launch, unless a grid axis cannot hold the tiles
    for (a.tile_w0 = 0u; a.tile_w0 < tiles_w; a.tile_w0 += kAxis)
        for (a.tile_t0 = 0u; a.tile_t0 < tiles_t; a.tile_t0 += kAxis) {
            const uint32_t nt = tiles_t - a.tile_t0, nw = tiles_w - a.tile_w0;
            cfg.gridDim = dim3(split, nt < kAxis ? nt : kAxis, nw < kAxis ? nw : kAxis);
            if (cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tw0, tw1, tx, a); e != cudaSuccess) return (int)e;
        }
    return pdk_launch_status();
}

template <uint32_t BN>
int launch_kind(const Call& c, int planes, bool bf16, uint32_t split, cudaStream_t st) {
    if (planes == 2) return launch_bn<BN, 2, float>(c, split, st);
    return bf16 ? launch_bn<BN, 1, __nv_bfloat16>(c, split, st) : launch_bn<BN, 1, float>(c, split, st);
}

}  // namespace

// resident[c]: how many clusters of s CTAs are resident at once with 32 << c tokens a tile.  0 or a cudaError_t.
int pdk_f8blk_split_clusters(int planes, const uint32_t* resident[2]) {
    if (int rc = planes == 2 ? clusters<32, 2, float>(&resident[0]) : clusters<32, 1, float>(&resident[0])) return rc;
    return planes == 2 ? clusters<64, 2, float>(&resident[1]) : clusters<64, 1, float>(&resident[1]);
}

int pdk_f8blk_split(const Call& c, int planes, bool bf16, uint32_t cols, uint32_t split, cudaStream_t st) {
    return cols == 32u ? launch_kind<32>(c, planes, bf16, split, st) : launch_kind<64>(c, planes, bf16, split, st);
}
