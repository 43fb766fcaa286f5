// f8blk_wide.cu - products of block-scaled e4m3 operands at prompt widths.
//
// Persistent CTAs, one per SM, tiles of 128 tokens x 256 channels (tcgen05, M = 128 x N = 256 x K = 32 per instruction).  Tokens are
// the lanes, so a thread owns one token, and a block's two scales are one number per thread: the block's sums come out of tensor
// memory and go onto the product with one fused multiply-add each.
//
//   warp 0      producer: a block of K of the tokens (16 KB) and of the channels (32 KB) per stage
//   warp 1      MMA issuer: four MMAs per block into one of two buffers of 256 tensor-memory columns
//   warps 2, 3  the scales: of the tokens, times those of the two halves of the channels, into shared memory.  They arrive on the stage's
//               barrier like the boxes, so whoever has a block's sums has its scales, without a wait of its own: the issuer, which has waited
//               for that barrier, arrives on the sums' one beside the tensor core, and its release hands the scales' stores on
//   warps 4..11 the product: warp w has tokens 32 (w % 4) .. + 31 and 128 of the 256 columns, 128 registers a thread, and 64 more for columns on
//               their way; the first four warps hand registers over for that
//
// Gated front: the first 128 channels of a tile are gate's, the others up's beside them.  A warp's columns are then 64 of gate's and the
// same 64 of up's, so a thread gates its own sums; only the maximum of a token's block crosses to the other half's warp.
//
// Tiles of 128 channels, four buffers of 128 columns and half the columns a warp, where tiles of 256 would leave SMs without one: 200 tokens
// through 5120 x 5120 15.2 us instead of 22.2.
//
// What bounds it (cycles per block of a 256-channel tile, 512 tokens through 17408 x 9472, one tile per SM): the tensor core needs 514, loads from
// tensor memory and additions by themselves 357, both with their hand-over 630 with operands in place, the boxes from L2 (48 KB) 730
// without the additions; all together 851.  4096 tokens through 5120 x 17408: 350 us in short runs (2.1 PFLOP/s), about 400 in long ones, where
// the power limit takes the clock to 1.4 GHz.  Measured on the way there:
//   scales read from global memory by the eight warps, 32 sectors a load              +330 cycles
//   brought by warps 2 and 3, but under barriers of their own                         +170
//   packed multiply-adds (fma.rn.f32x2): their pairs are moved together first         +200
//   a block's loads started in front of the last block's additions                    +100
//   pairs of SMs (cta_group::2, two thirds of the L2 traffic)                         +140 to +250: every block crosses between the SMs twice
// Every wait is bounded; a role that gives up goes on through the loop without waiting or touching memory, so that the named
// barriers of the others meet.
#include "f8blk_tc5.cuh"

namespace {

using namespace f8blk;

constexpr uint32_t BM = 128, BK = 128;                        // tokens of a tile, K per stage
constexpr uint32_t kABytes = BM * BK;
constexpr uint32_t kWarps = 8, kFirst = 4;                    // that keep the product, and the first of them
constexpr uint32_t kThreads = (kFirst + kWarps) * 32u;
// registers a thread: 168 at launch (64,512 in all), 56 for the first four warps and 224 for the others after the split (64,512)
constexpr uint32_t kRegsFew = 56, kRegsMany = 224;
static_assert(kFirst * 32u * kRegsFew + kWarps * 32u * kRegsMany <= kThreads * 168u, "the split draws on what the launch has");
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kAhead = 2;                                // blocks whose scales a lane loads together
constexpr uint32_t kSlots = 16;

// BN columns of a tile: 256, or 128 where tiles of 256 would leave SMs without one
template <uint32_t BN>
struct Cfg {
    static constexpr uint32_t kParts = BN / 128u;             // boxes of 128 channels, each with weight scales of its own
    static constexpr uint32_t kStageBytes = kABytes + kParts * 128u * BK;
    static constexpr uint32_t kStages = BN == 256u ? 4u : 6u;
    static constexpr uint32_t kBufs = kTmemCols / BN;
    static constexpr uint32_t kCols = BN / 2u;                // of a warp
    // Warps that issue MMAs, alternate blocks each.  A block costs its issuer about 600 cycles of waits and issue: too many for 128 columns.
    // With two buffers a second issuer's MMAs would only mix with the first's and finish both blocks late (359 us instead of 343).
    static constexpr uint32_t kIssuers = BN == 256u ? 1u : 2u, kScalers = 3u - kIssuers, kRows = 4u / kScalers;   // and tokens a lane of the others
    // scales are written when a stage is free and read when its sums are: at most the stages and the buffers lie between
    static_assert(kStages + kBufs <= kSlots, "a slot is written again after it was read");
    // a stage is summed again only after this buffer was handed back kBufs blocks later: the phase that is waited for cannot be missed
    static_assert(kStages >= kBufs && kStages % kIssuers == 0u && kBufs % kIssuers == 0u, "an issuer keeps its own stages and buffers");
};
constexpr uint32_t kMaxStages = 6, kMaxBufs = 4;

template <uint32_t kParts>
struct Shared {
    uint64_t full[kMaxStages];         // boxes and scales are there
    uint64_t done[kMaxStages];         // the block is summed: its stage is free, its buffer full
    uint64_t acc_empty[kMaxBufs];
    uint32_t tmem_base;
    int abort_flag;
    float amax[2][BM];
    float scale[kSlots][kParts][BM];   // block % kSlots: the products of the scales, per 128 channels and token
};

struct Args {
    const float *ws0, *ws1, *xs;
    void* y;
    float* hs;
    uint32_t out_dim, batch, num_kb;
    uint32_t row_align;              // bytes, 32, 16 or less, that every row of y starts on
    unsigned int* err;
};

__device__ __forceinline__ void store32(void* p, const uint4& a, const uint4& b) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y),
                 "r"(b.z), "r"(b.w)
                 : "memory");
}
// 16 bytes of a row: 4 f32 or 8 bf16
__device__ __forceinline__ uint4 piece(const float* v, float*) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ uint4 piece(const float* v, __nv_bfloat16*) {
    return make_uint4(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]), bf16x2(v[4], v[5]), bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// a thread's N channels of its token's row, `left` of which the row has
template <uint32_t N, typename TO>
__device__ __forceinline__ void store_row(TO* out, const float (&v)[N], uint32_t left, uint32_t align) {
    constexpr uint32_t kPer = 16u / sizeof(TO);
    if (align >= 16u) {       // rows end on a piece too
        const bool wide = align >= 32u;
#pragma unroll
        for (uint32_t i = 0; i < N; i += 2u * kPer) {
            const uint4 a = piece(v + i, out), b = piece(v + i + kPer, out);
            if (wide) {
                if (i < left) store32(out + i, a, b);
            } else {
                if (i < left) *reinterpret_cast<uint4*>(out + i) = a;
                if (i + kPer < left) *reinterpret_cast<uint4*>(out + i + kPer) = b;
            }
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i)
            if (i < left) put(out + i, v[i]);
    }
}

// Where tile number `tile` lies: token tiles fastest, so that a round of CTAs shares few of the weights and all of the tokens' rows in L2.  From
// 49 token tiles on those are too many, and 32 at a time are gone through instead: 8192 tokens 8192 x 8192 544 -> 505 us, 5120 x 8192 340 -> 333.
// (Groups of 16, or weights fastest, are slower below that: 4096 tokens 5120 x 17408 354 and 425 us instead of 349.  The gated front gains
// nothing from groups: 8192 tokens 5120 x 4096 340 us, without 336.)
template <int kPlanes>
__device__ __forceinline__ uint2 place(uint32_t tile, uint32_t tiles_m, uint32_t tiles_n) {
    if (kPlanes == 2) return make_uint2(tile % tiles_m, tile / tiles_m);
    const uint32_t group = tiles_m > 48u ? 32u : tiles_m, g = tile / (group * tiles_n), in = tile - g * group * tiles_n;
    const uint32_t here = min(group, tiles_m - g * group);
    return make_uint2(g * group + in % here, in / here);
}

template <int kPlanes, uint32_t BN, typename TO>
__global__ void __launch_bounds__(kThreads, 1)
f8blk_wide_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w0,
                  const __grid_constant__ CUtensorMap tmap_w1, const Args a) {
    using C = Cfg<BN>;
    constexpr uint32_t kStages = C::kStages, kStageBytes = C::kStageBytes, kBufs = C::kBufs, kParts = C::kParts;
    static_assert(kPlanes == 1 || BN == 256u, "a block of h has its 128 channels of gate and up in one tile");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~(uintptr_t)1023u);
    Shared<kParts>* sh = reinterpret_cast<Shared<kParts>*>(tiles + kStages * kStageBytes);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    constexpr uint32_t kTileN = kPlanes == 2 ? 128u : BN;      // channels of y (of h) per tile
    const uint32_t tiles_m = (a.batch + BM - 1u) / BM, tiles_n = (a.out_dim + kTileN - 1u) / kTileN;
    const uint32_t n_tiles = tiles_m * tiles_n, w_blocks = (a.out_dim + 127u) / 128u;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            tc5::mbar_init(&sh->full[s], 1u + C::kScalers);     // the expected-bytes arrival, the scales
            tc5::mbar_init(&sh->done[s], 2);                    // the tensor core's arrival, the issuer's
        }
        for (uint32_t b = 0; b < kBufs; ++b) tc5::mbar_init(&sh->acc_empty[b], kWarps);
        sh->abort_flag = 0;
        tc5::mbar_fence_init();
        tc5::tma_prefetch_desc(&tmap_x);
        tc5::tma_prefetch_desc(&tmap_w0);
        if (kPlanes == 2) tc5::tma_prefetch_desc(&tmap_w1);
    }
    if (warp == 1u) {
        tc5::tmem_alloc(&sh->tmem_base, kTmemCols);
        tc5::tmem_relinquish();
    }
    tc5::fence_before_sync();
    __syncthreads();
    tc5::fence_after_sync();
    const uint32_t tmem_base = sh->tmem_base;
    const tc5::WaitCtx ctx{&sh->abort_flag, a.err};
    pdk_pdl_launch_dependents();

    if (warp < kFirst) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
        bool ok = true;
        if (warp == 0u) {
            // -------------------------------------------------------- TMA producer (whole warp, one lane issues)
            uint32_t stage = 0, phase = 0;
            pdk_pdl_wait();
            for (uint32_t tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
                const uint2 at = place<kPlanes>(tile, tiles_m, tiles_n);
                const uint32_t m0 = at.x * BM, n0 = at.y * kTileN;
                for (uint32_t kb = 0; kb < a.num_kb; ++kb) {
                    ok = __all_sync(0xffffffffu, wait_soon(&sh->done[stage], phase ^ 1u, ctx, tc5::kErrEmptyWait, stage));
                    if (!ok) break;
                    uint8_t* s = tiles + stage * kStageBytes;
                    tc5::mbar_arrive_expect_tx_elect(&sh->full[stage], kStageBytes);
                    tc5::tma_load_2d_elect(s, &tmap_x, &sh->full[stage], (int32_t)(kb * BK), (int32_t)m0);
                    tc5::tma_load_2d_elect(s + kABytes, &tmap_w0, &sh->full[stage], (int32_t)(kb * BK), (int32_t)n0);
                    if (kParts == 2u)
                        tc5::tma_load_2d_elect(s + kABytes + 128u * BK, kPlanes == 2 ? &tmap_w1 : &tmap_w0, &sh->full[stage], (int32_t)(kb * BK),
                                               (int32_t)(kPlanes == 2 ? n0 : n0 + 128u));
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
        } else if (warp <= C::kIssuers) {
            // -------------------------------------------------------- MMA issuers (whole warp, one lane issues)
            constexpr uint32_t idesc = tc5::idesc_f32acc(0u, 0u, BM, BN);
            const uint32_t mine = warp - 1u, blocks = ((n_tiles - 1u - blockIdx.x) / gridDim.x + 1u) * a.num_kb;
            uint32_t stage = mine, phase = 0, buf = mine, bphase = 0;
            pdk_pdl_wait();   // the boxes come behind it: a limit that started earlier would count the launch in front
            for (uint32_t block = mine; block < blocks && ok; block += C::kIssuers) {
                const bool empty = wait_soon(&sh->acc_empty[buf], bphase ^ 1u, ctx, tc5::kErrTmemEmptyWait, buf);
                ok = __all_sync(0xffffffffu, wait_soon(&sh->full[stage], phase, ctx, tc5::kErrFullWait, stage) && empty);
                if (!ok) break;
                tc5::fence_after_sync();
                const uint32_t a_addr = tc5::smem_u32(tiles + stage * kStageBytes);
                tc5::mma_f8f6f4_x4_elect(tmem_base + buf * BN, tc5::smem_desc_sw128(a_addr), tc5::smem_desc_sw128(a_addr + kABytes), idesc, 0u);
                tc5::mma_commit_elect(&sh->done[stage]);
                mbar_arrive_elect(&sh->done[stage]);
                if ((stage += C::kIssuers) >= kStages) { stage = mine; phase ^= 1u; }
                if ((buf += C::kIssuers) >= kBufs) { buf = mine; bphase ^= 1u; }
            }
        } else {
            // -------------------------------------------------------- scales
            constexpr uint32_t kRows = C::kRows;
            const uint32_t row0 = (warp - 1u - C::kIssuers) * 32u * kRows + lane;
            uint32_t stage = 0, phase = 0, block = 0;
            pdk_pdl_wait();
            for (uint32_t tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
                const uint2 at = place<kPlanes>(tile, tiles_m, tiles_n);
                const uint32_t t = at.x * BM + row0, nb = at.y * kTileN / 128u;
                const float* x[kRows];
#pragma unroll
                for (uint32_t i = 0; i < kRows; ++i) x[i] = a.xs + (size_t)min(t + 32u * i, a.batch - 1u) * a.num_kb;
                const float* w0 = a.ws0 + (size_t)nb * a.num_kb;
                const float* w1 = kPlanes == 2 ? a.ws1 + (size_t)nb * a.num_kb : a.ws0 + (size_t)min(nb + kParts - 1u, w_blocks - 1u) * a.num_kb;
                float nx[kRows][kAhead], nw[kParts][kAhead];      // the next blocks', on their way while the last ones are handed on
                auto fetch = [&](uint32_t k0) {
#pragma unroll
                    for (uint32_t j = 0; j < kAhead; ++j) {
                        const uint32_t kb = min(k0 + j, a.num_kb - 1u);
#pragma unroll
                        for (uint32_t i = 0; i < kRows; ++i) nx[i][j] = x[i][kb];
                        nw[0][j] = w0[kb];
                        if (kParts == 2u) nw[kParts - 1u][j] = w1[kb];
                    }
                };
                fetch(0u);
                for (uint32_t k0 = 0; k0 < a.num_kb && ok; k0 += kAhead) {
                    float cx[kRows][kAhead], cw[kParts][kAhead];
#pragma unroll
                    for (uint32_t j = 0; j < kAhead; ++j) {
#pragma unroll
                        for (uint32_t i = 0; i < kRows; ++i) cx[i][j] = nx[i][j];
#pragma unroll
                        for (uint32_t h = 0; h < kParts; ++h) cw[h][j] = nw[h][j];
                    }
                    fetch(k0 + kAhead);
#pragma unroll
                    for (uint32_t j = 0; j < kAhead; ++j) {
                        if (k0 + j >= a.num_kb || !ok) break;
                        ok = __all_sync(0xffffffffu, wait_soon(&sh->done[stage], phase ^ 1u, ctx, tc5::kErrEmptyWait, 16u + stage));
                        if (!ok) break;
                        float(&slot)[kParts][BM] = sh->scale[block++ % kSlots];
#pragma unroll
                        for (uint32_t h = 0; h < kParts; ++h)
#pragma unroll
                            for (uint32_t i = 0; i < kRows; ++i) slot[h][row0 + 32u * i] = cx[i][j] * cw[h][j];
                        __syncwarp();
                        if (lane == 0u) tc5::mbar_arrive(&sh->full[stage]);
                        if (++stage == kStages) { stage = 0; phase ^= 1u; }
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMany));
        // ------------------------------------------------------------ the product
        const uint32_t quarter = warp & 3u, half = (warp - kFirst) >> 2;
        const uint32_t row = quarter * 32u + lane;           // token of the tile
        // columns: half of the tile's in a row, or 64 of gate's and the same of up's
        constexpr uint32_t kCols = C::kCols, kSecond = kPlanes == 2 ? 128u : 64u;    // and where the second 64 start
        const uint32_t lanes = tmem_base + ((quarter * 32u) << 16) + half * (kPlanes == 2 ? 64u : kCols);
        uint32_t block = 0;
        bool ok = true;
        pdk_pdl_wait();
        for (uint32_t tile = blockIdx.x; tile < n_tiles; tile += gridDim.x) {
            float acc[kCols];
#pragma unroll
            for (uint32_t i = 0; i < kCols; ++i) acc[i] = 0.0f;
            for (uint32_t kb = 0; kb < a.num_kb && ok; ++kb, ++block) {
                const uint32_t buf = block % kBufs, stage = block % kStages;
                ok = __all_sync(0xffffffffu, wait_soon(&sh->done[stage], block / kStages & 1u, ctx, tc5::kErrTmemFullWait, stage));
                if (!ok) break;
                tc5::fence_after_sync();
                const float(&slot)[kParts][BM] = sh->scale[block % kSlots];
                const float s0 = slot[kPlanes == 2 || kParts == 1u ? 0u : half][row], s1 = kPlanes == 2 ? slot[kParts - 1u][row] : s0;
                // two loads on their way at a time; a second pair follows the first into its registers
                uint32_t r[2][32];
                const uint32_t from = lanes + buf * BN;
                auto add = [&](uint32_t c) {
#pragma unroll
                    for (uint32_t i = 0; i < 32u; ++i) acc[c * 32u + i] = fmaf(__uint_as_float(r[c & 1u][i]), c < 2u ? s0 : s1, acc[c * 32u + i]);
                };
                tc5::tmem_ld_32x32(from, r[0]);
                tc5::tmem_ld_32x32(from + 32u, r[1]);
                tmem_ld_wait(r[0]);
                tmem_ld_wait(r[1]);
                if constexpr (kCols == 128u) {
                    add(0u);
                    tc5::tmem_ld_32x32(from + kSecond, r[0]);
                    add(1u);
                    tc5::tmem_ld_32x32(from + kSecond + 32u, r[1]);
                    tmem_ld_wait(r[0]);
                    tmem_ld_wait(r[1]);
                }
                tc5::fence_before_sync();      // every column is in registers: the buffer goes back
                __syncwarp();
                if (lane == 0u) tc5::mbar_arrive(&sh->acc_empty[buf]);
                add(kCols / 32u - 2u);
                add(kCols / 32u - 1u);
            }
            const uint2 at = place<kPlanes>(tile, tiles_m, tiles_n);
            const uint32_t m0 = at.x * BM, n0 = at.y * kTileN;
            const uint32_t t = m0 + row;
            if constexpr (kPlanes == 1) {
                const uint32_t n = n0 + half * kCols;
                if (ok && t < a.batch && n < a.out_dim)
                    store_row(reinterpret_cast<TO*>(a.y) + (size_t)t * a.out_dim + n, acc, a.out_dim - n, a.row_align);
            } else {
                float m = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < 64u; ++i) {
                    acc[i] = gated(acc[i], acc[64u + i]);
                    m = fmaxf(m, fabsf(acc[i]));
                }
                sh->amax[half][row] = ok ? m : __int_as_float(0x7fffffff);       // NaN, which m never is: this half gave up
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const float other = sh->amax[1u - half][row], sc = scale_of(fmaxf(m, other)), inv = 1.0f / sc;
                asm volatile("bar.sync 1, 256;" ::: "memory");       // read before the next tile's is written
                if (ok && other == other && t < a.batch) {
                    const uint32_t n = n0 + half * 64u;
                    uint8_t* q = reinterpret_cast<uint8_t*>(a.y) + (size_t)t * a.out_dim + n;
#pragma unroll
                    for (uint32_t i = 0; i < 64u; i += 16u)
                        if (n + i < a.out_dim)        // ff % 16 == 0: whole pieces
                            *reinterpret_cast<uint4*>(q + i) = make_uint4(
                                codes4(acc[i], acc[i + 1u], acc[i + 2u], acc[i + 3u], inv), codes4(acc[i + 4u], acc[i + 5u], acc[i + 6u], acc[i + 7u], inv),
                                codes4(acc[i + 8u], acc[i + 9u], acc[i + 10u], acc[i + 11u], inv),
                                codes4(acc[i + 12u], acc[i + 13u], acc[i + 14u], acc[i + 15u], inv));
                    if (half == 0u) a.hs[(size_t)t * w_blocks + n0 / 128u] = sc;
                }
            }
        }
    }

    tc5::fence_before_sync();
    __syncthreads();
    if (sh->abort_flag) wait_for_copies();
    if (warp == 1u) {
        tc5::fence_after_sync();
        tc5::tmem_dealloc(tmem_base, kTmemCols);
    }
}

template <int kPlanes, uint32_t BN, typename TO>
int launch_wide(const Call& c, cudaStream_t st) {
    CUtensorMap tx, tw0, tw1;
    if (int rc = pdk_make_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.xq, c.in_dim, c.batch, c.in_dim, BK, BM)) return rc;
    if (int rc = pdk_make_tmap_2d(&tw0, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.w[0], c.in_dim, c.out_dim, c.in_dim, BK, 128u)) return rc;
    tw1 = tw0;
    if (kPlanes == 2)
        if (int rc = pdk_make_tmap_2d(&tw1, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.w[1], c.in_dim, c.out_dim, c.in_dim, BK, 128u)) return rc;
    Args a{};
    a.ws0 = (const float*)c.ws[0]; a.ws1 = (const float*)c.ws[1]; a.xs = (const float*)c.xs; a.y = c.y; a.hs = (float*)c.hs;
    a.out_dim = c.out_dim; a.batch = c.batch; a.num_kb = blocks_of(c.in_dim);
    const uint64_t where = (uint64_t)(uintptr_t)c.y | (uint64_t)c.out_dim * sizeof(TO);
    a.row_align = where % 32u == 0u ? 32u : where % 16u == 0u ? 16u : (uint32_t)sizeof(TO);
    a.err = pdk_error_word();
    const size_t smem = (size_t)Cfg<BN>::kStages * Cfg<BN>::kStageBytes + sizeof(Shared<Cfg<BN>::kParts>) + 1024u;
    auto kern = f8blk_wide_kernel<kPlanes, BN, TO>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    const uint32_t tile_n = kPlanes == 2 ? 128u : BN;
    const uint64_t n_tiles = (uint64_t)((c.batch + BM - 1u) / BM) * ((c.out_dim + tile_n - 1u) / tile_n);
    if (n_tiles > 0x7fffffffull) return cudaErrorInvalidValue;
    const uint32_t sms = (uint32_t)pdk_sm_count();
    return pdk_launch_pdl(kern, dim3(n_tiles < sms ? (uint32_t)n_tiles : sms), dim3(kThreads), smem, st, tx, tw0, tw1, a);
}

}  // namespace

int pdk_f8blk_wide(const Call& c, int planes, bool bf16, uint32_t cols, cudaStream_t st) {
    if (planes == 2) return launch_wide<2, 256, float>(c, st);
    if (cols == 128u) return bf16 ? launch_wide<1, 128, __nv_bfloat16>(c, st) : launch_wide<1, 128, float>(c, st);
    return bf16 ? launch_wide<1, 256, __nv_bfloat16>(c, st) : launch_wide<1, 256, float>(c, st);
}
