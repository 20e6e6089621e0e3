// Product of two MXFP4 operands on the block-scaled tensor-core path (tcgen05.mma kind::mxf4):
//
//     out[m, n] = bf16( sum_k x[m, k] w[n, k] + bias[n] ),    x = xq * 2^(xs - 127), w = wq * 2^(ws - 127)
//
// The tensor cores multiply the 4-bit codes and apply both blocks' scales themselves; sums are fp32 in tensor memory,
// each result is rounded once.
//
// Pairs of CTAs (cta_group::2) own tiles of 256 x 256: each CTA stages 128 rows of x and 128 of w, 256 of K (128 bytes of
// codes, one swizzle row) per stage, and the scales of its 128 rows of x and of all 256 rows of w -- in the tile order of
// the codec a TMA copy of 512 bytes (128 rows x 4 blocks) is exactly what one tcgen05.cp moves into four columns of tensor
// memory.  Per stage the leader issues six such copies and four MMAs (M 256, N 256, K 64); copies and MMAs of one thread
// run in order.
//
// Tensor memory (512 columns): accumulator 0 in [0, 256), accumulator 1 in [208, 464), two sets of scales (8 + 16
// columns) behind.  The accumulators alternate between tiles and share columns [208, 256): the epilogue reads those
// first and hands them over, so the next tile starts while most of the previous one is still being stored.
//
// Small products run on tiles of 256 x 128 instead: eight stages of 26 KB, two accumulators side by side.
//
// Warps per CTA: 0 TMA, 1 MMA issue (leader CTA) and tensor memory, 2-9 epilogue (two per lane quadrant).
// Waits are bounded as in the fused dequantising product; the status word is read by tcb_fused_dequant_linear_check().
#include <type_traits>

#include "tcb_tcgen05.h"

namespace tcb {
bool mxfp4_few_rows(int64_t M, int64_t N, int64_t K);
int launch_mxfp4_few_rows(const char* who, const void* x, int dtype, const CUtensorMap& map_w, const CUtensorMap& map_ws, const uint16_t* bias,
                          uint16_t* out, int64_t M, int64_t N, int64_t K, cudaStream_t st);
}  // namespace tcb

namespace {

constexpr int kTileRows = 128, kPairRows = 256;
constexpr int kBlockK = 256;                       // values of K per stage
constexpr uint32_t kOperandBytes = 128 * 128;      // 16 KB: codes of x, one CTA, one stage
constexpr uint32_t kScaleBytesA = 1024;            // 128 rows x 8 blocks
constexpr int kEpilogueWarps = 8, kFirstEpilogueWarp = 2;
constexpr int kThreads = 32 * (kFirstEpilogueWarp + kEpilogueWarps);
constexpr uint32_t kScaleCols = 464;               // first tensor-memory column of the scales

// TB: columns of a tile (rows of w).
template <int TB>
struct Config {
    static constexpr int kStages = TB == 256 ? 6 : 8;
    static constexpr uint32_t kBytesB = TB / 2 * 128, kScaleBytesB = TB * 8;
    static constexpr uint32_t kStageBytes = kOperandBytes + kBytesB + kScaleBytesA + kScaleBytesB;
    static constexpr uint32_t kSmemTiles = kStages * kStageBytes + kEpilogueWarps * kStoreStageBytes;
    static constexpr uint32_t kSmem = kSmemTiles + 1024 /* alignment */ + 256 /* barriers */;
    static constexpr uint32_t kAcc1 = TB == 256 ? 208 : 128;   // second accumulator
    static constexpr uint32_t kColsB = TB / 32;                // columns of w's scales per 128 of K
    static_assert(kSmem <= 232448 && (2 * kStages + 3) * 8 + 8 <= 256 && kStageBytes % 1024 == 0, "shared memory");
};

struct Params {
    int64_t M, N;
    const uint16_t* bias;
    uint16_t* out;
    int tiles_m, tiles_n, tiles, num_kb;
};

// x, w: E2M1; scales: E8M0; M = 256, N = TB; K = 64.  sf: which half of a 32-bit word of scales (0 or 2).
template <int TB>
__device__ __forceinline__ constexpr uint32_t inst_desc(uint32_t sf) {
    return (sf << 4) | (1u << 7) | (1u << 10) | (uint32_t(TB >> 3) << 17) | (1u << 23) | (uint32_t(kPairRows >> 7) << 27) | (sf << 29);
}

// The four MMAs of a stage (64 of K = 32 bytes of codes each); the scales of MMAs 2 and 3 sit four (x) and TB / 32 (w)
// columns after those of 0 and 1, within a column the odd ones use the upper half.
template <int TB>
__device__ __forceinline__ void umma_mxf4_x4(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t sfa, uint32_t sfb, uint32_t accumulate_first) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b64 a, b;\n\t.reg .b32 al, bl, sa, sb;\n\t"
        "setp.ne.b32 p, %8, 0;\n\t"
        "setp.eq.b32 t, %8, %8;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %4, [%6], [%7], p;\n\t"
        "add.u32 al, %1, 2;\n\tadd.u32 bl, %2, 2;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %5, [%6], [%7], t;\n\t"
        "add.u32 al, %1, 4;\n\tadd.u32 bl, %2, 4;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
        "add.u32 sa, %6, 4;\n\tadd.u32 sb, %7, %9;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %4, [sa], [sb], t;\n\t"
        "add.u32 al, %1, 6;\n\tadd.u32 bl, %2, 6;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %5, [sa], [sb], t;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(inst_desc<TB>(0)), "r"(inst_desc<TB>(2)), "r"(sfa), "r"(sfb), "r"(accumulate_first), "n"(TB / 32)
        : "memory");
}

// 512 bytes of scales (32 rows of 16 bytes; no swizzle, 8-row groups 128 bytes apart) -> four columns, in both CTAs, each
// from its own shared memory and repeated in all four lane quadrants.
__device__ __forceinline__ void copy_scales(uint32_t d_tmem, uint32_t smem_addr) {
    const uint32_t lo = ((smem_addr & 0x3FFFFu) >> 4) | ((128u >> 4) << 16), hi = (128u >> 4) | (1u << 14);
    asm volatile(
        "{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\t"
        "tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t}" ::"r"(d_tmem),
        "r"(lo), "r"(hi)
        : "memory");
}

struct Tile {
    int m, n;
};
// Bands of 8 tile rows, down the band first, so that the tiles in flight share their operands in L2.
__device__ __forceinline__ Tile decode_tile(const Params& p, int t) {
    const int band = t / (8 * p.tiles_n), first = band * 8;
    const int height = p.tiles_m - first < 8 ? p.tiles_m - first : 8;
    const int u = t - first * p.tiles_n;
    return {first + u % height, u / height};
}

template <int TB>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
mxfp4_linear_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                    const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_ws, const Params p) {
    using C = Config<TB>;
    constexpr int S = C::kStages;
    constexpr uint32_t kStageBytes = C::kStageBytes;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    // stages (codes of x, codes of w, scales of x, scales of w, 1024-byte aligned each), store buffers, barriers
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kSmemTiles);
    // barriers: full (leader), empty, accumulator full [2], shared columns free (leader)
    constexpr int FULL = 0, EMPTY = S, TFULL = 2 * S, TFREE = 2 * S + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 3);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const uint32_t bar0 = smem_u32(bars), smem0 = smem_u32(smem);
    auto bar = [&](int id) { return bar0 + 8u * uint32_t(id); };
    auto leader_bar = [&](int id) { return map_to_cta(bar(id), 0); };
    const uint32_t abort_peer = map_to_cta(smem_u32(const_cast<int*>(abort_flag)), rank ^ 1);

    if (threadIdx.x == 0) {
        prefetch_map(&map_x);
        prefetch_map(&map_w);
        prefetch_map(&map_xs);
        prefetch_map(&map_ws);
        for (int s = 0; s < S; ++s) {
            mbar_init(bar(FULL + s), 2);
            mbar_init(bar(EMPTY + s), 1);
        }
        mbar_init(bar(TFULL), 1);
        mbar_init(bar(TFULL + 1), 1);
        mbar_init(bar(TFREE), 2 * kEpilogueWarps);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    cluster_sync_all();   // both CTAs of the pair are resident before either touches the other's shared or tensor memory
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_slot), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    tcb::await_predecessor();
    const int first = int(blockIdx.x >> 1), step = int(gridDim.x >> 1);

    if (warp == 0) {
        // ---------------------------------------------------------------- TMA
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int tile = first; ok && tile < p.tiles; tile += step) {
                const Tile t = decode_tile(p, tile);
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    ok = mbar_wait(bar(EMPTY + s), ph ^ 1, abort_flag, abort_peer, (1 << 8) | (EMPTY + s));
                    if (!ok) break;
                    const uint32_t full = leader_bar(FULL + s), dst = smem0 + uint32_t(s) * kStageBytes;
                    tma_load_2d_pair(dst, &map_x, kb * 128, t.m * kPairRows + int(rank) * kTileRows, full);
                    tma_load_2d_pair(dst + kOperandBytes, &map_w, kb * 128, t.n * TB + int(rank) * (TB / 2), full);
                    tma_load_2d_pair(dst + kOperandBytes + C::kBytesB, &map_xs, kb * 128, t.m * 2 + int(rank), full);
                    tma_load_2d_pair(dst + kOperandBytes + C::kBytesB + kScaleBytesA, &map_ws, kb * 128, t.n * (TB / 128), full);
                    if (leader) mbar_arrive_expect_tx(bar(FULL + s), 2 * kStageBytes);
                    else mbar_arrive_cluster(full);
                    if (++s == S) { s = 0; ph ^= 1; }
                }
            }
            if (!ok) {   // aborting: copies still in flight land in this CTA's shared memory within microseconds
                const long long t0 = clock64();
                while (clock64() - t0 < 4000000LL) __nanosleep(1000);
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issue
        if (leader) {
            int s = 0, local = 0;
            uint32_t ph = 0, set = 0;
            bool ok = true;
            const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
            const bool elected = elect_one();
            for (int tile = first; ok && tile < p.tiles; tile += step, ++local) {
                // the columns the two accumulators share have been read (and with them everything of the tile before that)
                ok = __all_sync(0xffffffffu, mbar_wait(bar(TFREE), (local & 1) ^ 1, abort_flag, abort_peer, (2 << 8) | TFREE));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + ((local & 1) ? C::kAcc1 : 0u);
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    ok = __all_sync(0xffffffffu, mbar_wait(bar(FULL + s), ph, abort_flag, abort_peer, (2 << 8) | (FULL + s)));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t src = smem0 + uint32_t(s) * kStageBytes;
                    const uint32_t sa = src + kOperandBytes + C::kBytesB, sb = sa + kScaleBytesA;
                    const uint32_t ta = tmem + kScaleCols + (8u + 2 * C::kColsB) * set, tb = ta + 8u;
                    if (elected) {
#pragma unroll
                        for (uint32_t c = 0; c < 2; ++c) {   // 128 of K: four scales a row
                            copy_scales(ta + 4 * c, sa + 512 * c);
#pragma unroll
                            for (uint32_t j = 0; j < TB / 128; ++j)   // 128 rows of w
                                copy_scales(tb + C::kColsB * c + 4 * j, sb + 1024 * j + 512 * c);
                        }
                        umma_mxf4_x4<TB>(d, smem_desc_lo(src), smem_desc_lo(src + kOperandBytes), ta, tb, kb > 0 ? 1u : 0u);
                        umma_commit_both(bar(EMPTY + s));
                    }
                    __syncwarp();
                    set ^= 1;
                    if (++s == S) { s = 0; ph ^= 1; }
                }
                if (ok && elected) umma_commit_both(bar(TFULL + (local & 1)));
                __syncwarp();
            }
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        const int quad = warp & 3, half = (warp - kFirstEpilogueWarp) >> 2;
        const StoreMode mode = store_mode(p.out, p.N, p.bias);
        uint32_t* stage = reinterpret_cast<uint32_t*>(smem + S * kStageBytes + (warp - kFirstEpilogueWarp) * kStoreStageBytes);
        int local = 0;
        bool ok = true;
        for (int tile = first; ok && tile < p.tiles; tile += step, ++local) {
            const Tile t = decode_tile(p, tile);
            const int buf = local & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(bar(TFULL + buf), (local >> 1) & 1, abort_flag, abort_peer, (4 << 8) | (TFULL + buf)));
            if (!ok) break;
            tc_fence_after();
            const int64_t row0 = int64_t(t.m) * kPairRows + int64_t(rank) * kTileRows + quad * 32;
            const uint32_t taddr = tmem_base + (uint32_t(quad * 32) << 16) + (buf ? C::kAcc1 : 0u);
#pragma unroll 1
            for (int i = 0; i < TB / 64; ++i) {
                // chunks of 32 columns; the two of shared columns come first (the last two of accumulator 0, the first two of 1)
                const int c = buf ? 2 * i + half : TB / 32 - 1 - 2 * i - half;
                const int64_t col0 = int64_t(t.n) * TB + c * 32;
                uint32_t v[32];
                tmem_ld32(taddr + uint32_t(c * 32), v);
                tmem_ld_wait();
                if (i == 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(leader_bar(TFREE));
                }
                if (col0 < p.N) store_32x32(p.out, p.N, row0, p.M, col0, p.N, p.bias, v, mode, stage);
            }
        }
    }

    // Neither CTA leaves while the other may still arrive on its barriers or read its shared memory.
    tc_fence_before();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

// ------------------------------------------------------------------------ host

int64_t scale_bytes(int64_t rows, int64_t K) { return (rows + 127) / 128 * ((K + 127) / 128) * 512; }
int64_t code_bytes(int64_t rows, int64_t K) { return (rows * (K / 2) + 511) / 512 * 512; }

// Codes: rows of K / 2 bytes in boxes of `code_rows` rows x 128 bytes.  Scales: one row of the map per 128 rows of the operand,
// in 8-byte elements, boxes of `box_rows` x 1024 bytes.  What lies outside is read as 0.
int encode_maps(const char* who, CUtensorMap* codes_map, CUtensorMap* scales_map, const uint8_t* codes, const uint8_t* scales, int64_t rows,
                int64_t K, int code_rows, int box_rows) {
    EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return tcb::fail(TCB_ERR_CUDA, "%s: cuTensorMapEncodeTiled is not available from the driver", who);
    const cuuint32_t estr[2] = {1, 1};
    const cuuint64_t cdims[2] = {cuuint64_t(K / 2), cuuint64_t(rows)}, cstride[1] = {cuuint64_t(K / 2)};
    const cuuint32_t cbox[2] = {128, cuuint32_t(code_rows)};
    CUresult cr = encode(codes_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), cdims, cstride, cbox, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) return tcb::fail(TCB_ERR_CUDA, "%s: cuTensorMapEncodeTiled (codes) failed with %d", who, int(cr));
    const int64_t tk = (K + 127) / 128;
    const cuuint64_t sdims[2] = {cuuint64_t(tk * 64), cuuint64_t((rows + 127) / 128)}, sstride[1] = {cuuint64_t(tk * 512)};
    const cuuint32_t sbox[2] = {128, cuuint32_t(box_rows)};
    cr = encode(scales_map, CU_TENSOR_MAP_DATA_TYPE_INT64, 2, const_cast<uint8_t*>(scales), sdims, sstride, sbox, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) return tcb::fail(TCB_ERR_CUDA, "%s: cuTensorMapEncodeTiled (scales) failed with %d", who, int(cr));
    return TCB_OK;
}

}  // namespace

namespace tcb {
int take_mxfp4_status(int* status) { return take_status(g_status, status); }
}  // namespace tcb

extern "C" int64_t tcb_mxfp4_linear_workspace(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || tcb::mxfp4_few_rows(M, N, K)) return 0;
    return code_bytes(M, K) + scale_bytes(M, K);
}

extern "C" int tcb_mxfp4_linear(const void* x, int dtype, const uint8_t* wq, const uint8_t* w_scales, const uint16_t* bias_or_null, uint16_t* out,
                                int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "tcb_mxfp4_linear";
    const int64_t limit = (int64_t(1) << 31) - 1024;   // coordinates of the last tile stay within 32 bits
    if (dtype < TCB_DT_BF16 || dtype > TCB_DT_F32) return tcb::fail(TCB_ERR_BAD_ARG, "%s: unknown dtype %d", who, dtype);
    if (M < 0 || N < 0 || K < 0) return tcb::fail(TCB_ERR_BAD_ARG, "%s: negative size", who);
    if (M == 0 || N == 0) return TCB_OK;
    if (K <= 0 || K % 32 != 0) return tcb::fail(TCB_ERR_BAD_ARG, "%s: K = %lld must be a positive multiple of 32", who, (long long)K);
    if (M > limit || N > limit || K > limit) return tcb::fail(TCB_ERR_TOO_LARGE, "%s: dimension beyond 2^31 - 1024", who);
    const int64_t tiles_m = (M + kPairRows - 1) / kPairRows, tiles_n = (N + kPairRows - 1) / kPairRows;
    if (tiles_m * tiles_n > (int64_t(1) << 30)) return tcb::fail(TCB_ERR_TOO_LARGE, "%s: too many output tiles", who);
    if (!x || !wq || !w_scales || !out) return tcb::fail(TCB_ERR_BAD_ARG, "%s: null pointer", who);
    if ((reinterpret_cast<uintptr_t>(x) & 31) || ((reinterpret_cast<uintptr_t>(wq) | reinterpret_cast<uintptr_t>(w_scales)) & 15))
        return tcb::fail(TCB_ERR_ALIGNMENT, "%s: x must be 32-byte and codes and scales 16-byte aligned", who);
    if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias_or_null)) & 1)
        return tcb::fail(TCB_ERR_ALIGNMENT, "%s: bias and out must be 2-byte aligned", who);
    const int64_t need = tcb_mxfp4_linear_workspace(M, N, K);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
        return tcb::fail(TCB_ERR_BAD_ARG, "%s: the workspace is too small or not 16-byte aligned", who);
    CUtensorMap map_x, map_w, map_xs, map_ws;
    if (need == 0) {   // few rows: w in boxes of 128 rows, x quantised by the product itself
        const int few = encode_maps(who, &map_w, &map_ws, wq, w_scales, N, K, kTileRows, 1);
        return few != TCB_OK ? few : tcb::launch_mxfp4_few_rows(who, x, dtype, map_w, map_ws, bias_or_null, out, M, N, K, static_cast<cudaStream_t>(stream));
    }
    uint8_t* xq = static_cast<uint8_t*>(workspace);
    uint8_t* xs = xq + code_bytes(M, K);
    int rc = tcb_quantize_mxfp4(x, dtype, M, K, xq, xs, stream);
    if (rc == TCB_OK) rc = encode_maps(who, &map_x, &map_xs, xq, xs, M, K, kTileRows, 1);
    if (rc != TCB_OK) return rc;
    // Tiles of 256 x 128 where all of them run at once: half the products and half the results to store per SM (us with the
    // quantisation, halved / whole tiles: 446 x 1001 x 768 8.4 / 11.2, 64 x 4096 x 4096 10.9 / 12.0, 512 x 4736 x 4096 12.5 / 13.6,
    // 1024 x 1024 x 1024 7.9 / 9.2).  With more of them the second round costs more than that (64 x 10240 x 4096 16.0 / 12.9, 512 x
    // 5120 x 4096 17.2 / 14.0, 2048 x 4096 x 4096 31.8 / 23.8; on short sums it does not matter: 1024 x 4096 x 768 9.8 / 10.1).
    const int pairs = tcb::sm_count() / 2 > 0 ? tcb::sm_count() / 2 : 1;
    Params p;
    p.M = M;
    p.N = N;
    p.bias = bias_or_null;
    p.out = out;
    p.tiles_m = int(tiles_m);
    p.num_kb = int((K + kBlockK - 1) / kBlockK);
    const auto run = [&](auto tag) {
        constexpr int TB = decltype(tag)::value;
        p.tiles_n = int((N + TB - 1) / TB);
        p.tiles = p.tiles_m * p.tiles_n;
        const int status = encode_maps(who, &map_w, &map_ws, wq, w_scales, N, K, TB / 2, TB / 128);
        if (status != TCB_OK) return status;
        static std::atomic<bool> attr_set[64] = {};
        int dev = 0;
        TCB_CUDA_TRY(cudaGetDevice(&dev));
        if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
            TCB_CUDA_TRY(cudaFuncSetAttribute(mxfp4_linear_kernel<TB>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Config<TB>::kSmem)));
            if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
        }
        TCB_CUDA_TRY(tcb::launch_overlapped(mxfp4_linear_kernel<TB>, dim3(2 * (p.tiles < pairs ? p.tiles : pairs)), dim3(kThreads), Config<TB>::kSmem,
                                            static_cast<cudaStream_t>(stream), map_x, map_w, map_xs, map_ws, p));
        return int(TCB_OK);
    };
    return tiles_m * ((N + 127) / 128) <= pairs ? run(std::integral_constant<int, 128>()) : run(std::integral_constant<int, 256>());
}
