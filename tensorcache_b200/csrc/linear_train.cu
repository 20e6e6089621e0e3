// Training step of a linear layer whose input is kept in 8 bits: three products on the tcgen05 tensor cores.
//
//     forward       y[m, n]  = sum_k x[m, k] w[n, k] + b[n]
//     input grad    dx[m, k] = sum_n dy[m, n] w[n, k]
//     weight grad   dw[n, k] = sum_m dy[m, n] deq(q)[m, k]          db[n] = sum_m dy[m, n]
//
// x, w, dy, y and the gradients are bf16, sums are fp32 (TMEM accumulators, fp32 partial sums) and rounded once.  The
// kept input exists as int8 / uint8 codes and group scales only; deq(q) is the bf16 number the decode kernels
// produce (finite always: convert16), made in shared memory by producer warps, and never goes to global memory.  (code x scale has up to 16 bits and the
// tensor cores take 8 of them: half a step of bf16 per term, 1.6e-3 of the norm of dw in all, as much as dw's own rounding.
// Codes alone would be exact, but their scales change along the columns of a tile and cannot move to the other operand.)
//
// One kernel serves all three: D[a, b] = sum_c A[a, c] B[b, c] on tiles of a pair of CTAs (tcgen05.mma.cta_group::2),
// 64 of the contraction per stage.  What differs is which way the operands lie in memory:
//     forward       A = x  (contraction contiguous)        B = w   (contraction contiguous)
//     input grad    A = dy (contraction contiguous)        B = w   (rows contiguous)
//     weight grad   A = dy (rows contiguous)               B = q   (rows contiguous, dequantised)
// An operand whose contraction is contiguous is staged as 128 rows x 64 (128-byte rows, 128-byte swizzle), one whose
// rows are contiguous as two boxes of 64 contraction steps x 64 rows, in the same swizzle: the tensor core reads either
// (the "major" bits of the instruction descriptor), so nothing is transposed by anyone.
//
// Forward and input gradient: tiles of 256 x 256 (each CTA stages 128 rows of A and 128 of B), or 256 x 128 for small
// products; the two accumulators alternate between tiles, so a tile's epilogue runs under the next one's products.
// Weight gradient: tiles of 512 x 256, both accumulators on one tile.  Decoding 128 rows costs the producers and the
// shared-memory pipe about as long as one 256 x 256 step of MMAs takes (measured with 256 x 256 tiles: 854 us for 16384
// x 4096 x 4096, 330 us for the products without decoding); used against 512 rows of A it hides behind two of them.
// A tile whose second half would lie outside runs one half only, and so do all tiles of a small product.
// Where the output has too few tiles to fill the GPU the contraction is split: each part leaves fp32 sums in a workspace
// and a second kernel adds them in a fixed order (results do not depend on timing).
//
// Warps per CTA: 0 TMA, 1 MMA issue (leader CTA) and TMEM, then eight epilogue warps, then eight dequantising producers
// (weight gradient only).
//
// Waits are bounded as in the fused dequantising product; the status word is read by tcb_fused_dequant_linear_check().
#include <type_traits>

#include "tcb_tcgen05.h"

namespace {

constexpr int kTileRows = 128;                       // rows of each operand per CTA
constexpr int kPairRows = 256;                       // per pair
constexpr int kBlockK = 64;                          // contraction per stage
constexpr uint32_t kOperandBytes = 128 * 64 * 2;     // 16 KB: one operand, one CTA, one stage
constexpr uint32_t kCodeBytes = 128 * 64;            // 8 KB of raw codes
constexpr uint32_t kBoxBytes = 64 * 64 * 2;          // 8 KB: 64 contraction steps x 64 rows
constexpr int kProducerWarps = 8, kFirstEpilogueWarp = 2;
constexpr uint32_t kMaxSmem = 232448;

enum Source { kContraction, kRows, kCodes };         // how an operand lies in memory (kCodes: rows contiguous, 8-bit codes)

template <Source B, int TB>
struct Config {
    static_assert(TB == 256 || (TB == 128 && B != kCodes), "columns of a tile");
    static constexpr bool kDeq = B == kCodes;
    static constexpr int kGroups = kDeq ? 2 : 1;             // accumulators per tile = 128-row units of A per CTA
    static constexpr int kBuffers = 2 / kGroups;             // tiles in flight in tensor memory
    static constexpr int kRowsB = TB / 2;                    // rows of B per CTA
    static constexpr int kEpilogueWarps = 8;                 // per lane quadrant: one per accumulator, or two per tile
    static constexpr int kFirstProducerWarp = kFirstEpilogueWarp + kEpilogueWarps;
    static constexpr int kThreads = 32 * (kFirstProducerWarp + (kDeq ? kProducerWarps : 0));
    static constexpr int kStages = kDeq ? 4 : TB == 256 ? 6 : 8;
    static constexpr uint32_t kBytesA = kGroups * kOperandBytes, kBytesB = kRowsB * kBlockK * 2;
    // store buffers of the epilogue; the weight gradient's columns are a multiple of 16 and its output aligned: none
    static constexpr uint32_t kStore = kDeq ? 0 : kEpilogueWarps * kStoreStageBytes;
    static constexpr uint32_t kTiles = kStages * (kBytesA + kBytesB + (kDeq ? kCodeBytes : 0)) + kStore;
    static constexpr uint32_t kSmem = kTiles + 1024 /* alignment */ + 256 /* barriers */;
    static_assert(kSmem <= kMaxSmem && (3 * kStages + 4) * 8 + 8 <= 256, "shared memory");
};

struct Params {
    int64_t rows_a, rows_b;     // output rows and columns
    const uint16_t* bias;       // null, or one per column (only without a split)
    uint16_t* out;              // [rows_a, rows_b]
    float* partial;             // split: [splits][rows_a][ld_partial]
    int64_t ld_partial;
    const uint16_t* columns;    // weight gradient: null, or dy, whose column sums the epilogue warps leave ...
    int64_t ld_columns;
    float* column_parts;        // ... here, [warps of all CTAs by their row slice][rows_a]
    const uint16_t* scales;     // codes: [contraction, rows_b / G]
    const uint8_t* zp;
    int64_t contraction;
    int tiles_a, tiles_b, tiles;    // tiles = tiles_a * tiles_b
    int tile_a;                     // output rows per tile: 256, or 512 (weight gradient)
    int num_kb, kb_per_split, items;
};

struct Item {
    int row_a, tb, split, kb0, kb1;   // first output row of the tile, tile column, part and stages of the contraction
    int groups;                       // 256-row halves of the tile that hold rows of the output
};

// Work items: the tiles of split 0, then those of split 1, ...  Tiles run in bands of 8 tile rows, down the band first,
// so that the tiles in flight share their operands in L2.
template <int GROUPS>
__device__ __forceinline__ Item decode_item(const Params& p, int item) {
    Item r;
    r.split = item / p.tiles;
    const int t = item - r.split * p.tiles;
    const int band = t / (8 * p.tiles_b), first = band * 8;
    const int height = p.tiles_a - first < 8 ? p.tiles_a - first : 8;
    const int u = t - first * p.tiles_b;
    r.row_a = (first + u % height) * p.tile_a;
    r.tb = u / height;
    r.kb0 = r.split * p.kb_per_split;
    r.kb1 = r.kb0 + p.kb_per_split < p.num_kb ? r.kb0 + p.kb_per_split : p.num_kb;
    r.groups = GROUPS == 2 && p.tile_a > kPairRows && int64_t(r.row_a) + kPairRows < p.rows_a ? 2 : 1;
    return r;
}

// Leading byte offset (in 16-byte units) of an operand's descriptor: contraction contiguous -- unused, 1; rows
// contiguous -- from one box of 64 rows to the next.  The stride (1024 bytes: 8 rows of 128 bytes) is the same.
template <bool ROWS>
__device__ __forceinline__ uint32_t operand_lo(uint32_t smem_addr) {
    return ((smem_addr & 0x3FFFFu) >> 4) | ((ROWS ? kBoxBytes >> 4 : 1u) << 16);
}

// The four MMAs (16 of the contraction each) of a stage.
template <uint32_t STEP_A, uint32_t STEP_B>
__device__ __forceinline__ void umma_x4(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate_first) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b64 a, b;\n\t.reg .b32 al, bl;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "setp.eq.b32 t, %5, %5;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, p;\n\t"
        "add.u32 al, %1, %6;\n\tadd.u32 bl, %2, %7;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, t;\n\t"
        "add.u32 al, al, %6;\n\tadd.u32 bl, bl, %7;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, t;\n\t"
        "add.u32 al, al, %6;\n\tadd.u32 bl, bl, %7;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, t;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate_first), "n"(STEP_A), "n"(STEP_B)
        : "memory");
}

// ROWS rows of an operand for one stage: rows [row, row + ROWS), contraction [c, c + 64).
template <Source S, int ROWS>
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap* map, int row, int c, uint32_t bar) {
    if constexpr (S == kContraction) {
        tma_load_2d_pair(dst, map, c, row, bar);
    } else {
#pragma unroll
        for (int i = 0; i < ROWS / 64; ++i) tma_load_2d_pair(dst + i * kBoxBytes, map, row + 64 * i, c, bar);
    }
}

// How the column sums of [rows, cols] are shared out: a warp takes blocks of 64 columns; with fewer than eight blocks the
// eight warps of a CTA take slices of the rows as well.
struct ColumnShare {
    int blocks, slices;   // column blocks; row slices per CTA
    __host__ __device__ explicit ColumnShare(int64_t cols) : blocks(int((cols + 63) / 64)), slices(blocks >= 8 ? 1 : 8 / blocks) {}
};

// Column sums of one warp: 64 columns (8 lanes of 16 bytes a row), every parts-th run of 16 rows, fp32.
__device__ __forceinline__ void sum_columns(const uint16_t* __restrict__ x, int64_t rows, int64_t cols, int64_t ld, int block, int part, int parts,
                                            float* __restrict__ out) {
    const int lane = threadIdx.x & 31;
    const int64_t col = int64_t(block) * 64 + (lane & 7) * 8;
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (col < cols)   // ld is a multiple of 8: a whole 16-byte piece is there
        for (int64_t row = int64_t(part) * 16 + (lane >> 3); row < rows; row += int64_t(parts) * 16) {
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = row + 4 * j < rows ? __ldg(reinterpret_cast<const uint4*>(x + (row + 4 * j) * ld + col)) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[2 * i] += __uint_as_float(w[i] << 16);
                    s[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
                }
            }
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 8);
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 16);
        if (lane < 8 && col + i < cols) out[int64_t(part) * cols + col + i] = s[i];
    }
}

template <Source A, Source B, int TB, int LOG2_G, bool HAS_ZP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Config<B, TB>::kThreads, 1)
linear_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
    using C = Config<B, TB>;
    constexpr int S = C::kStages;
    // bf16 x bf16 -> fp32, M = 256, N = TB; bits 15 / 16: rows contiguous
    constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((A != kContraction ? 1u : 0u) << 15) |
                                ((B != kContraction ? 1u : 0u) << 16) | (uint32_t(TB >> 3) << 17) | (uint32_t(kPairRows >> 4) << 24);
    // 16 of the contraction in the descriptor's 16-byte units: 32 bytes along a row, or 16 rows of 128 bytes
    constexpr uint32_t kStepA = A == kContraction ? 2 : 128, kStepB = B == kContraction ? 2 : 128;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* smem_a = smem;
    uint8_t* smem_b = smem_a + S * C::kBytesA;
    uint8_t* smem_c = smem_b + S * C::kBytesB;
    uint8_t* smem_e = smem + C::kTiles - C::kStore;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kTiles);
    // barriers: full (leader), empty, full_c (raw codes), accumulator full [2], accumulator empty [2] (leader)
    constexpr int FULL = 0, EMPTY = S, FULL_C = 2 * S, TFULL = 3 * S, TEMPTY = 3 * S + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * S + 4);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int id) { return bar0 + 8u * uint32_t(id); };
    auto leader_bar = [&](int id) { return map_to_cta(bar(id), 0); };
    const uint32_t abort_peer = map_to_cta(smem_u32(const_cast<int*>(abort_flag)), rank ^ 1);

    if (threadIdx.x == 0) {
        prefetch_map(&map_a);
        prefetch_map(&map_b);
        for (int s = 0; s < S; ++s) {
            mbar_init(bar(FULL + s), 2 + (C::kDeq ? 2 * kProducerWarps : 0));
            mbar_init(bar(EMPTY + s), 1);
            mbar_init(bar(FULL_C + s), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(TFULL + i), 1);
            mbar_init(bar(TEMPTY + i), 2 * C::kEpilogueWarps);
        }
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
            for (int item = first; ok && item < p.items; item += step) {
                const Item t = decode_item<C::kGroups>(p, item);
                const int units = t.groups;   // 128-row units of A per CTA
                const int row_a = t.row_a + int(rank) * units * kTileRows, row_b = t.tb * TB + int(rank) * C::kRowsB;
                for (int kb = t.kb0; kb < t.kb1; ++kb) {
                    ok = mbar_wait(bar(EMPTY + s), ph ^ 1, abort_flag, abort_peer, (1 << 8) | (EMPTY + s));
                    if (!ok) break;
                    const uint32_t full = leader_bar(FULL + s), dst_a = smem_u32(smem_a) + uint32_t(s) * C::kBytesA;
                    for (int u = 0; u < units; ++u)
                        load_operand<A, kTileRows>(dst_a + uint32_t(u) * kOperandBytes, &map_a, row_a + u * kTileRows, kb * kBlockK, full);
                    if constexpr (C::kDeq) {
                        mbar_arrive_expect_tx(bar(FULL_C + s), kCodeBytes);
                        tma_load_2d(smem_u32(smem_c + s * kCodeBytes), &map_b, row_b, kb * kBlockK, bar(FULL_C + s));
                    } else {
                        load_operand<B, C::kRowsB>(smem_u32(smem_b + s * C::kBytesB), &map_b, row_b, kb * kBlockK, full);
                    }
                    if (leader) mbar_arrive_expect_tx(bar(FULL + s), 2 * (uint32_t(units) * kOperandBytes + (C::kDeq ? 0u : C::kBytesB)));
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
            uint32_t ph = 0;
            bool ok = true;
            const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
            const bool elected = elect_one();
            const uint32_t a0 = operand_lo<A != kContraction>(smem_u32(smem_a)), b0 = operand_lo<B != kContraction>(smem_u32(smem_b));
            for (int item = first; ok && item < p.items; item += step, ++local) {
                const Item t = decode_item<C::kGroups>(p, item);
                const int buf = local % C::kBuffers;
                ok = __all_sync(0xffffffffu, mbar_wait(bar(TEMPTY + buf), ((local / C::kBuffers) & 1) ^ 1, abort_flag, abort_peer,
                                                       (2 << 8) | (TEMPTY + buf)));
                if (!ok) break;
                tc_fence_after();
                // once per number of groups, so that the issue sequence of a stage has no branch in it
                auto sum_up = [&](auto groups_tag) {
                    for (int kb = t.kb0; kb < t.kb1; ++kb) {
                        ok = __all_sync(0xffffffffu, mbar_wait(bar(FULL + s), ph, abort_flag, abort_peer, (2 << 8) | (FULL + s)));
                        if (!ok) break;
                        tc_fence_after();
                        if (elected) {
#pragma unroll
                            for (int h = 0; h < decltype(groups_tag)::value; ++h)
                                umma_x4<kStepA, kStepB>(tmem + uint32_t((buf + h) * kPairRows),
                                                        a0 + (uint32_t(s) * C::kBytesA + uint32_t(h) * kOperandBytes) / 16,
                                                        b0 + uint32_t(s) * (C::kBytesB / 16), kIdesc, kb > t.kb0 ? 1u : 0u);
                            umma_commit_both(bar(EMPTY + s));
                        }
                        __syncwarp();
                        if (++s == S) { s = 0; ph ^= 1; }
                    }
                };
                if (C::kGroups == 2 && t.groups == 2) sum_up(std::integral_constant<int, C::kGroups>());
                else sum_up(std::integral_constant<int, 1>());
                if (ok && elected) umma_commit_both(bar(TFULL + buf));
                __syncwarp();
            }
        }
    } else if (warp < C::kFirstProducerWarp) {
        // ---------------------------------------------------------------- epilogue
        const int quad = warp & 3;                            // the TMEM lanes this warp may read
        const int upper = (warp - kFirstEpilogueWarp) >> 2;   // one of the two warps of a lane quadrant
        const StoreMode mode = store_mode(p.out, p.rows_b, p.bias);
        uint32_t* stage = reinterpret_cast<uint32_t*>(smem_e + (C::kStore ? (warp - kFirstEpilogueWarp) * kStoreStageBytes : 0));
        if constexpr (C::kDeq) {
            // Bias gradient: these warps have nothing to do until the first tile is complete, and memory has time to spare (57,088 x
            // 1000: 39 us less than with a kernel of its own).
            if (p.columns) {
                const ColumnShare share(p.rows_a);
                const int w = warp - kFirstEpilogueWarp;
                if (w / share.blocks < share.slices)
                    for (int block = w % share.blocks; block < share.blocks; block += 8)
                        sum_columns(p.columns, p.contraction, p.rows_a, p.ld_columns, block, int(blockIdx.x) * share.slices + w / share.blocks,
                                    int(gridDim.x) * share.slices, p.column_parts);
            }
        }
        int local = 0;
        bool ok = true;
        for (int item = first; ok && item < p.items; item += step, ++local) {
            const Item t = decode_item<C::kGroups>(p, item);
            const int buf = local % C::kBuffers;
            ok = __all_sync(0xffffffffu,
                            mbar_wait(bar(TFULL + buf), (local / C::kBuffers) & 1, abort_flag, abort_peer, (4 << 8) | (TFULL + buf)));
            if (!ok) break;
            tc_fence_after();
            // two accumulators: one each; one: every second chunk of its columns
            const int group = C::kGroups == 2 && t.groups == 2 ? upper : 0, chunk0 = upper - group, step_c = t.groups == 2 ? 1 : 2;
            const int64_t row0 = int64_t(t.row_a) + (int64_t(rank) * t.groups + group) * kTileRows + quad * 32;
            const uint32_t taddr = tmem_base + (uint32_t(quad * 32) << 16) + uint32_t((buf + group) * kPairRows);
#pragma unroll 1
            for (int c = chunk0; c < TB / 32; c += step_c) {
                const int64_t col0 = int64_t(t.tb) * TB + c * 32;
                if (col0 >= p.rows_b) break;   // warp-uniform
                if (p.partial) {
                    store_32x32_f32(taddr + uint32_t(c * 32), p.partial + int64_t(t.split) * p.rows_a * p.ld_partial, p.ld_partial, row0, p.rows_a, col0);
                    continue;
                }
                uint32_t v[32];
                tmem_ld32(taddr + uint32_t(c * 32), v);
                tmem_ld_wait();
                store_32x32(p.out, p.rows_b, row0, p.rows_a, col0, p.rows_b, p.bias, v, mode, stage);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(leader_bar(TEMPTY + buf));
        }
    } else if constexpr (C::kDeq) {
        // ---------------------------------------------------------------- dequantising producers
        // Warp pw takes contraction rows [8 pw, 8 pw + 8) of the stage, a lane 2 x 16 codes of one row: columns
        // 16 kq + 64 h of the CTA's 128 (h = 0, 1).  Rows of odd number read their upper half first, so that neither the
        // reads of codes nor the writes of operand pieces meet in a bank.
        const int pw = warp - C::kFirstProducerWarp, r = pw * 8 + (lane >> 2), kq = lane & 3, h0 = r & 1;
        const uint32_t piece0 = uint32_t(((2 * kq) ^ (r & 7)) * 16), piece1 = piece0 ^ 16u;
        const int64_t gpr = p.rows_b >> LOG2_G, stage_groups = gpr * kBlockK;
        // Scale and zero point of the lane's two pieces are fetched a whole ring ahead, into registers named by the stage: the
        // loop is unrolled over the ring, because moving (or even shifting) a value that is still on its way would wait for it
        // -- that cost a tenth of the kernel's time.
        int pf_item = first, pf_kb = 0, pf_end = 0;
        int64_t g[2] = {0, 0};        // group of the piece in the row being fetched; negative: outside
        auto start = [&]() {
            const Item t = decode_item<C::kGroups>(p, pf_item);
            pf_kb = t.kb0;
            pf_end = t.kb1;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t k = int64_t(t.tb) * TB + int64_t(rank) * C::kRowsB + 16 * kq + 64 * (h0 ^ i);
                g[i] = k < p.rows_b ? (int64_t(pf_kb) * kBlockK + r) * gpr + (k >> LOG2_G) : INT64_MIN;
            }
        };
        start();
        uint32_t scale[S][2], zero[S][2];
        auto fetch = [&](int slot) {
            const bool inside = pf_item < p.items && pf_kb * kBlockK + r < int(p.contraction);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool ok = inside && g[i] >= 0;
                scale[slot][i] = ok ? __ldg(p.scales + g[i]) : uint16_t(0);
                zero[slot][i] = HAS_ZP && ok ? __ldg(p.zp + g[i]) : uint8_t(0);
                g[i] += stage_groups;
            }
            if (++pf_kb == pf_end) {
                pf_item += step;
                if (pf_item < p.items) start();
            }
        };
        int total = 0;                // stages of all of this pair's items
        for (int item = first; item < p.items; item += step) {
            const Item t = decode_item<C::kGroups>(p, item);
            total += t.kb1 - t.kb0;
        }
#pragma unroll
        for (int s = 0; s < S; ++s) fetch(s);
        uint32_t ph = 0;
        bool ok = true;
        for (int i0 = 0; ok && i0 < total; i0 += S, ph ^= 1) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                if (i0 + s >= total) break;
                const uint32_t sz0 = (scale[s][0] << 16) | zero[s][0], sz1 = (scale[s][1] << 16) | zero[s][1];
                fetch(s);
                // warp-uniform verdict: the warp-level sync below needs every lane
                ok = __all_sync(0xffffffffu, mbar_wait(bar(FULL_C + s), ph, abort_flag, abort_peer, (3 << 8) | (FULL_C + s)));
                if (!ok) break;
                const uint8_t* c = smem_c + s * kCodeBytes + r * 128 + kq * 16;
                const uint4 c0 = *reinterpret_cast<const uint4*>(c + 64 * h0), c1 = *reinterpret_cast<const uint4*>(c + 64 * (h0 ^ 1));
                uint8_t* d = smem_b + s * C::kBytesB + r * 128;
                uint8_t *d0 = d + h0 * kBoxBytes, *d1 = d + (h0 ^ 1) * kBoxBytes;
                convert16<HAS_ZP>(c0, sz0, d0 + piece0, d0 + piece1);
                convert16<HAS_ZP>(c1, sz1, d1 + piece0, d1 + piece1);
                fence_proxy_async();   // the stores above become visible to the tensor cores
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(leader_bar(FULL + s));
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

// Sums what the kernels above left in parts, in a fixed order.  Blocks [0, column_blocks): 32 column sums each, eight warps take
// every eighth part.  The others: out[a, b] = bf16(sum over the splits + bias[b]), four columns per thread.
struct Parts {
    const float* partial;       // [splits][rows][ld]
    int splits;
    int64_t rows, cols, ld;
    const uint16_t* bias;
    uint16_t* out;
    const float* columns;       // [column_parts][num_columns]
    int column_parts, column_blocks;
    int64_t num_columns;
    uint16_t* column_out;
};
__global__ void __launch_bounds__(256) add_parts_kernel(const Parts p) {
    tcb::await_predecessor();
    if (int(blockIdx.x) < p.column_blocks) {
        __shared__ float acc[8][32];
        const int r = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const int64_t col = int64_t(blockIdx.x) * 32 + lane;
        float sum = 0.0f;
        if (col < p.num_columns) {
#pragma unroll 4
            for (int i = r; i < p.column_parts; i += 8) sum += p.columns[int64_t(i) * p.num_columns + col];
        }
        acc[r][lane] = sum;
        __syncthreads();
        if (r == 0 && col < p.num_columns) {
#pragma unroll
            for (int i = 1; i < 8; ++i) sum += acc[i][lane];
            p.column_out[col] = f32_to_bf16_bits(sum);
        }
        return;
    }
    const int64_t quads = p.ld / 4, total = p.rows * quads, step = int64_t(gridDim.x - p.column_blocks) * 256;
    for (int64_t i = int64_t(blockIdx.x - p.column_blocks) * 256 + threadIdx.x; i < total; i += step) {
        const int64_t row = i / quads, col = (i - row * quads) * 4;
        if (col >= p.cols) continue;
        float4 sum = __ldcs(reinterpret_cast<const float4*>(p.partial + row * p.ld + col));
#pragma unroll 4
        for (int s = 1; s < p.splits; ++s) {
            const float4 v = __ldcs(reinterpret_cast<const float4*>(p.partial + (int64_t(s) * p.rows + row) * p.ld + col));
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        const float f[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < p.cols) {
                const float b = p.bias ? __uint_as_float(uint32_t(p.bias[col + j]) << 16) : 0.0f;
                p.out[row * p.cols + col + j] = f32_to_bf16_bits(f[j] + b);
            }
    }
}

// Column sums where no weight gradient is wanted: a warp per block of columns and part.
__global__ void __launch_bounds__(256) column_sums_kernel(const uint16_t* __restrict__ dy, int64_t rows, int64_t cols, int64_t ld, int parts,
                                                          float* __restrict__ out) {
    tcb::await_predecessor();
    const ColumnShare share(cols);
    const int64_t unit = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (unit < int64_t(share.blocks) * parts) sum_columns(dy, rows, cols, ld, int(unit % share.blocks), int(unit / share.blocks), parts, out);
}

// ------------------------------------------------------------------------ host

struct Plan {
    int tile_a = kPairRows, tile_b = 256;
    int64_t tiles_a = 0, tiles_b = 0, num_kb = 0;
    int splits = 1, kb_per_split = 0;
    int64_t ld_partial = 0;
    int64_t partial_bytes(int64_t rows_a) const { return splits > 1 ? int64_t(splits) * rows_a * ld_partial * 4 : 0; }
};

// Tiles and split of a product (codes: the weight gradient), by the estimated time in us of the longest pair of CTAs:
//     stages x time of a stage + end of a tile + (split: 4 for the second kernel and the partial sums' way through memory at 5 TB/s)
// A stage takes 0.27 (256 x 256), 0.25 (256 x 128; it saves little once many pairs load), 0.74 (512 x 256 from codes) or 0.7 (256 x 256 from
// codes: the producers are what it waits for).  Results leave an SM at 26 bytes a clock, plus 1 us until the last have arrived.  Halved
// tiles come into question where all of them run at once.  Measured, us, halved or not / whole tiles: 446 x 768 x 768 forward 6.7 / 8.5,
// weight gradient 8.6 / 11.9; 1 x 4096 x 4096 forward in two halved parts 17.9, in four whole ones 12.7; step on 57,088 x 768 codes
// for 1000 outputs with a halved weight gradient 224, a whole one 202; 1024 x 1024 x 1024 forward split in two 12.4, not split 10.0.
Plan make_plan(int64_t rows_a, int64_t rows_b, int64_t contraction, bool codes) {
    const int64_t pairs = tcb::sm_count() / 2 > 0 ? tcb::sm_count() / 2 : 1, num_kb = (contraction + kBlockK - 1) / kBlockK;
    const int64_t ld_partial = (rows_b + 7) / 8 * 8;
    const double part = double(rows_a) * double(ld_partial) * 8.0 / 5e6;
    Plan best;
    double best_time = 0.0;
    for (int halved = 0; halved < 2; ++halved) {
        Plan p;
        p.tile_a = codes && !halved ? 512 : 256;
        p.tile_b = !codes && halved ? 128 : 256;
        p.tiles_a = (rows_a + p.tile_a - 1) / p.tile_a;
        p.tiles_b = (rows_b + p.tile_b - 1) / p.tile_b;
        p.num_kb = num_kb;
        p.ld_partial = ld_partial;
        const int64_t tiles = p.tiles_a * p.tiles_b;
        if (halved && tiles > pairs) break;
        const double stage = codes ? (halved ? 0.7 : 0.74) : (halved ? 0.25 : 0.27);
        const double store = double(p.tile_a / 2) * p.tile_b / 49400.0;   // us per byte of a result
        for (int64_t s = 1; s == 1 || (s <= pairs / tiles && s <= num_kb); ++s) {
            const double t = double((num_kb + s - 1) / s) * stage + 1.0 + store * (s > 1 ? 4.0 : 2.0) + (s > 1 ? 4.0 + double(s) * part : 0.0);
            if ((halved == 0 && s == 1) || t < best_time) {
                best_time = t;
                best = p;
                best.kb_per_split = int((num_kb + s - 1) / s);
                best.splits = int((num_kb + best.kb_per_split - 1) / best.kb_per_split);
            }
        }
    }
    return best;
}

int64_t weight_partial_bytes(int64_t M, int64_t N, int64_t K) {
    return (make_plan(N, K, M, true).partial_bytes(N) + 31) / 32 * 32;
}

// Parts of the column sums: at most one per CTA (a GPU has no more than one CTA per SM of these kernels) and row slice.
int64_t column_bytes(int64_t cols) { return int64_t(tcb::sm_count()) * ColumnShare(cols).slices * cols * 4; }

// Workspace of the backward pass: split sums of a product, then the parts of the column sums.
struct Columns {
    const uint16_t* dy = nullptr;
    int64_t ld = 0;
    float* parts = nullptr;
    uint16_t* out = nullptr;
};

int launch_add(const Plan& plan, const float* partial, int64_t rows, int64_t cols, const uint16_t* bias, uint16_t* out, const Columns& columns,
               int column_parts, int64_t num_columns, cudaStream_t st) {
    Parts a;
    a.partial = partial;
    a.splits = plan.splits;
    a.rows = plan.splits > 1 ? rows : 0;
    a.cols = cols;
    a.ld = plan.ld_partial;
    a.bias = bias;
    a.out = out;
    a.columns = columns.parts;
    a.column_parts = column_parts;
    a.column_blocks = columns.out ? int((num_columns + 31) / 32) : 0;
    a.num_columns = num_columns;
    a.column_out = columns.out;
    const int64_t most = int64_t(tcb::sm_count()) * 8;
    int64_t blocks = (a.rows * (plan.ld_partial / 4) + 255) / 256;
    if (blocks > most) blocks = most;
    if (blocks + a.column_blocks == 0) return TCB_OK;
    TCB_CUDA_TRY(tcb::launch_overlapped(add_parts_kernel, dim3(unsigned(blocks + a.column_blocks)), dim3(256), 0, st, a));
    return TCB_OK;
}

// A tensor map over a row-major [outer, inner] array with rows of `ld` elements.
int encode_map(const char* who, CUtensorMap* map, bool bytes, const void* base, int64_t inner, int64_t outer, int64_t ld, int box_inner,
               int box_outer) {
    EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return tcb::fail(TCB_ERR_CUDA, "%s: cuTensorMapEncodeTiled is not available from the driver", who);
    const cuuint64_t dims[2] = {cuuint64_t(inner), cuuint64_t(outer)};
    const cuuint64_t strides[1] = {cuuint64_t(ld) * (bytes ? 1 : 2)};
    const cuuint32_t box[2] = {cuuint32_t(box_inner), cuuint32_t(box_outer)}, estr[2] = {1, 1};
    const CUresult cr = encode(map, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
                               strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               bytes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return cr == CUDA_SUCCESS ? TCB_OK : tcb::fail(TCB_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed with %d", who, int(cr));
}

struct Operand {
    const void* base;
    int64_t rows, contraction, ld;
};

// `rows`: rows of the operand a CTA stages.
template <Source S>
int operand_map(const char* who, CUtensorMap* map, const Operand& o, int rows) {
    if (S == kContraction) return encode_map(who, map, false, o.base, o.contraction, o.rows, o.ld, kBlockK, rows);
    if (S == kRows) return encode_map(who, map, false, o.base, o.rows, o.contraction, o.ld, 64, kBlockK);
    return encode_map(who, map, true, o.base, o.rows, o.contraction, o.ld, rows, kBlockK);
}

template <Source A, Source B, int TB, int LOG2_G, bool HAS_ZP>
int launch_tiles(const char* who, const Operand& a, const Operand& b, Params& p, cudaStream_t st, int* grid) {
    using C = Config<B, TB>;
    CUtensorMap map_a, map_b;
    int rc = operand_map<A>(who, &map_a, a, kTileRows);
    if (rc == TCB_OK) rc = operand_map<B>(who, &map_b, b, C::kRowsB);
    if (rc != TCB_OK) return rc;
    const auto kernel = linear_kernel<A, B, TB, LOG2_G, HAS_ZP>;
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    TCB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
        TCB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(C::kSmem)));
        if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
    }
    const int pairs = tcb::sm_count() / 2 > 0 ? tcb::sm_count() / 2 : 1;
    *grid = 2 * (p.items < pairs ? p.items : pairs);
    TCB_CUDA_TRY(tcb::launch_overlapped(+kernel, dim3(*grid), dim3(C::kThreads), C::kSmem, st, map_a, map_b, p));
    return TCB_OK;
}

template <Source A, Source B, int LOG2_G, bool HAS_ZP>
int launch(const char* who, const Operand& a, const Operand& b, const uint16_t* scales, const uint8_t* zp, const uint16_t* bias, uint16_t* out,
           void* workspace, int64_t workspace_bytes, cudaStream_t st, const Columns& columns = Columns()) {
    const Plan plan = make_plan(a.rows, b.rows, a.contraction, B == kCodes);
    if (plan.tiles_a * plan.tiles_b * plan.splits > (int64_t(1) << 30)) return tcb::fail(TCB_ERR_TOO_LARGE, "%s: too many output tiles", who);
    if (plan.partial_bytes(a.rows) > workspace_bytes)
        return tcb::fail(TCB_ERR_BAD_ARG, "%s: the workspace holds %lld bytes, %lld are needed", who, (long long)workspace_bytes,
                         (long long)plan.partial_bytes(a.rows));
    Params p;
    p.rows_a = a.rows;
    p.rows_b = b.rows;
    p.bias = plan.splits > 1 ? nullptr : bias;
    p.out = out;
    p.partial = plan.splits > 1 ? static_cast<float*>(workspace) : nullptr;
    p.ld_partial = plan.ld_partial;
    p.columns = columns.dy;
    p.ld_columns = columns.ld;
    p.column_parts = columns.parts;
    p.scales = scales;
    p.zp = zp;
    p.contraction = a.contraction;
    p.tiles_a = int(plan.tiles_a);
    p.tiles_b = int(plan.tiles_b);
    p.tiles = p.tiles_a * p.tiles_b;
    p.tile_a = plan.tile_a;
    p.num_kb = int(plan.num_kb);
    p.kb_per_split = plan.kb_per_split;
    p.items = p.tiles * plan.splits;
    int rc = TCB_OK, grid = 0;
    if constexpr (B == kCodes) {
        rc = launch_tiles<A, B, 256, LOG2_G, HAS_ZP>(who, a, b, p, st, &grid);
    } else {
        rc = plan.tile_b == 128 ? launch_tiles<A, B, 128, LOG2_G, HAS_ZP>(who, a, b, p, st, &grid)
                                : launch_tiles<A, B, 256, LOG2_G, HAS_ZP>(who, a, b, p, st, &grid);
    }
    if (rc != TCB_OK) return rc;
    return launch_add(plan, p.partial, a.rows, b.rows, bias, out, columns, grid * ColumnShare(a.rows).slices, a.rows, st);
}

int check_sizes(const char* who, int64_t M, int64_t N, int64_t K) {
    const int64_t limit = (int64_t(1) << 31) - 1024;   // coordinates of the last tile stay within 32 bits
    if (M < 0 || N < 0 || K < 0) return tcb::fail(TCB_ERR_BAD_ARG, "%s: negative size", who);
    if (M > limit || N > limit || K > limit) return tcb::fail(TCB_ERR_TOO_LARGE, "%s: dimension beyond 2^31 - 1024", who);
    if (M > 0 && N > 0 && (K <= 0 || K % 8 != 0)) return tcb::fail(TCB_ERR_BAD_ARG, "%s: K = %lld must be a positive multiple of 8", who, (long long)K);
    return TCB_OK;
}

int check_operands(const char* who, const void* a, const void* b, const void* out, const void* bias, const void* workspace) {
    if (!a || !b || !out) return tcb::fail(TCB_ERR_BAD_ARG, "%s: null pointer", who);
    if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15)
        return tcb::fail(TCB_ERR_ALIGNMENT, "%s: operands must be 16-byte aligned", who);
    if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias)) & 1)
        return tcb::fail(TCB_ERR_ALIGNMENT, "%s: bias and output must be 2-byte aligned", who);
    if (reinterpret_cast<uintptr_t>(workspace) & 31)
        return tcb::fail(TCB_ERR_ALIGNMENT, "%s: the workspace must be 32-byte aligned", who);
    return TCB_OK;
}

int check_group(const char* who, int64_t K, int group_size) {
    if (!tcb::core_group_size_ok(group_size) && group_size != 128)
        return tcb::fail(TCB_ERR_GROUP_SIZE, "%s: group_size %d not in {16, 32, 64, 128}", who, group_size);
    if (K % group_size != 0)
        return tcb::fail(TCB_ERR_BAD_ARG, "%s: K = %lld must be a multiple of the group size %d", who, (long long)K, group_size);
    return TCB_OK;
}

}  // namespace

namespace tcb {
int take_linear_status(int* status) { return take_status(g_status, status); }
}  // namespace tcb

extern "C" int64_t tcb_linear_workspace(int64_t M, int64_t N, int64_t K, int gradients) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    if (gradients == 0) return make_plan(M, N, K, false).partial_bytes(M);
    const int64_t dx = gradients & 1 ? make_plan(M, K, N, false).partial_bytes(M) : 0;
    const int64_t rest = (gradients & 2 ? weight_partial_bytes(M, N, K) : 0) + (gradients & 4 ? column_bytes(N) : 0);
    return dx > rest ? dx : rest;
}

extern "C" int tcb_linear_forward(const uint16_t* x, const uint16_t* w, const uint16_t* bias_or_null, uint16_t* y, uint8_t* q_or_null,
                                  uint16_t* scales_or_null, int64_t M, int64_t N, int64_t K, int group_size, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
    const char* who = "tcb_linear_forward";
    int rc = check_sizes(who, M, N, K);
    if (rc == TCB_OK && q_or_null) rc = check_group(who, K, group_size);
    if (rc != TCB_OK || M == 0 || N == 0) return rc;
    rc = check_operands(who, x, w, y, bias_or_null, workspace);
    if (rc != TCB_OK) return rc;
    if (q_or_null) {
        if (!scales_or_null) return tcb::fail(TCB_ERR_BAD_ARG, "%s: codes without scales", who);
        rc = tcb_compress_sym(x, TCB_DT_BF16, M * K, group_size, nullptr, 0, reinterpret_cast<int8_t*>(q_or_null), scales_or_null, stream);
        if (rc != TCB_OK) return rc;
    }
    return launch<kContraction, kContraction, 0, false>(who, Operand{x, M, K, K}, Operand{w, N, K, K}, nullptr, nullptr, bias_or_null, y, workspace,
                                                        workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int tcb_linear_backward(const uint16_t* dy, int64_t ld_dy, const uint16_t* w_or_null, const uint8_t* q_or_null,
                                   const uint16_t* scales_or_null, const uint8_t* zp_or_null, uint16_t* dx_or_null, uint16_t* dw_or_null,
                                   uint16_t* db_or_null, int64_t M, int64_t N, int64_t K, int group_size, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
    const char* who = "tcb_linear_backward";
    int rc = check_sizes(who, M, N, K);
    if (rc == TCB_OK && (ld_dy < N || ld_dy % 8 != 0))
        rc = tcb::fail(TCB_ERR_BAD_ARG, "%s: rows of dy are %lld elements apart: a multiple of 8, at least N = %lld, is needed", who,
                       (long long)ld_dy, (long long)N);
    if (rc == TCB_OK && dw_or_null) rc = check_group(who, K, group_size);
    if (rc != TCB_OK || M == 0 || N == 0) return rc;
    if (dx_or_null) rc = check_operands(who, dy, w_or_null, dx_or_null, nullptr, workspace);
    if (rc == TCB_OK && dw_or_null) {
        if (!scales_or_null) return tcb::fail(TCB_ERR_BAD_ARG, "%s: null pointer", who);
        rc = check_operands(who, dy, q_or_null, dw_or_null, scales_or_null, workspace);
        // rows of dw are multiples of 32 bytes: aligned to 16 it is stored straight from the registers
        if (rc == TCB_OK && (reinterpret_cast<uintptr_t>(dw_or_null) & 15)) rc = tcb::fail(TCB_ERR_ALIGNMENT, "%s: dw must be 16-byte aligned", who);
    }
    if (rc == TCB_OK && db_or_null) rc = check_operands(who, dy, dy, db_or_null, nullptr, workspace);
    if (rc != TCB_OK) return rc;
    const int64_t dw_bytes = dw_or_null ? weight_partial_bytes(M, N, K) : 0;
    if (db_or_null && workspace_bytes < dw_bytes + column_bytes(N))
        return tcb::fail(TCB_ERR_BAD_ARG, "%s: the workspace holds %lld bytes, %lld are needed", who, (long long)workspace_bytes,
                         (long long)(dw_bytes + column_bytes(N)));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dx_or_null) {
        rc = launch<kContraction, kRows, 0, false>(who, Operand{dy, M, N, ld_dy}, Operand{w_or_null, K, N, K}, nullptr, nullptr, nullptr, dx_or_null,
                                                   workspace, workspace_bytes, st);
        if (rc != TCB_OK) return rc;
    }
    Columns columns;
    if (db_or_null) {
        columns.dy = dy;
        columns.ld = ld_dy;
        columns.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + dw_bytes);
        columns.out = db_or_null;
    }
    if (!dw_or_null) {
        if (!db_or_null) return TCB_OK;
        const ColumnShare share(N);
        const int64_t most = int64_t(tcb::sm_count()) * share.slices, runs = (M + 127) / 128;
        const int parts = int(runs < most ? runs : most);
        TCB_CUDA_TRY(tcb::launch_overlapped(column_sums_kernel, dim3(unsigned((int64_t(share.blocks) * parts + 7) / 8)), dim3(256), 0, st, dy, M, N, ld_dy,
                                            parts, columns.parts));
        return launch_add(Plan(), nullptr, 0, 0, nullptr, nullptr, columns, parts, N, st);
    }
    const Operand a{dy, N, M, ld_dy}, b{q_or_null, K, M, K};
    const uint16_t* scales = scales_or_null;
    uint16_t* dw = dw_or_null;
    const uint8_t* zp = zp_or_null;
    switch (group_size) {
    case 16: return zp ? launch<kRows, kCodes, 4, true>(who, a, b, scales, zp, nullptr, dw, workspace, workspace_bytes, st, columns)
                       : launch<kRows, kCodes, 4, false>(who, a, b, scales, zp, nullptr, dw, workspace, workspace_bytes, st, columns);
    case 32: return zp ? launch<kRows, kCodes, 5, true>(who, a, b, scales, zp, nullptr, dw, workspace, workspace_bytes, st, columns)
                       : launch<kRows, kCodes, 5, false>(who, a, b, scales, zp, nullptr, dw, workspace, workspace_bytes, st, columns);
    case 64: return zp ? launch<kRows, kCodes, 6, true>(who, a, b, scales, zp, nullptr, dw, workspace, workspace_bytes, st, columns)
                       : launch<kRows, kCodes, 6, false>(who, a, b, scales, zp, nullptr, dw, workspace, workspace_bytes, st, columns);
    default: return zp ? launch<kRows, kCodes, 7, true>(who, a, b, scales, zp, nullptr, dw, workspace, workspace_bytes, st, columns)
                       : launch<kRows, kCodes, 7, false>(who, a, b, scales, zp, nullptr, dw, workspace, workspace_bytes, st, columns);
    }
}
