// MXFP4 product for few rows of x (up to 32: single tokens, small batches), bound by reading the weight once.
//
//     out[m, n] = bf16( sum_k x[m, k] w[n, k] + bias[n] )
//
// The weight is the M side of the tensor-core tile: a CTA owns 128 rows of w, the rows of x are its 16 or 32 columns
// (tcgen05.mma kind::mxf4, one CTA, M 128).  x is quantised by the CTA itself, straight into the operand layout in
// shared memory, while the first tiles of w are on their way: no launch and no memory traffic of its own.  The sum over
// K is split over a cluster of 1 to 8 CTAs, so that a weight with few rows still occupies the GPU; the parts meet in shared
// memory over the cluster and are added in a fixed order.
//
// Warps: 0 TMA (one lane; then quantising), 1 MMA issue and tensor memory, all quantise, 4-7 epilogue.
// Waits are bounded as in the fused dequantising product; the status word is read by tcb_fused_dequant_linear_check().
#include "tcb_mxfp4.h"
#include "tcb_tcgen05.h"

namespace {

constexpr int kThreads = 256;
constexpr int kTileRows = 128;                        // rows of w per CTA
constexpr int kBlockK = 256;                          // values of K per stage
constexpr uint32_t kCodeBytes = kTileRows * 128;      // 16 KB
constexpr uint32_t kScaleBytes = 1024;                // 128 rows x 8 blocks
constexpr uint32_t kStageBytes = kCodeBytes + kScaleBytes;
constexpr uint32_t kMaxSmem = 232448;
constexpr uint32_t kTmemCols = 128;                   // accumulator in [0, 32), two sets of scales (8 + 8 columns) from 32
constexpr uint32_t kScaleCols = 32;

struct Params {
    const void* x;
    const uint16_t* bias;
    uint16_t* out;
    int64_t N, K;
    int M, num_kb, kb_per_cta, stages;
};

// x, w: E2M1; scales: E8M0; M = 128; K = 64.  sf: which half of a 32-bit word of scales (0 or 2).
template <int COLS>
__device__ __forceinline__ constexpr uint32_t inst_desc(uint32_t sf) {
    return (sf << 4) | (1u << 7) | (1u << 10) | (uint32_t(COLS >> 3) << 17) | (1u << 23) | (1u << 27) | (sf << 29);
}

template <int COLS>
__device__ __forceinline__ void umma_mxf4_x4(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t sfa, uint32_t sfb, uint32_t accumulate_first) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t.reg .b64 a, b;\n\t.reg .b32 al, bl, sa, sb;\n\t"
        "setp.ne.b32 p, %8, 0;\n\t"
        "setp.eq.b32 t, %8, %8;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %4, [%6], [%7], p;\n\t"
        "add.u32 al, %1, 2;\n\tadd.u32 bl, %2, 2;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %5, [%6], [%7], t;\n\t"
        "add.u32 al, %1, 4;\n\tadd.u32 bl, %2, 4;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
        "add.u32 sa, %6, 4;\n\tadd.u32 sb, %7, 4;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %4, [sa], [sb], t;\n\t"
        "add.u32 al, %1, 6;\n\tadd.u32 bl, %2, 6;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %5, [sa], [sb], t;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(inst_desc<COLS>(0)), "r"(inst_desc<COLS>(2)), "r"(sfa), "r"(sfb), "r"(accumulate_first)
        : "memory");
}

__device__ __forceinline__ void copy_scales(uint32_t d_tmem, uint32_t smem_addr) {
    const uint32_t lo = ((smem_addr & 0x3FFFFu) >> 4) | ((128u >> 4) << 16), hi = (128u >> 4) | (1u << 14);
    asm volatile(
        "{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\t"
        "tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t}" ::"r"(d_tmem),
        "r"(lo), "r"(hi)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
    return v;
}

// A CTA's part of x: blocks [b0, b0 + 8 stages) of rows 0..M-1 as codes (rows of 128 bytes, 128-byte swizzle, COLS rows a
// stage) and scales (tile order, 512 bytes per four blocks).  Blocks past the end of a row are written as zeros: the tensor
// core multiplies them with the zeros that the TMA fills in, and whatever else lies there could be a NaN.
template <int COLS, typename T>
__device__ __forceinline__ void quantize_rows(const Params& p, int64_t b0, int blocks, uint8_t* codes, uint8_t* scales) {
    const int64_t bpr = p.K / 32;
    const T* x = static_cast<const T*>(p.x);
    constexpr int kAhead = sizeof(T) == 2 ? 4 : 2;   // blocks of a thread in flight
    const int total = p.M * blocks;
    for (int i0 = threadIdx.x; i0 < total; i0 += kAhead * kThreads) {
        Block32<T> v[kAhead];
        int row[kAhead], blk[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = i0 + j * kThreads;
            row[j] = i / blocks;
            blk[j] = i - row[j] * blocks;
            if (i < total && b0 + blk[j] < bpr) v[j].load(x + (int64_t(row[j]) * bpr + b0 + blk[j]) * 32);
            else v[j].zero();       // a block of zeros has scale byte and codes 0
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (i0 + j * kThreads >= total) break;
            uint4 c;
            const uint32_t byte = encode_block(v[j], c);
            *reinterpret_cast<uint4*>(codes + (blk[j] >> 3) * (COLS * 128) + row[j] * 128 + (((blk[j] & 7) ^ (row[j] & 7)) * 16)) = c;
            scales[(blk[j] >> 2) * 512 + row[j] * 16 + (blk[j] & 3)] = uint8_t(byte);
        }
    }
}

template <int COLS, typename T>
__global__ void __launch_bounds__(kThreads)
mxfp4_few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_ws, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    // ring of w (codes 16 KB + scales 1 KB a stage, codes first), codes of x, scales of x, barriers; the partial sums take
    // the place of the ring at the end
    const int S = p.stages;
    uint8_t* ring = smem;
    uint8_t* x_codes = ring + S * kStageBytes;
    uint8_t* x_scales = x_codes + p.kb_per_cta * (COLS * 128);
    uint64_t* bars = reinterpret_cast<uint64_t*>(x_scales + p.kb_per_cta * 1024);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int FULL = 0, EMPTY = S, DONE = 2 * S;

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const uint32_t bar0 = smem_u32(bars), ring0 = smem_u32(ring), scale0 = ring0 + uint32_t(S) * kCodeBytes;
    auto bar = [&](int id) { return bar0 + 8u * uint32_t(id); };
    const uint32_t rank = cluster_ctarank(), parts = gridDim.y;     // the cluster spans the whole y dimension
    const int tile = int(blockIdx.x);
    const int kb0 = int(rank) * p.kb_per_cta;
    const int my_kb = p.num_kb - kb0 < p.kb_per_cta ? p.num_kb - kb0 : p.kb_per_cta;   // at least 1

    if (threadIdx.x == 0) {
        prefetch_map(&map_w);
        prefetch_map(&map_ws);
        for (int s = 0; s < S; ++s) {
            mbar_init(bar(FULL + s), 1);
            mbar_init(bar(EMPTY + s), 1);
        }
        mbar_init(bar(DONE), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcb::await_predecessor();
    if (threadIdx.x == 0) {
        // the first tiles of w, before anything else
        for (int s = 0; s < S && s < my_kb; ++s) {
            mbar_arrive_expect_tx(bar(FULL + s), kStageBytes);
            tma_load_2d(ring0 + uint32_t(s) * kCodeBytes, &map_w, (kb0 + s) * 128, tile * kTileRows, bar(FULL + s));
            tma_load_2d(scale0 + uint32_t(s) * kScaleBytes, &map_ws, (kb0 + s) * 128, tile, bar(FULL + s));
        }
    }
    quantize_rows<COLS, T>(p, int64_t(kb0) * 8, my_kb * 8, x_codes, x_scales);
    fence_proxy_async();   // the codes and scales of x become visible to the tensor core
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // ---------------------------------------------------------------- TMA, the rest of w
        if (lane == 0) {
            bool ok = true;
            for (int kb = S; ok && kb < my_kb; ++kb) {
                const int s = kb % S;
                ok = mbar_wait(bar(EMPTY + s), uint32_t(kb / S - 1) & 1, abort_flag, 0u, (1 << 8) | (EMPTY + s));
                if (!ok) break;
                mbar_arrive_expect_tx(bar(FULL + s), kStageBytes);
                tma_load_2d(ring0 + uint32_t(s) * kCodeBytes, &map_w, (kb0 + kb) * 128, tile * kTileRows, bar(FULL + s));
                tma_load_2d(scale0 + uint32_t(s) * kScaleBytes, &map_ws, (kb0 + kb) * 128, tile, bar(FULL + s));
            }
            if (!ok) {   // aborting: copies still in flight land in this CTA's shared memory within microseconds
                const long long t0 = clock64();
                while (clock64() - t0 < 4000000LL) __nanosleep(1000);
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issue
        const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
        const bool elected = elect_one();
        const uint32_t xc0 = smem_u32(x_codes), xs0 = smem_u32(x_scales);
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int kb = 0; kb < my_kb; ++kb) {
            ok = __all_sync(0xffffffffu, mbar_wait(bar(FULL + s), ph, abort_flag, 0u, (2 << 8) | (FULL + s)));
            if (!ok) break;
            tc_fence_after();
            if (elected) {
                const uint32_t ta = tmem + kScaleCols + 16u * (kb & 1), tb = ta + 8u;
                const uint32_t sa = scale0 + uint32_t(s) * kScaleBytes, sb = xs0 + uint32_t(kb) * 1024u;
                copy_scales(ta, sa);
                copy_scales(tb, sb);
                copy_scales(ta + 4, sa + 512);
                copy_scales(tb + 4, sb + 512);
                umma_mxf4_x4<COLS>(tmem, smem_desc_lo(ring0 + uint32_t(s) * kCodeBytes), smem_desc_lo(xc0 + uint32_t(kb) * (COLS * 128)), ta, tb,
                                   kb > 0 ? 1u : 0u);
                umma_commit(bar(EMPTY + s));
            }
            __syncwarp();
            if (++s == S) { s = 0; ph ^= 1; }
        }
        if (ok && elected) umma_commit(bar(DONE));
        __syncwarp();
    } else if (warp >= 4) {
        // ---------------------------------------------------------------- sums of this CTA: one row of w per lane
        const bool ok = __all_sync(0xffffffffu, mbar_wait(bar(DONE), 0, abort_flag, 0u, (4 << 8) | DONE));
        if (ok) {
            tc_fence_after();
            const int quad = warp & 3;
            uint32_t v[32];
            tmem_ld32(tmem_base + (uint32_t(quad * 32) << 16), v);
            tmem_ld_wait();
            const int r = quad * 32 + lane;
            if (parts == 1) {
                const int64_t n = int64_t(tile) * kTileRows + r;
                if (n < p.N) {
                    const float b = p.bias ? __uint_as_float(uint32_t(p.bias[n]) << 16) : 0.0f;
#pragma unroll
                    for (int m = 0; m < COLS; ++m)
                        if (m < p.M) p.out[int64_t(m) * p.N + n] = f32_to_bf16_bits(__uint_as_float(v[m]) + b);
                }
            } else {
                // every load of the ring has been consumed by the MMAs that are done
                float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
                for (int m = 0; m < COLS; ++m)
                    if (m < p.M) sums[m * kTileRows + r] = __uint_as_float(v[m]);
            }
        }
    }

    __syncwarp();
    if (parts > 1) {
        cluster_sync_all();   // every CTA's sums are written (or it has given up)
        const int rows_each = kTileRows / int(parts), first = int(rank) * rows_each;
        const uint32_t mine = smem_u32(ring);
        if (!*abort_flag)
            for (int i = threadIdx.x; i < p.M * rows_each; i += kThreads) {
                const int m = i / rows_each, r = first + i - m * rows_each;
                const int64_t n = int64_t(tile) * kTileRows + r;
                if (n >= p.N) continue;
                float sum = 0.0f;
                for (uint32_t c = 0; c < parts; ++c) sum += ld_cluster_f32(map_to_cta(mine + uint32_t(m * kTileRows + r) * 4u, c));
                if (p.bias) sum += __uint_as_float(uint32_t(p.bias[n]) << 16);
                p.out[int64_t(m) * p.N + n] = f32_to_bf16_bits(sum);
            }
        cluster_sync_all();   // nobody leaves while its sums may still be read
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    }
}

// Shape of a launch; stages == 0: this kernel does not take the sizes.
//
// Rules and what they were measured on (us, consecutive calls on different weights in a graph; rows of x x rows of w x K):
//   this kernel against tiles of 256 rows of x after a quantisation of their own
//     1 x 4096 x 4096: 5.5 / 10.4    1 x 14336 x 4096: 9.6 / 15.4    1 x 4096 x 14336: 9.8 / 25.4    1 x 28672 x 8192: 29.2 / 41.7
//     1 x 128256 x 4096: 60.7 / 71.2   16 x 14336 x 4096: 12.4 / 14.1   32 x 4096 x 4096: 7.3 / 11.0   32 x 14336 x 4096: 14.6 / 12.9
//     the last because every CTA quantises all of its K for every row: above 16 rows only where that is at most 8 stages.  Up to 16
//     rows always, although several waves of CTAs pay for that too: 16 x 28672 x 8192: 41.3 / 35.6, 16 x 128256 x 4096: 82.2 / 69.4
//   K split over a cluster or not   1 x 4096 x 4096: 4.6 / 7.0     1 x 1024 x 4096: 3.7 / 6.8
//   ring: as deep as it goes where every CTA has an SM to itself (1 x 14336 x 4096 9.1, with room for a second CTA 8.2, but 1 x 4096 x
//     4096 4.6 / 4.9).  With more tiles than SMs it leaves room for a second CTA as long as that keeps four stages: up to 16 rows
//     of x take 3 KB a stage of K, so up to K = 3584.  Beyond that four stages stay and one CTA runs per SM.
struct Shape {
    int cols, parts, kb_per_cta, stages;
    uint32_t smem;
};

Shape few_rows_shape(int64_t M, int64_t N, int64_t K) {
    Shape s{M <= 16 ? 16 : 32, 1, 0, 0, 0};
    const int64_t tiles = (N + kTileRows - 1) / kTileRows, num_kb = (K + kBlockK - 1) / kBlockK;
    if (M > 32 || num_kb > 4096) return s;
    // split K as long as all CTAs run at once on SMs of their own and a part keeps at least two stages
    while (s.parts < 8 && 2 * tiles * s.parts <= tcb::sm_count() && num_kb >= 4 * s.parts) s.parts *= 2;
    int64_t per = (num_kb + s.parts - 1) / s.parts;
    while (s.parts > 1 && per * (s.parts - 1) >= num_kb) {   // the last part would be empty
        s.parts /= 2;
        per = (num_kb + s.parts - 1) / s.parts;
    }
    if (M > 16 && per > 8) return s;
    s.kb_per_cta = int(per);
    const uint32_t fixed = uint32_t(per) * (s.cols * 128 + 1024) + 1024 /* alignment */ + 256 /* barriers */;
    const uint32_t room = tiles * s.parts <= tcb::sm_count() ? kMaxSmem : kMaxSmem / 2 - 1024;
    int stages = int(per < 12 ? per : 12);
    while (stages > 4 && fixed + stages * kStageBytes > room) --stages;
    while (stages > 1 && fixed + stages * kStageBytes > kMaxSmem) --stages;
    if (fixed + stages * kStageBytes > kMaxSmem) return s;
    s.stages = stages;
    s.smem = fixed + stages * kStageBytes;
    return s;
}

template <int COLS, typename T>
int launch(const char* who, const Shape& s, int64_t tiles, const CUtensorMap& map_w, const CUtensorMap& map_ws, const Params& p, cudaStream_t st) {
    const auto kernel = mxfp4_few_rows_kernel<COLS, T>;
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    TCB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
        TCB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kMaxSmem)));
        if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(tiles), unsigned(s.parts));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = s.smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = unsigned(s.parts);
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, map_w, map_ws, p);
    return e == cudaSuccess ? TCB_OK : tcb::cuda_fail(e, who);
}

template <int COLS>
int launch_typed(const char* who, int dtype, const Shape& s, int64_t tiles, const CUtensorMap& map_w, const CUtensorMap& map_ws, const Params& p,
                 cudaStream_t st) {
    switch (dtype) {
    case TCB_DT_BF16: return launch<COLS, __nv_bfloat16>(who, s, tiles, map_w, map_ws, p, st);
    case TCB_DT_F16: return launch<COLS, __half>(who, s, tiles, map_w, map_ws, p, st);
    default: return launch<COLS, float>(who, s, tiles, map_w, map_ws, p, st);
    }
}

}  // namespace

namespace tcb {

int take_mxfp4_few_status(int* status) { return take_status(g_status, status); }

bool mxfp4_few_rows(int64_t M, int64_t N, int64_t K) { return few_rows_shape(M, N, K).stages > 0; }

// Arguments have been checked by tcb_mxfp4_linear; the maps describe w in boxes of 128 rows.
int launch_mxfp4_few_rows(const char* who, const void* x, int dtype, const CUtensorMap& map_w, const CUtensorMap& map_ws, const uint16_t* bias,
                          uint16_t* out, int64_t M, int64_t N, int64_t K, cudaStream_t st) {
    const Shape s = few_rows_shape(M, N, K);
    const int64_t tiles = (N + kTileRows - 1) / kTileRows;
    Params p;
    p.x = x;
    p.bias = bias;
    p.out = out;
    p.N = N;
    p.K = K;
    p.M = int(M);
    p.num_kb = int((K + kBlockK - 1) / kBlockK);
    p.kb_per_cta = s.kb_per_cta;
    p.stages = s.stages;
    return s.cols == 16 ? launch_typed<16>(who, dtype, s, tiles, map_w, map_ws, p, st) : launch_typed<32>(who, dtype, s, tiles, map_w, map_ws, p, st);
}

}  // namespace tcb
