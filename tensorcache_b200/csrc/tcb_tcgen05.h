// PTX helpers shared by the tensor-core kernels (tcgen05 / TMEM / TMA / mbarrier), the bounded barrier wait and
// the look-up of the tensor-map encoder.  Included by device code only; everything has internal linkage.
#pragma once
#include <atomic>

#include <cuda.h>
#include <cuda_bf16.h>

#include "tcb_common.h"

namespace {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// shared::cluster address of `addr` (a shared::cta address of this CTA) in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_to_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// Called by whole warps; their lanes meet first: an .aligned instruction must be reached by all of them together, and what comes
// before it (one lane's set-up, loops whose length differs from lane to lane) may have parted them.
__device__ __forceinline__ void cluster_sync_all() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
// Arrival on a barrier that may live in the other CTA of the pair (shared::cluster address).  The plain form: with
// .release.cluster on every arrival the arriving warp stalled for about a thousand clocks per stage.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// One poll of a barrier phase.  Cluster-scope acquire: most of these barriers take arrivals from the other CTA of
// the pair or from MMAs both CTAs take part in.  No suspend-time hint: it made no difference here.
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

constexpr long long kWaitBudgetClocks = 2000000000LL;  // ~1 s at 2 GHz

// Per source file (there is no device linking): 0 ok; otherwise (role << 8 | barrier id) of the first wait that ran out.
__device__ int g_status = 0;

// Bounded wait.  Returns false if the CTA pair is aborting (or this wait ran out).  `abort_peer` is the
// shared::cluster address of the other CTA's abort flag (0: no pair).
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t abort_peer, int who,
                                          long long budget = kWaitBudgetClocks) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if (clock64() - t0 > budget) {
            *abort_flag = 1;
            if (abort_peer) st_cluster_u32(abort_peer, 1u);
            atomicCAS(&g_status, 0, who);
            return false;
        }
    }
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
// Load into this CTA's shared memory that signals a barrier of either CTA of the pair
// (`cluster_bar` is a shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t cluster_bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(map), "r"(c0), "r"(c1), "r"(cluster_bar)
        : "memory");
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Arrival on the barrier at offset `bar` of BOTH CTAs of the pair once every MMA this thread has issued so far has completed.
__device__ __forceinline__ void umma_commit_both(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(uint16_t(3))
                 : "memory");
}

// One lane of the warp.  The issuing warp stays converged and only the tensor-core instructions are predicated on this:
// addresses and descriptors then live in uniform registers, where these instructions want them.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Index of this warp in the block, as a value the compiler knows to be the same in all lanes.
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0); }

// The lanes meet first, as above: the stores of the columns before leave out lanes whose rows lie outside the output.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// Shared-memory operand descriptor: K-major, 128-byte swizzle, rows of 128 bytes, 8-row groups 1024 bytes apart.
// Low word: start address in 16-byte units (14 bits) and the (unused) leading byte offset 1 at bit 16; high word: stride
// byte offset 1024 >> 4, descriptor version 1 (bit 46 of the 64), layout type 2 = 128-byte swizzle (bits 61..63).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t smem_desc_lo(uint32_t smem_addr) { return ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16); }

// (v - base) * scale of two numbers, as bf16.
__device__ __forceinline__ uint32_t decode_pair(uint32_t v0, uint32_t v1, float minus_base, float scale) {
    uint32_t r;
    asm("{\n\t.reg .b64 v, m, s;\n\t.reg .f32 lo, hi;\n\t"
        "mov.b64 v, {%1, %2};\n\tmov.b64 m, {%3, %3};\n\tmov.b64 s, {%4, %4};\n\t"
        "add.rn.f32x2 v, v, m;\n\t"
        "mul.rn.f32x2 v, v, s;\n\t"
        "mov.b64 {lo, hi}, v;\n\t"
        "cvt.rn.satfinite.bf16x2.f32 %0, hi, lo;\n\t}"
        : "=r"(r)
        : "r"(v0), "r"(v1), "f"(minus_base), "f"(scale));
    return r;
}

// 16 codes of one group -> 16 bf16 values, written as two 16-byte pieces of the 128-byte-swizzled operand row.
//
// A byte permute puts the code into the mantissa of 2^15; minus (2^15 + zero point) it is the whole number q - zp, and times the
// scale the numbers of the decode kernels: both steps are exact (9 x 8 significant bits), the conversion rounds once.  Two values at a
// time, so that they take as many instructions as one FMA per value with -(2^15 + zp) * scale as its addend, which overflows
// from scales of 2^113 on (16384 x 4096 x 4096 forward and weight gradient 370 + 372 us, with the FMAs 370 + 370).
// A product past the largest bf16 number stays at it, where the decode kernels give infinity: 127 steps of the scale
// that the lowest bf16 number gets are beyond it, and a padding row of that number must add 0 to a sum that multiplies it with 0.
// An infinite scale becomes a NaN first, so that this hides none.
template <bool HAS_ZP>
__device__ __forceinline__ void convert16(uint4 c, uint32_t sz_word, uint8_t* piece0, uint8_t* piece1) {
    uint32_t w[4] = {c.x, c.y, c.z, c.w};
    const float s = __uint_as_float(sz_word & 0xFFFF0000u), scale = __fmaf_rn(s, 0.0f, s);
    float base;
    if (HAS_ZP) {
        base = __uint_as_float(__byte_perm(sz_word, 0x47000000u, 0x7604));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] ^= 0x80808080u;
        base = __uint_as_float(0x47008000u);
    }
    const uint32_t magic = 0x47000000u;
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o[2 * i] = decode_pair(__byte_perm(w[i], magic, 0x7604), __byte_perm(w[i], magic, 0x7614), -base, scale);
        o[2 * i + 1] = decode_pair(__byte_perm(w[i], magic, 0x7624), __byte_perm(w[i], magic, 0x7634), -base, scale);
    }
    *reinterpret_cast<uint4*>(piece0) = make_uint4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<uint4*>(piece1) = make_uint4(o[4], o[5], o[6], o[7]);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint16_t f32_to_bf16_bits(float v) {
    __nv_bfloat16 b = __float2bfloat16_rn(v);
    return *reinterpret_cast<uint16_t*>(&b);
}

// ---------------------------------------------------------------------- epilogue stores
//
// A warp holds 32 columns of 32 consecutive output rows, one row per lane.  Rows whose start is a multiple of 32 (16) bytes
// take 32-byte (16-byte) stores straight from the registers; any other row length goes through a small buffer of
// the warp's own, 8 columns at a time, so that 8 neighbouring lanes write one row (a lane of its own per row would touch
// 32 sectors with every 2-byte store).
enum StoreMode { kStaged, kVec16, kVec32 };
constexpr uint32_t kStoreStageBytes = 32 * 9 * 4;   // per warp: rows of 9 words, so that neither side meets in a bank

__device__ __forceinline__ StoreMode store_mode(const void* out, int64_t ld, const void* bias) {
    const uintptr_t o = reinterpret_cast<uintptr_t>(out);
    if (reinterpret_cast<uintptr_t>(bias) & 3) return kStaged;
    return (ld % 16 == 0 && (o & 31) == 0) ? kVec32 : (ld % 8 == 0 && (o & 15) == 0) ? kVec16 : kStaged;
}

// Lane l stores bf16(v + bias) to out[row0 + l, col0 .. col0 + 31] as far as that lies inside [rows, cols].  Called by the
// whole warp; `stage` is the warp's buffer (kStaged only).
__device__ __forceinline__ void store_32x32(uint16_t* out, int64_t ld, int64_t row0, int64_t rows, int64_t col0, int64_t cols,
                                            const uint16_t* bias, const uint32_t (&v)[32], StoreMode mode, uint32_t* stage) {
    const int lane = threadIdx.x & 31;
    if (mode != kStaged) {
        if (row0 + lane >= rows) return;
        uint16_t* dst = out + (row0 + lane) * ld + col0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float a = __uint_as_float(v[16 * h + 2 * i]), b = __uint_as_float(v[16 * h + 2 * i + 1]);
                if (bias && col0 + 16 * h + 2 * i < cols) {
                    const uint32_t bb = __ldg(reinterpret_cast<const uint32_t*>(bias + col0) + 8 * h + i);
                    a += __uint_as_float(bb << 16);
                    b += __uint_as_float(bb & 0xFFFF0000u);
                }
                w[i] = pack_bf16(a, b);
            }
            if (mode == kVec32) {   // cols is a multiple of 16
                if (col0 + 16 * h < cols) st_global_v8(dst + 16 * h, w);
            } else {                // a multiple of 8
                if (col0 + 16 * h < cols) *reinterpret_cast<uint4*>(dst + 16 * h) = make_uint4(w[0], w[1], w[2], w[3]);
                if (col0 + 16 * h + 8 < cols) *reinterpret_cast<uint4*>(dst + 16 * h + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            }
        }
        return;
    }
    // the bias joins before the one rounding, so the buffer holds fp32
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) stage[lane * 9 + i] = v[8 * g + i];
        __syncwarp();
        const int64_t col = col0 + 8 * g + (lane & 7);
        if (col >= cols) continue;
        const float b = bias ? __uint_as_float(uint32_t(bias[col]) << 16) : 0.0f;
        int64_t row = row0 + (lane >> 3);
        uint16_t* dst = out + row * ld + col;
        const uint32_t* src = stage + (lane >> 3) * 9 + (lane & 7);
#pragma unroll
        for (int i = 0; i < 8; ++i, row += 4, dst += 4 * ld)
            if (row < rows) *dst = f32_to_bf16_bits(__uint_as_float(src[36 * i]) + b);
    }
}

// Lane a, piece b becomes lane b, piece a within groups of four lanes.
__device__ __forceinline__ void transpose_pieces(uint32_t (&u)[4][8]) {
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int b = 0; b < 4; b += 2) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? u[b][i] : u[b + 1][i], 1);
            if (odd) u[b][i] = got;
            else u[b + 1][i] = got;
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, high ? u[b][i] : u[b + 2][i], 2);
            if (high) u[b][i] = got;
            else u[b + 2][i] = got;
        }
    }
}

// Stores 32 tensor-memory columns from `taddr` as fp32 (lanes: rows row0 ...); ld a multiple of 8, out 32-byte aligned, columns up to
// ld may be written.  Four neighbouring lanes exchange 32-byte pieces first, so that an instruction writes eight rows of 128
// contiguous bytes (partial sums of 2048 x 1024 over 8192: 38 us with the second kernel, 42 without).  For bf16 results the same
// exchange gains nothing and holds the accumulator longer (8192 x 14336 x 4096 in MXFP4: 216 us with it, 195 without).
__device__ __forceinline__ void store_32x32_f32(uint32_t taddr, float* out, int64_t ld, int64_t row0, int64_t rows, int64_t col0) {
    const int lane = threadIdx.x & 31;
    uint32_t v[32], u[4][8];
    tmem_ld32(taddr, v);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) u[i >> 3][i & 7] = v[i];
    transpose_pieces(u);
    const int64_t col = col0 + 8 * (lane & 3);
    int64_t row = row0 + (lane & 28);
    float* dst = out + row * ld + col;
#pragma unroll
    for (int r = 0; r < 4; ++r, ++row, dst += ld)
        if (row < rows && col < ld) st_global_v8(dst, u[r]);
}

// ---------------------------------------------------------------------- host

// Reads and clears a file's status word (the stream has been synchronised).
inline int take_status(const int& symbol, int* status) {
    *status = 0;
    TCB_CUDA_TRY(cudaMemcpyFromSymbol(status, symbol, sizeof(int)));
    if (*status) {
        const int zero = 0;
        TCB_CUDA_TRY(cudaMemcpyToSymbol(symbol, &zero, sizeof(int)));
    }
    return TCB_OK;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The encoder, with the current device's context bound to this thread: the encoder is a driver call, and a thread that
// has made no CUDA call of its own yet (a backward pass runs on one of the autograd engine's) has no context.
EncodeTiledFn encode_tiled_fn() {
    static std::atomic<EncodeTiledFn> cached{nullptr};
    static thread_local int bound = -1;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
    if (dev != bound) {
        if (cudaSetDevice(dev) != cudaSuccess) return nullptr;
        bound = dev;
    }
    EncodeTiledFn fn = cached.load(std::memory_order_acquire);
    if (!fn) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess &&
            qres == cudaDriverEntryPointSuccess) {
            fn = reinterpret_cast<EncodeTiledFn>(sym);
            cached.store(fn, std::memory_order_release);
        }
    }
    return fn;
}

}  // namespace
