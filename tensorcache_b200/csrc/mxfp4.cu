// Microscaled 4-bit floating point (MXFP4): blocks of 32 values along the last dimension, E2M1 elements, one
// power-of-two scale (E8M0 byte) per block.
//
//     byte  = max(exponent field of max|x| - 2, 0)        the scale is 2^(byte - 127), so max|x| / scale is in [4, 8)
//     code  = E2M1 nearest to x / scale, ties to even, magnitudes above 6 become 6
//     value = code * 2^(byte - 127)                        exact in bf16 (two significant bits)
//
// The exponent field is that of fp32.  Values that are not finite count as 0, as in the int8 codecs.  A scale byte
// of 255 (never written here) decodes to NaN.
//
// Codes: [rows, cols / 2] bytes, element 2i in the low half.  Scales: the order in which the tensor cores read them,
// tiles of 128 rows x 4 blocks (512 bytes), tile (r / 128, block / 4) row-major; inside a tile the byte of row r and
// block b sits at (r % 32) * 16 + (r % 128) / 32 * 4 + b % 4.  Rows and blocks that pad the last tiles hold 0.
//
// Both kernels are bound by HBM: bf16 in, 2 + 0.5 + 1/32 bytes a value.  One thread block owns one scale tile (128
// rows x 128 columns): thread (row = t / 4, block = t % 4) takes rows row, row + 32, row + 64 and row + 96, so a warp
// reads 8 rows x 256 contiguous bytes with 8 loads of 32 bytes a thread in flight, and the 512 scale bytes of the tile
// leave as contiguous 16-byte pieces after a 4 x 4 byte transpose over four lanes.
#include "tcb_mxfp4.h"

namespace {

constexpr int kThreads = 128;
constexpr int kTileRows = 128, kTileCols = 128;

template <typename T>
__global__ void __launch_bounds__(kThreads)
quantize_mxfp4_kernel(const T* __restrict__ x, int64_t rows, int64_t blocks_per_row, int64_t tiles_k, uint8_t* __restrict__ codes,
                      uint8_t* __restrict__ scales) {
    tcb::await_predecessor();
    constexpr int kAhead = sizeof(T) == 2 ? 4 : 2;   // rows of a thread loaded at once (fp32: 64 registers either way)
    const int64_t tile_r = blockIdx.x / tiles_k, tile_k = blockIdx.x % tiles_k;
    const int kb = threadIdx.x & 3, r0 = threadIdx.x >> 2;
    const int64_t blk = tile_k * 4 + kb;
    const bool col_ok = blk < blocks_per_row;
    uint32_t packed = 0;   // scale bytes of this thread's four rows
#pragma unroll
    for (int i0 = 0; i0 < 4; i0 += kAhead) {
        Block32<T> b[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t row = tile_r * kTileRows + (i0 + i) * 32 + r0;
            if (col_ok && row < rows) b[i].load(x + (row * blocks_per_row + blk) * 32);
            else b[i].zero();
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t row = tile_r * kTileRows + (i0 + i) * 32 + r0;
            uint4 c;
            const uint32_t byte = encode_block(b[i], c);
            if (col_ok && row < rows) *reinterpret_cast<uint4*>(codes + (row * blocks_per_row + blk) * 16) = c;
            packed |= byte << (8 * (i0 + i));
        }
    }
    // 4 x 4 byte transpose over the four lanes of a row: lane kb ends up with the four blocks of row 32 kb + r0
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t other = __shfl_sync(0xffffffffu, packed, (threadIdx.x & 28) | j);
        mine |= ((other >> (8 * kb)) & 255u) << (8 * j);
    }
    *reinterpret_cast<uint32_t*>(scales + int64_t(blockIdx.x) * 512 + r0 * 16 + kb * 4) = mine;
}

// Eight codes -> eight bf16 values times 2^(byte - 127).  The magnitudes come from two byte tables (byte permutes
// that index with the three magnitude bits), the packed product is exact.
__device__ __forceinline__ void decode8(uint32_t c, __nv_bfloat162 scale, uint32_t* o) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t q = h ? c >> 16 : c;
        const uint32_t sel = q & 0x7777u;
        const uint32_t hi = __byte_perm(0x3f3f3f00u, 0x40404040u, sel);   // 0 .5 1 1.5 | 2 3 4 6, high bytes
        const uint32_t lo = __byte_perm(0xc0800000u, 0xc0804000u, sel);   // low bytes
        const uint32_t v0 = __byte_perm(lo, hi, 0x5140) | ((q & 0x8u) << 12) | ((q & 0x80u) << 24);
        const uint32_t v1 = __byte_perm(lo, hi, 0x7362) | ((q & 0x800u) << 4) | ((q & 0x8000u) << 16);
        const __nv_bfloat162 p0 = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v0), scale);
        const __nv_bfloat162 p1 = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v1), scale);
        o[2 * h] = *reinterpret_cast<const uint32_t*>(&p0);
        o[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&p1);
    }
}

__global__ void __launch_bounds__(kThreads)
dequantize_mxfp4_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows, int64_t blocks_per_row,
                        int64_t tiles_k, uint16_t* __restrict__ out) {
    tcb::await_predecessor();
    const int64_t tile_r = blockIdx.x / tiles_k, tile_k = blockIdx.x % tiles_k;
    const int kb = threadIdx.x & 3, r0 = threadIdx.x >> 2;
    const int64_t blk = tile_k * 4 + kb;
    const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(scales + int64_t(blockIdx.x) * 512 + r0 * 16 + kb * 4));
    uint32_t packed = 0;   // scale bytes of this lane's block in rows r0, r0 + 32, r0 + 64, r0 + 96
#pragma unroll
    for (int j = 0; j < 4; ++j) packed |= ((__shfl_sync(0xffffffffu, word, (threadIdx.x & 28) | j) >> (8 * kb)) & 255u) << (8 * j);
    if (blk >= blocks_per_row) return;
    uint4 c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = tile_r * kTileRows + i * 32 + r0;
        c[i] = row < rows ? __ldcs(reinterpret_cast<const uint4*>(codes + (row * blocks_per_row + blk) * 16)) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = tile_r * kTileRows + i * 32 + r0;
        if (row >= rows) continue;
        const uint32_t byte = (packed >> (8 * i)) & 255u;
        // 2^(byte - 127) as bf16: the exponent field, except 2^-127 (subnormal) and NaN
        const uint32_t sbits = byte == 0u ? 0x0040u : byte == 255u ? 0x7fffu : byte << 7;
        const uint32_t s2 = sbits | (sbits << 16);
        const __nv_bfloat162 scale = *reinterpret_cast<const __nv_bfloat162*>(&s2);
        const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
        uint16_t* dst = out + (row * blocks_per_row + blk) * 32;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint32_t o[8];
            decode8(w[2 * k], scale, o);
            decode8(w[2 * k + 1], scale, o + 4);
            tcb::stg_stream_v8(dst + 16 * k, o);
        }
    }
}

// Common argument checks; *tiles receives the number of scale tiles (0: nothing to do).
int check_codec(const char* who, int64_t rows, int64_t cols, const void* a, const void* codes, const void* scales, int64_t* tiles) {
    *tiles = 0;
    if (rows < 0 || cols < 0) return tcb::fail(TCB_ERR_BAD_ARG, "%s: negative size", who);
    if (cols % 32 != 0) return tcb::fail(TCB_ERR_BAD_ARG, "%s: the last dimension (%lld) must be a multiple of 32", who, (long long)cols);
    if (rows == 0 || cols == 0) return TCB_OK;
    if (!a || !codes || !scales) return tcb::fail(TCB_ERR_BAD_ARG, "%s: null pointer", who);
    if ((reinterpret_cast<uintptr_t>(a) & 31) || ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15))
        return tcb::fail(TCB_ERR_ALIGNMENT, "%s: the values must be 32-byte and codes and scales 16-byte aligned", who);
    const int64_t limit = (int64_t(1) << 31) - 1, tr = (rows + kTileRows - 1) / kTileRows, tk = (cols + kTileCols - 1) / kTileCols;
    if (tr > limit || tk > limit || tr * tk > limit) return tcb::fail(TCB_ERR_TOO_LARGE, "%s: more than 2^31 - 1 tiles of 128 x 128", who);
    *tiles = tr * tk;
    return TCB_OK;
}

}  // namespace

extern "C" int tcb_quantize_mxfp4(const void* x, int dtype, int64_t rows, int64_t cols, uint8_t* codes, uint8_t* scales, void* stream) {
    const char* who = "tcb_quantize_mxfp4";
    if (dtype < TCB_DT_BF16 || dtype > TCB_DT_F32) return tcb::fail(TCB_ERR_BAD_ARG, "%s: unknown dtype %d", who, dtype);
    int64_t tiles = 0;
    const int rc = check_codec(who, rows, cols, x, codes, scales, &tiles);
    if (rc != TCB_OK || tiles == 0) return rc;
    const int64_t bpr = cols / 32, tk = (cols + kTileCols - 1) / kTileCols;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid(unsigned(tiles), 1, 1), block(kThreads, 1, 1);
    cudaError_t e;
    switch (dtype) {
    case TCB_DT_BF16:
        e = tcb::launch_overlapped(quantize_mxfp4_kernel<__nv_bfloat16>, grid, block, 0, st, static_cast<const __nv_bfloat16*>(x), rows, bpr, tk, codes, scales);
        break;
    case TCB_DT_F16:
        e = tcb::launch_overlapped(quantize_mxfp4_kernel<__half>, grid, block, 0, st, static_cast<const __half*>(x), rows, bpr, tk, codes, scales);
        break;
    default: e = tcb::launch_overlapped(quantize_mxfp4_kernel<float>, grid, block, 0, st, static_cast<const float*>(x), rows, bpr, tk, codes, scales);
    }
    return e == cudaSuccess ? TCB_OK : tcb::cuda_fail(e, who);
}

extern "C" int tcb_dequantize_mxfp4(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, uint16_t* out, void* stream) {
    const char* who = "tcb_dequantize_mxfp4";
    int64_t tiles = 0;
    const int rc = check_codec(who, rows, cols, out, codes, scales, &tiles);
    if (rc != TCB_OK || tiles == 0) return rc;
    const cudaError_t e = tcb::launch_overlapped(dequantize_mxfp4_kernel, dim3(unsigned(tiles)), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), codes,
                                                 scales, rows, cols / 32, (cols + kTileCols - 1) / kTileCols, out);
    return e == cudaSuccess ? TCB_OK : tcb::cuda_fail(e, who);
}
