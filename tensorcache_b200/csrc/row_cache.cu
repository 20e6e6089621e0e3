// Rows of a device-resident cache of symmetric int8 codes: quantised as they are written, decoded as they are read.
//
//     write:  codes[i, :], scales[i, :] = int8 codes and bf16 scales of x[t, :]      i = indices[t]
//             scale = bf16(max|x| / 127) per group of G values, code = rne(x / scale), the numbers of tcb_compress_sym
//     read:   out[t, :] = bf16(codes[i, :] * scales[i, :])                            the numbers of tcb_decompress_sym
//
// An index outside [0, num_rows) skips its row (write) or yields zeros (read).  If an index occurs more than once in
// one write, the last occurrence is the one that stays, whole: up to kScanRows rows a block looks through the later
// indices itself (one launch: what a step of a few rows costs is its latency); beyond that the rows first claim their
// slot with an atomic maximum over (call number << 32 | row).  The call number lives in device memory and is advanced
// by the write kernel, so that claims need no clearing and a captured graph can be replayed.
//
// Both kernels are bound by HBM.  A thread takes V values of one group (G = 8: 8; 16, 32, 64, 128: 16; 24, 48: 24),
// 1, 2, 4 or 8 neighbouring lanes make up a group and combine max|x| by shuffles.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tcb_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int64_t kScanRows = 1024;

template <int G>
struct Split {
    static constexpr int V = G == 8 ? 8 : G % 24 == 0 ? 24 : 16;   // values per thread
    static constexpr int LPG = G / V;                              // lanes per group
};

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }

__device__ __forceinline__ bool finite_f32(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

// V values of one group (8-value pieces are 16 or 32 bytes and 16-byte aligned) -> codes at q and, from the group's
// first lane, the scale.  Every lane of the warp calls this; `live` lanes store.
template <int G, typename T>
__device__ __forceinline__ void encode_unit(const T* __restrict__ x, bool live, int8_t* __restrict__ q, uint16_t* __restrict__ scale) {
    constexpr int V = Split<G>::V, LPG = Split<G>::LPG;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; i += 16 / int(sizeof(T))) {
        union {
            uint4 w;
            T t[16 / sizeof(T)];
        } u;
        u.w = live ? __ldcs(reinterpret_cast<const uint4*>(x + i)) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 16 / int(sizeof(T)); ++j) v[i + j] = widen<T>(u.t[j]);
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        v[i] = finite_f32(v[i]) ? v[i] : 0.0f;
        amax = fmaxf(amax, fabsf(v[i]));
    }
#pragma unroll
    for (int off = 1; off < LPG; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    const uint16_t sbits = __bfloat16_as_ushort(__float2bfloat16_rn(__fdiv_rn(fmaxf(amax, 1e-8f), 127.0f)));
    const float s = __uint_as_float(uint32_t(sbits) << 16), r = __frcp_rn(s);
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        uint32_t c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // The IEEE quotient: the residual of rn(x * rn(1 / s)) is exact in one FMA because s has 8 significant
            // bits, and one more corrects the quotient (Markstein).  |x / s| < 127.3, so the clamp to [-128, 127]
            // never binds; adding 1.5 * 2^23 rounds to nearest even.
            const float x1 = v[4 * i + j], t = __fmul_rn(x1, r);
            c[j] = __float_as_uint(__fadd_rn(__fmaf_rn(__fmaf_rn(-t, s, x1), r, t), 12582912.0f));
        }
        w[i] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    }
    if (!live) return;
    if constexpr (V == 16) {
        __stcs(reinterpret_cast<uint4*>(q), make_uint4(w[0], w[1], w[2], w[3]));
    } else {
#pragma unroll
        for (int i = 0; i < V / 8; ++i) __stcs(reinterpret_cast<uint2*>(q) + i, make_uint2(w[2 * i], w[2 * i + 1]));
    }
    if ((threadIdx.x & (LPG - 1)) == 0) *scale = sbits;
}

__global__ void claim_rows_kernel(const int64_t* __restrict__ indices, int64_t n, int64_t num_rows, unsigned long long* __restrict__ claims) {
    const int64_t t = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (t >= n) return;
    const int64_t i = indices[t];
    if (i < 0 || i >= num_rows) return;
    atomicMax(claims + i, (claims[num_rows] << 32) | static_cast<unsigned long long>(t));
}

// Few rows: block (t, part) writes one part of row t after it has looked for a later row of the same index.
template <int G, typename T>
__global__ void __launch_bounds__(kThreads)
write_rows_scan_kernel(const T* __restrict__ x, const int64_t* __restrict__ indices, int n, int8_t* __restrict__ codes,
                       uint16_t* __restrict__ scales, int64_t num_rows, int64_t width) {
    constexpr int V = Split<G>::V;
    const int t = blockIdx.x;
    const int64_t row = indices[t];
    bool taken = row < 0 || row >= num_rows;
    for (int j = t + 1 + threadIdx.x; j < n; j += kThreads) taken |= indices[j] == row;
    if (__syncthreads_or(taken)) return;
    const int64_t units = width / V;
    // the bound of the loop is the same for all lanes of a warp: the shuffles need them
    for (int64_t u0 = int64_t(blockIdx.y) * kThreads; u0 < units; u0 += int64_t(gridDim.y) * kThreads) {
        const int64_t u = u0 + threadIdx.x;
        const bool live = u < units;
        encode_unit<G, T>(x + int64_t(t) * width + u * V, live, codes + row * width + u * V, scales + row * (width / G) + u * V / G);
    }
}

// Many rows: units of all rows in one grid-stride loop; a row whose claim did not stay is left out.
template <int G, typename T>
__global__ void __launch_bounds__(kThreads)
write_rows_kernel(const T* __restrict__ x, const int64_t* __restrict__ indices, int64_t n, int8_t* __restrict__ codes,
                  uint16_t* __restrict__ scales, int64_t num_rows, int64_t width, unsigned long long* __restrict__ claims) {
    constexpr int V = Split<G>::V;
    const int64_t upr = width / V, units = n * upr;
    for (int64_t u0 = int64_t(blockIdx.x) * kThreads; u0 < units; u0 += int64_t(gridDim.x) * kThreads) {
        const int64_t u = u0 + threadIdx.x;
        int64_t t = 0, k = 0, row = -1;
        if (u < units) {
            t = u / upr;
            k = u - t * upr;
            row = __ldg(indices + t);
            if (row >= num_rows || (row >= 0 && uint32_t(claims[row]) != uint32_t(t))) row = -1;
        }
        const bool live = row >= 0;
        encode_unit<G, T>(x + t * width + k * V, live, codes + row * width + k * V, scales + row * (width / G) + k * V / G);
    }
    // nothing in this launch reads the call number: the claims of the next call get another one
    if (blockIdx.x == 0 && threadIdx.x == 0) claims[num_rows] += 1;
}

template <int G>
__global__ void __launch_bounds__(kThreads)
read_rows_kernel(const int8_t* __restrict__ codes, const uint16_t* __restrict__ scales, int64_t num_rows, int64_t width,
                 const int64_t* __restrict__ indices, int64_t n, uint16_t* __restrict__ out) {
    constexpr int V = Split<G>::V;
    const int64_t upr = width / V, units = n * upr;
    for (int64_t u = int64_t(blockIdx.x) * kThreads + threadIdx.x; u < units; u += int64_t(gridDim.x) * kThreads) {
        const int64_t t = u / upr, k = u - t * upr, row = __ldg(indices + t);
        uint32_t c[V / 4];
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V / 4; ++i) c[i] = 0;
        if (row >= 0 && row < num_rows) {
            const int8_t* q = codes + row * width + k * V;
            s = __uint_as_float(uint32_t(__ldg(scales + row * (width / G) + k * V / G)) << 16);
            if constexpr (V == 16) {
                const uint4 w = __ldcs(reinterpret_cast<const uint4*>(q));
                c[0] = w.x, c[1] = w.y, c[2] = w.z, c[3] = w.w;
            } else {
#pragma unroll
                for (int i = 0; i < V / 8; ++i) {
                    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(q) + i);
                    c[2 * i] = w.x, c[2 * i + 1] = w.y;
                }
            }
        }
        // code byte + 128 in the mantissa of 2^23, minus (2^23 + 128): the code, exactly; one rounding of the product
        uint32_t o[V / 2];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const uint32_t w = c[i] ^ 0x80808080u;
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                f[j] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | j)), 8388736.0f), s);
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[2 * i]) : "f"(f[1]), "f"(f[0]));
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[2 * i + 1]) : "f"(f[3]), "f"(f[2]));
        }
        uint4* dst = reinterpret_cast<uint4*>(out + t * width + k * V);
#pragma unroll
        for (int i = 0; i < V / 8; ++i) __stcs(dst + i, make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
    }
}

template <int G, typename T>
cudaError_t launch_write(const void* x, const int64_t* indices, int64_t n, int8_t* codes, uint16_t* scales, int64_t num_rows,
                         int64_t width, int64_t* claims, cudaStream_t st) {
    const int64_t upr = width / Split<G>::V;
    if (n <= kScanRows) {
        const int64_t parts = (upr + kThreads - 1) / kThreads;
        const dim3 grid(unsigned(n), unsigned(parts < 1024 ? parts : 1024));
        write_rows_scan_kernel<G, T><<<grid, kThreads, 0, st>>>(static_cast<const T*>(x), indices, int(n), codes, scales, num_rows, width);
        return cudaGetLastError();
    }
    unsigned long long* c = reinterpret_cast<unsigned long long*>(claims);
    claim_rows_kernel<<<unsigned((n + kThreads - 1) / kThreads), kThreads, 0, st>>>(indices, n, num_rows, c);
    const int64_t blocks = (n * upr + kThreads - 1) / kThreads, most = int64_t(tcb::sm_count()) * 8;
    write_rows_kernel<G, T><<<unsigned(blocks < most ? blocks : most), kThreads, 0, st>>>(static_cast<const T*>(x), indices, n, codes, scales,
                                                                                         num_rows, width, c);
    return cudaGetLastError();
}

template <int G>
cudaError_t launch_write_typed(const void* x, int dtype, const int64_t* indices, int64_t n, int8_t* codes, uint16_t* scales,
                               int64_t num_rows, int64_t width, int64_t* claims, cudaStream_t st) {
    switch (dtype) {
    case TCB_DT_BF16: return launch_write<G, __nv_bfloat16>(x, indices, n, codes, scales, num_rows, width, claims, st);
    case TCB_DT_F16: return launch_write<G, __half>(x, indices, n, codes, scales, num_rows, width, claims, st);
    default: return launch_write<G, float>(x, indices, n, codes, scales, num_rows, width, claims, st);
    }
}

template <int G>
cudaError_t launch_read(const int8_t* codes, const uint16_t* scales, int64_t num_rows, int64_t width, const int64_t* indices, int64_t n,
                        uint16_t* out, cudaStream_t st) {
    const int64_t blocks = (n * (width / Split<G>::V) + kThreads - 1) / kThreads, most = int64_t(tcb::sm_count()) * 8;
    read_rows_kernel<G><<<unsigned(blocks < most ? blocks : most), kThreads, 0, st>>>(codes, scales, num_rows, width, indices, n, out);
    return cudaGetLastError();
}

int check_cache(const char* who, const void* data, const void* codes, const void* scales, int64_t num_rows, int64_t width, int group_size,
                const void* indices, int64_t n) {
    if (!tcb::group_size_ok(group_size))
        return tcb::fail(TCB_ERR_GROUP_SIZE, "%s: group_size %d not in {8, 16, 24, 32, 48, 64, 128}", who, group_size);
    if (num_rows < 0 || width < 0 || n < 0) return tcb::fail(TCB_ERR_BAD_ARG, "%s: negative size", who);
    if (width % group_size != 0)
        return tcb::fail(TCB_ERR_BAD_ARG, "%s: the row width %lld must be a multiple of the group size %d", who, (long long)width, group_size);
    if (n > (int64_t(1) << 31) - 1) return tcb::fail(TCB_ERR_TOO_LARGE, "%s: more than 2^31 - 1 rows in one call", who);
    if (n == 0 || width == 0) return TCB_OK;
    if (!data || !indices || (num_rows > 0 && (!codes || !scales))) return tcb::fail(TCB_ERR_BAD_ARG, "%s: null pointer", who);
    if ((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(codes)) & 15)
        return tcb::fail(TCB_ERR_ALIGNMENT, "%s: data and codes must be 16-byte aligned", who);
    if ((reinterpret_cast<uintptr_t>(indices) & 7) || (reinterpret_cast<uintptr_t>(scales) & 1))
        return tcb::fail(TCB_ERR_ALIGNMENT, "%s: indices must be 8-byte and scales 2-byte aligned", who);
    return TCB_OK;
}

}  // namespace

extern "C" int tcb_cache_write(const void* x, int dtype, const int64_t* indices, int64_t n, int8_t* codes, uint16_t* scales,
                               int64_t num_rows, int64_t width, int group_size, int64_t* claims, void* stream) {
    const char* who = "tcb_cache_write";
    if (dtype < TCB_DT_BF16 || dtype > TCB_DT_F32) return tcb::fail(TCB_ERR_BAD_ARG, "%s: unknown dtype %d", who, dtype);
    const int rc = check_cache(who, x, codes, scales, num_rows, width, group_size, indices, n);
    if (rc != TCB_OK || n == 0 || width == 0 || num_rows == 0) return rc;
    if (!claims || (reinterpret_cast<uintptr_t>(claims) & 7)) return tcb::fail(TCB_ERR_BAD_ARG, "%s: claims is null or not 8-byte aligned", who);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    switch (group_size) {
    case 8: e = launch_write_typed<8>(x, dtype, indices, n, codes, scales, num_rows, width, claims, st); break;
    case 16: e = launch_write_typed<16>(x, dtype, indices, n, codes, scales, num_rows, width, claims, st); break;
    case 24: e = launch_write_typed<24>(x, dtype, indices, n, codes, scales, num_rows, width, claims, st); break;
    case 32: e = launch_write_typed<32>(x, dtype, indices, n, codes, scales, num_rows, width, claims, st); break;
    case 48: e = launch_write_typed<48>(x, dtype, indices, n, codes, scales, num_rows, width, claims, st); break;
    case 64: e = launch_write_typed<64>(x, dtype, indices, n, codes, scales, num_rows, width, claims, st); break;
    default: e = launch_write_typed<128>(x, dtype, indices, n, codes, scales, num_rows, width, claims, st);
    }
    return e == cudaSuccess ? TCB_OK : tcb::cuda_fail(e, who);
}

extern "C" int tcb_cache_read(const int8_t* codes, const uint16_t* scales, int64_t num_rows, int64_t width, int group_size,
                              const int64_t* indices, int64_t n, uint16_t* out, void* stream) {
    const char* who = "tcb_cache_read";
    const int rc = check_cache(who, out, codes, scales, num_rows, width, group_size, indices, n);
    if (rc != TCB_OK || n == 0 || width == 0) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    switch (group_size) {
    case 8: e = launch_read<8>(codes, scales, num_rows, width, indices, n, out, st); break;
    case 16: e = launch_read<16>(codes, scales, num_rows, width, indices, n, out, st); break;
    case 24: e = launch_read<24>(codes, scales, num_rows, width, indices, n, out, st); break;
    case 32: e = launch_read<32>(codes, scales, num_rows, width, indices, n, out, st); break;
    case 48: e = launch_read<48>(codes, scales, num_rows, width, indices, n, out, st); break;
    case 64: e = launch_read<64>(codes, scales, num_rows, width, indices, n, out, st); break;
    default: e = launch_read<128>(codes, scales, num_rows, width, indices, n, out, st);
    }
    return e == cudaSuccess ? TCB_OK : tcb::cuda_fail(e, who);
}
