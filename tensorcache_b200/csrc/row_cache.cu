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
// Both kernels are bound by HBM.  A thread takes V values of one group (write: G = 8: 8; 16, 32, 64, 128: 16; 24, 48: 24;
// read: 32 for G = 32, 64, 128), so that most accesses are 32 bytes; 1 to 8 neighbouring lanes make up a group and combine
// max|x| by shuffles.  Two units a thread are in flight: each starts with a chain of dependent loads (index, claim, data).
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tcb_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int64_t kScanRows = 1024;   // rows of 768 bf16 values, us, scan / claim: 1: 1.8 / 4.1, 1024: 3.6 / 4.8, 2048: 5.8 / 5.2, 16384: 57 / 10.5

template <int G>
struct Split {
    static constexpr int V = G == 8 ? 8 : G % 24 == 0 ? 24 : 16;   // values per thread, write
    static constexpr int LPG = G / V;                              // lanes per group
    static constexpr int R = G % 32 == 0 ? 32 : V;                 // values per thread, read
};

// BYTES contiguous bytes: 32 at a time where a unit's size keeps them aligned, else 16, else 8.
template <int BYTES>
__device__ __forceinline__ void load_bytes(const void* p, uint32_t* w) {
    if constexpr (BYTES % 32 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 32; ++i) tcb::ldg_stream_v8(static_cast<const uint8_t*>(p) + 32 * i, w + 8 * i);
    } else if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const uint4 v = __ldcs(static_cast<const uint4*>(p) + i);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else {
        static_assert(BYTES % 8 == 0, "units are multiples of 8 bytes");
#pragma unroll
        for (int i = 0; i < BYTES / 8; ++i) {
            const uint2 v = __ldcs(static_cast<const uint2*>(p) + i);
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    }
}
template <int BYTES>
__device__ __forceinline__ void store_bytes(void* p, const uint32_t* w) {
    if constexpr (BYTES % 32 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 32; ++i) tcb::stg_stream_v8(static_cast<uint8_t*>(p) + 32 * i, w + 8 * i);
    } else if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) __stcs(static_cast<uint4*>(p) + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 8; ++i) __stcs(static_cast<uint2*>(p) + i, make_uint2(w[2 * i], w[2 * i + 1]));
    }
}

// Value i of a unit held as packed words.
template <typename T>
__device__ __forceinline__ float value_of(const uint32_t* w, int i);
template <>
__device__ __forceinline__ float value_of<__nv_bfloat16>(const uint32_t* w, int i) {
    return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
}
template <>
__device__ __forceinline__ float value_of<__half>(const uint32_t* w, int i) {
    return __half2float(__ushort_as_half(uint16_t((i & 1) ? (w[i >> 1] >> 16) : (w[i >> 1] & 0xffffu))));
}
template <>
__device__ __forceinline__ float value_of<float>(const uint32_t* w, int i) { return __uint_as_float(w[i]); }

__device__ __forceinline__ bool finite_f32(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

// max|x| over a unit, NaN or infinity if a value is not finite: the order of the bit patterns without sign is the order of
// the magnitudes, and everything that is not finite lies above.  16-bit types compare two at once.
template <typename T, int WORDS>
__device__ __forceinline__ float max_magnitude(const uint32_t (&w)[WORDS]) {
    uint32_t m = 0;
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) m = max(m, w[i] & 0x7fffffffu);
        return __uint_as_float(m);
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
        const uint32_t one[1] = {max(m & 0xffffu, m >> 16)};
        return value_of<T>(one, 0);
    }
}
// Values that are not finite become 0.
template <typename T, int WORDS>
__device__ __forceinline__ void clear_nonfinite(uint32_t (&w)[WORDS]) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        if constexpr (std::is_same<T, float>::value) {
            if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] = 0;
        } else {
            constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
            if ((w[i] & kExp) == kExp) w[i] &= 0xffff0000u;
            if ((w[i] & (kExp << 16)) == (kExp << 16)) w[i] &= 0x0000ffffu;
        }
    }
}

// The V values of a unit -> packed codes; returns the group's scale.  Every lane of the warp calls this.
template <int G, typename T>
__device__ __forceinline__ uint16_t encode_unit(uint32_t (&raw)[Split<G>::V * sizeof(T) / 4], uint32_t (&w)[Split<G>::V / 4]) {
    constexpr int V = Split<G>::V, LPG = Split<G>::LPG;
    float amax = max_magnitude<T>(raw);
    if (__builtin_expect(!finite_f32(amax), 0)) {
        clear_nonfinite<T>(raw);
        amax = max_magnitude<T>(raw);
    }
#pragma unroll
    for (int off = 1; off < LPG; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    const uint16_t sbits = __bfloat16_as_ushort(__float2bfloat16_rn(__fdiv_rn(fmaxf(amax, 1e-8f), 127.0f)));
    const float s = __uint_as_float(uint32_t(sbits) << 16), r = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        uint32_t c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // The IEEE quotient: the residual of rn(x * rn(1 / s)) is exact in one FMA because s has 8 significant
            // bits, and one more corrects the quotient (Markstein).  |x / s| < 127.3, so the clamp to [-128, 127]
            // never binds; adding 1.5 * 2^23 rounds to nearest even.
            const float x1 = value_of<T>(raw, 4 * i + j), t = __fmul_rn(x1, r);
            c[j] = __float_as_uint(__fadd_rn(__fmaf_rn(__fmaf_rn(-t, s, x1), r, t), 12582912.0f));
        }
        w[i] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    }
    return sbits;
}

// Codes of a unit and, from the group's first lane, the scale.
template <int G>
__device__ __forceinline__ void store_unit(const uint32_t (&w)[Split<G>::V / 4], uint16_t sbits, int8_t* __restrict__ q, uint16_t* __restrict__ scale) {
    store_bytes<Split<G>::V>(q, w);
    if ((threadIdx.x & (Split<G>::LPG - 1)) == 0) *scale = sbits;
}

// Launched plainly, so everything before it on the stream has finished; the write kernel may start under it.
__global__ void claim_rows_kernel(const int64_t* __restrict__ indices, int64_t n, int64_t num_rows, unsigned long long* __restrict__ claims) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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
        uint32_t raw[V * sizeof(T) / 4] = {};
        if (live) load_bytes<V * int(sizeof(T))>(x + int64_t(t) * width + u * V, raw);
        uint32_t w[V / 4];
        const uint16_t sbits = encode_unit<G, T>(raw, w);
        if (live) store_unit<G>(w, sbits, codes + row * width + u * V, scales + row * (width / G) + u * V / G);
    }
}

// Row and unit of a position in the list of all rows' units; Index is 32 bits wide where that suffices: the division costs
// 57,088 rows of 768 written 29.1 us instead of 30.2.
template <typename Index>
struct Place {
    Index t, k;
    __device__ __forceinline__ Place(int64_t u, Index upr) : t(Index(u) / upr), k(Index(u) - t * upr) {}
};

// Many rows: units of all rows in one grid-stride loop, two at a time (fp32: one; the other way round 57,088 x 768 bf16
// values take 32.6 us instead of 30.5, 20,000 x 1560 fp32 values 29.0 instead of 25.7); a row whose claim did not stay is
// left out.
template <int G, typename T, typename Index>
__global__ void __launch_bounds__(kThreads)
write_rows_kernel(const T* __restrict__ x, const int64_t* __restrict__ indices, int64_t n, int8_t* __restrict__ codes,
                  uint16_t* __restrict__ scales, int64_t num_rows, int64_t width, unsigned long long* __restrict__ claims) {
    constexpr int V = Split<G>::V, kUnits = sizeof(T) == 2 ? 2 : 1;
    const Index upr = Index(width / V);
    const int64_t units = n * int64_t(upr), gpr = width / G;
    bool waited = false;
    for (int64_t u0 = int64_t(blockIdx.x) * (kThreads * kUnits); u0 < units; u0 += int64_t(gridDim.x) * (kThreads * kUnits)) {
        int64_t row[kUnits], k[kUnits];
        uint32_t place[kUnits], raw[kUnits][V * sizeof(T) / 4];
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            const int64_t u = u0 + j * kThreads + threadIdx.x;
            row[j] = -1;
            k[j] = 0;
            place[j] = 0;
#pragma unroll
            for (int i = 0; i < V * int(sizeof(T)) / 4; ++i) raw[j][i] = 0;
            if (u < units) {
                const Place<Index> at(u, upr);
                row[j] = __ldg(indices + at.t);
                k[j] = int64_t(at.k);
                place[j] = uint32_t(at.t);
                load_bytes<V * int(sizeof(T))>(x + u * V, raw[j]);   // before the row is known to stay
            }
        }
        // The claims, past L1: what it holds of them may be older than the claiming kernel.  They arrive while the units are
        // encoded.
        if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
        waited = true;
        uint32_t claim[kUnits];
#pragma unroll
        for (int j = 0; j < kUnits; ++j) claim[j] = row[j] >= 0 && row[j] < num_rows ? uint32_t(__ldcg(claims + row[j])) : place[j] + 1;
        uint32_t w[kUnits][V / 4];
        uint16_t sbits[kUnits];
#pragma unroll
        for (int j = 0; j < kUnits; ++j) sbits[j] = encode_unit<G, T>(raw[j], w[j]);
#pragma unroll
        for (int j = 0; j < kUnits; ++j)
            if (claim[j] == place[j]) store_unit<G>(w[j], sbits[j], codes + row[j] * width + k[j] * V, scales + row[j] * gpr + k[j] * V / G);
    }
    // nothing in this launch reads the call number: the claims of the next call get another one (a block without units has not
    // waited for this call's claims yet)
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x == 0 && threadIdx.x == 0) claims[num_rows] += 1;
}

template <int G, typename Index>
__global__ void __launch_bounds__(kThreads)
read_rows_kernel(const int8_t* __restrict__ codes, const uint16_t* __restrict__ scales, int64_t num_rows, int64_t width,
                 const int64_t* __restrict__ indices, int64_t n, uint16_t* __restrict__ out) {
    constexpr int R = Split<G>::R, kUnits = 2;
    const Index upr = Index(width / R);
    const int64_t units = n * int64_t(upr), gpr = width / G;
    for (int64_t u0 = int64_t(blockIdx.x) * (kThreads * kUnits) + threadIdx.x; u0 < units; u0 += int64_t(gridDim.x) * (kThreads * kUnits)) {
        uint32_t c[kUnits][R / 4];
        float s[kUnits];
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            const int64_t u = u0 + j * kThreads;
            s[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < R / 4; ++i) c[j][i] = 0;
            if (u < units) {
                const Place<Index> at(u, upr);
                const int64_t row = __ldg(indices + at.t), k = int64_t(at.k);
                if (row >= 0 && row < num_rows) {
                    s[j] = __uint_as_float(uint32_t(__ldg(scales + row * gpr + k * R / G)) << 16);
                    load_bytes<R>(codes + row * width + k * R, c[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            const int64_t u = u0 + j * kThreads;
            if (u >= units) break;
            // code byte + 128 in the mantissa of 2^23, minus (2^23 + 128): the code, exactly; one rounding of the product
            uint32_t o[R / 2];
#pragma unroll
            for (int i = 0; i < R / 4; ++i) {
                const uint32_t w = c[j][i] ^ 0x80808080u;
                float f[4];
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    f[h] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | h)), 8388736.0f), s[j]);
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[2 * i]) : "f"(f[1]), "f"(f[0]));
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[2 * i + 1]) : "f"(f[3]), "f"(f[2]));
            }
            store_bytes<2 * R>(out + u * R, o);
        }
    }
}

// Blocks of a grid-stride loop over `units` units, two per thread: one wave at most.
int64_t wave(int64_t units) {
    const int64_t blocks = (units + 2 * kThreads - 1) / (2 * kThreads), most = int64_t(tcb::sm_count()) * 8;
    return blocks < most ? blocks : most;
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
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const dim3 grid(unsigned(wave(n * upr))), block(kThreads);
    const T* xt = static_cast<const T*>(x);
    if (n * upr < (int64_t(1) << 32))
        return tcb::launch_overlapped(write_rows_kernel<G, T, uint32_t>, grid, block, 0, st, xt, indices, n, codes, scales, num_rows, width, c);
    return tcb::launch_overlapped(write_rows_kernel<G, T, int64_t>, grid, block, 0, st, xt, indices, n, codes, scales, num_rows, width, c);
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
    const int64_t units = n * (width / Split<G>::R);
    const unsigned grid = unsigned(wave(units));
    if (units < (int64_t(1) << 32))
        read_rows_kernel<G, uint32_t><<<grid, kThreads, 0, st>>>(codes, scales, num_rows, width, indices, n, out);
    else
        read_rows_kernel<G, int64_t><<<grid, kThreads, 0, st>>>(codes, scales, num_rows, width, indices, n, out);
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
    if ((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(codes)) & 31)
        return tcb::fail(TCB_ERR_ALIGNMENT, "%s: data and codes must be 32-byte aligned", who);
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
