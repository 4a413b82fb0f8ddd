/*
 * Microscaled 4-bit floating point (MXFP4): values to codes and scales, and back.
 *
 * A row is cut into blocks of 32 columns (the last one filled up with zeros). With top = the largest magnitude of a block,
 *   X = 2^(floor(log2(top)) - 2), kept in a byte as its biased exponent (127 stands for 1), at least 2^-127
 *   code = sign and the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to |v| / X, ties to the even code, 6 for what is above
 * so top / X lies in [4, 8). floor(log2(top)) is the exponent field of top, and v / X an exact ldexp: the only rounding is that
 * to the code, and it is the conversion instruction's (v_cvt_scalef32_pk_fp4_f32, whose own scale stays 1: it takes the exponent
 * field of a float, which 2^-127 does not have). A block of zeros has scale 0. A block with an infinity or a NaN has scale 255,
 * which stands for NaN, and codes 0. Back: code times scale, exact in f32 and in bf16 (two significant bits).
 *
 * A thread takes 8 values: four lanes hold a block and find its largest magnitude with two DPP exchanges, each stores 4 bytes of
 * codes, so that a wave's stores are 256 contiguous bytes, and the first lane of the four the scale. Rows may start anywhere: the
 * loads are 16 bytes wide whatever their alignment, single values only where a row ends. Bound by memory: 4608 x 16384 bf16 there
 * 36 us and back 28 (5.4 and 6.9 TB/s with the codes), f32 62 and 77 (5.5 and 4.4); a row is a launch of 2 us.
 */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iris_kernels_hip.h"

namespace {

constexpr int THREADS = 256;
constexpr int UNROLL = 2;                        /* groups of 8 values in flight per thread */

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
/* 16 bytes at an address that only suits one value */
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    f32x2 p = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}

template <bool STREAM, typename V>
__device__ __forceinline__ u32x4 load16(const V *p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool STREAM, typename V>
__device__ __forceinline__ void store16(V *p, u32x4 v) {
    if constexpr (STREAM) __builtin_nontemporal_store(v, p);
    else *p = v;
}

/* 8 values, as the bits of floats; left: how many of them the row has (at least 1 here, zeros behind). STREAM: with the streaming hint. */
template <bool STREAM>
__device__ __forceinline__ void load8(const uint16_t *p, int left, uint32_t (&v)[8]) {
    if (left >= 8) {
        const u32x4 r = load16<STREAM>(reinterpret_cast<const u32x4_at2 *>(p));
#pragma unroll
        for (int i = 0; i < 4; i++) { v[2 * i] = r[i] << 16; v[2 * i + 1] = r[i] & 0xffff0000u; }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < left ? (uint32_t)p[i] << 16 : 0u;
    }
}
template <bool STREAM>
__device__ __forceinline__ void load8(const float *p, int left, uint32_t (&v)[8]) {
    if (left >= 8) {
        const u32x4_at4 *q = reinterpret_cast<const u32x4_at4 *>(p);
        const u32x4 a = load16<STREAM>(q), b = load16<STREAM>(q + 1);
#pragma unroll
        for (int i = 0; i < 4; i++) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < left ? __float_as_uint(p[i]) : 0u;
    }
}
template <bool STREAM>
__device__ __forceinline__ void store8(uint16_t *p, int left, const float (&v)[8]) {
    const u32x4 r = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
    if (left >= 8) {
        store16<STREAM>(reinterpret_cast<u32x4_at2 *>(p), r);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) p[i] = (uint16_t)(r[i / 2] >> (16 * (i & 1)));
    }
}
template <bool STREAM>
__device__ __forceinline__ void store8(float *p, int left, const float (&v)[8]) {
    if (left >= 8) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const u32x4 r = {__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]), __float_as_uint(v[4 * h + 2]), __float_as_uint(v[4 * h + 3])};
            store16<STREAM>(reinterpret_cast<u32x4_at4 *>(p) + h, r);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) p[i] = v[i];
    }
}

/* the largest of the four lanes of a quad */
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));       /* lane ^ 1 */
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));    /* lane ^ 2 */
}

/* Group i of 8 values is columns 8 c .. 8 c + 7 of row s, i = s * per_row + c with per_row = 4 blocks: a multiple of 4, as is
 * `groups`, so the lanes of a quad hold one block and leave together. 32-bit divisions where the count allows. */
__device__ __forceinline__ void place(size_t i, size_t groups, uint32_t per_row, size_t &s, uint32_t &c) {
    if (groups >> 32) { s = i / per_row; c = (uint32_t)(i - s * per_row); }
    else { const uint32_t q = (uint32_t)i / per_row; s = q; c = (uint32_t)i - q * per_row; }
}

template <typename T, bool STREAM>
__global__ void __launch_bounds__(THREADS)
k_to_mxfp4(uint32_t *__restrict__ codes, uint8_t *__restrict__ scales, const T *__restrict__ src, int ld, int cols, uint32_t per_row, size_t groups) {
    const size_t first = (size_t)blockIdx.x * (THREADS * UNROLL) + threadIdx.x;
    uint32_t v[UNROLL][8];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
        const size_t i = first + u * THREADS;
        size_t s;
        uint32_t c;
        place(i, groups, per_row, s, c);
        const int left = i < groups ? cols - 8 * (int)c : 0;
        if (left > 0) load8<STREAM>(src + s * ld + 8 * c, left, v[u]);
        else
#pragma unroll
            for (int k = 0; k < 8; k++) v[u][k] = 0u;
    }
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
        const size_t i = first + u * THREADS;
        if (i >= groups) return;
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) top = max(top, v[u][k] & 0x7fffffffu);
        top = quad_max(top);
        const bool finite = top < 0x7f800000u;
        const int e = max((int)(top >> 23) - 129, -127);       /* the exponent of X; denormals are far below it */
        uint32_t code = 0;
        auto scaled = [&](int k) { return __builtin_amdgcn_ldexpf(__uint_as_float(v[u][k]), -e); };
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, scaled(0), scaled(1), 1.0f, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, scaled(2), scaled(3), 1.0f, 1);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, scaled(4), scaled(5), 1.0f, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, scaled(6), scaled(7), 1.0f, 3);
        codes[i] = finite ? code : 0u;
        if ((i & 3) == 0) scales[i >> 2] = finite ? (uint8_t)(e + 127) : (uint8_t)255;
    }
}

template <typename T, bool STREAM>
__global__ void __launch_bounds__(THREADS)
k_mxfp4_to(T *__restrict__ dst, int ld, const uint32_t *__restrict__ codes, const uint8_t *__restrict__ scales, int cols, uint32_t per_row, size_t groups) {
    const size_t first = (size_t)blockIdx.x * (THREADS * UNROLL) + threadIdx.x;
    uint32_t code[UNROLL];
    int scale[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
        const size_t i = first + u * THREADS < groups ? first + u * THREADS : groups - 1;
        code[u] = codes[i];
        scale[u] = scales[i >> 2];
    }
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
        const size_t i = first + u * THREADS;
        if (i >= groups) return;
        size_t s;
        uint32_t c;
        place(i, groups, per_row, s, c);
        const int left = cols - 8 * (int)c;
        if (left <= 0) continue;
        const f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[u], 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[u], 1.0f, 1),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[u], 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[u], 1.0f, 3)};
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++)
            v[k] = scale[u] == 255 ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(p[k / 2][k & 1], scale[u] - 127);
        store8<STREAM>(dst + s * ld + 8 * c, left, v);
    }
}

/* Values of 2 bytes: 64 MB and more are read, 100 MB and more written, with the streaming hint, past the Infinity Cache (256 MB): they do not all stay there, and
 * the codes, which are read next, do. There and back, us, plain / streaming: 4608 x 16384 bf16 74.1 / 61.8 (6.2 TB/s with the codes), 4608 x 8192 40.3 / 34.6; with
 * both hints 4608 x 4096 18.8 / 19.7. Not f32, where a thread's 8 values are two accesses of 16 bytes, 32 bytes apart in neighbouring lanes, and with the hint the halves
 * of a line go their own ways. To codes, 1024 x 16384 12.4 / 15.4, 4608 x 16384 61.8 / 64.8 (and 2304 x 16384 with bf16 back 48.9 / 49.0); from codes, 1600 x 16384
 * 28.5 / 39.9, 4608 x 16384 78.0 / 121 (4.4 TB/s with the codes), 3001 x 16381 62 / 78. */
constexpr size_t STREAM_READ = (size_t)64 << 20, STREAM_WRITE = (size_t)100 << 20;

template <typename T, bool STREAM>
int launch_to(void *stream, uint8_t *codes, uint8_t *scales, const T *src, int ld, int rows, int cols) {
    const uint32_t per_row = 4u * (((uint32_t)cols + 31) / 32);
    const size_t groups = (size_t)rows * per_row, blocks = (groups + THREADS * UNROLL - 1) / (THREADS * UNROLL);
    if (blocks * THREADS >> 32) return (int)hipErrorInvalidValue;       /* a launch has fewer than 2^32 threads */
    hipLaunchKernelGGL((k_to_mxfp4<T, STREAM>), dim3((unsigned)blocks), dim3(THREADS), 0, (hipStream_t)stream, reinterpret_cast<uint32_t *>(codes), scales, src, ld,
                       cols, per_row, groups);
    return (int)hipGetLastError();
}
template <typename T, bool STREAM>
int launch_from(void *stream, T *dst, int ld, const uint8_t *codes, const uint8_t *scales, int rows, int cols) {
    const uint32_t per_row = 4u * (((uint32_t)cols + 31) / 32);
    const size_t groups = (size_t)rows * per_row, blocks = (groups + THREADS * UNROLL - 1) / (THREADS * UNROLL);
    if (blocks * THREADS >> 32) return (int)hipErrorInvalidValue;       /* a launch has fewer than 2^32 threads */
    hipLaunchKernelGGL((k_mxfp4_to<T, STREAM>), dim3((unsigned)blocks), dim3(THREADS), 0, (hipStream_t)stream, dst, ld, reinterpret_cast<const uint32_t *>(codes), scales,
                       cols, per_row, groups);
    return (int)hipGetLastError();
}

template <typename T>
int to_mxfp4(void *stream, uint8_t *codes, uint8_t *scales, const T *src, int ld, int rows, int cols) {
    if constexpr (sizeof(T) == 2)
        if ((size_t)rows * cols * sizeof(T) >= STREAM_READ) return launch_to<T, true>(stream, codes, scales, src, ld, rows, cols);
    return launch_to<T, false>(stream, codes, scales, src, ld, rows, cols);
}
template <typename T>
int mxfp4_to(void *stream, T *dst, int ld, const uint8_t *codes, const uint8_t *scales, int rows, int cols) {
    if constexpr (sizeof(T) == 2)
        if ((size_t)rows * cols * sizeof(T) >= STREAM_WRITE) return launch_from<T, true>(stream, dst, ld, codes, scales, rows, cols);
    return launch_from<T, false>(stream, dst, ld, codes, scales, rows, cols);
}

}  // namespace

extern "C" {

int iris_hip_f32_to_mxfp4(void *stream, uint8_t *codes, uint8_t *scales, const float *src, int ld, int rows, int cols) {
    return to_mxfp4(stream, codes, scales, src, ld, rows, cols);
}
int iris_hip_bf16_to_mxfp4(void *stream, uint8_t *codes, uint8_t *scales, const uint16_t *src, int ld, int rows, int cols) {
    return to_mxfp4(stream, codes, scales, src, ld, rows, cols);
}
int iris_hip_mxfp4_to_f32(void *stream, float *dst, int ld, const uint8_t *codes, const uint8_t *scales, int rows, int cols) {
    return mxfp4_to(stream, dst, ld, codes, scales, rows, cols);
}
int iris_hip_mxfp4_to_bf16(void *stream, uint16_t *dst, int ld, const uint8_t *codes, const uint8_t *scales, int rows, int cols) {
    return mxfp4_to(stream, dst, ld, codes, scales, rows, cols);
}

}  // extern "C"
