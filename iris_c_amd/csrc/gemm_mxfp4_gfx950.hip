/*
 * Linear layers in microscaled 4-bit floating point (MXFP4, see mxfp4_ops.hip), of all rows or of groups of rows with weights of
 * their own:
 *
 *   y[m, n] = sum over blocks b of 2^(xs[m, b] + ws[n, b] - 254) sum over the 32 columns i of b of x[m, i] W[n, i]
 *
 * f32 sums, f32 or bf16 output. v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands as they lie in memory: lane l holds the 32
 * codes (16 bytes) of row l % 16 in block l / 16 of the four, and that block's scale in a byte of another register. As in the bf16
 * layers the product is issued transposed (A = W rows, B = x rows), so that a lane holds four consecutive n of one output row.
 */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iris_kernels_hip.h"
#include "row_groups.h"

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

namespace {

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    f32x2 p = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}
__device__ __forceinline__ void store4(float *p, f32x4 v, int n_left) {
    if (n_left >= 4 && ((uintptr_t)p & 15) == 0) { *reinterpret_cast<f32x4 *>(p) = v; return; }
    for (int r = 0; r < 4 && r < n_left; r++) p[r] = v[r];
}
__device__ __forceinline__ void store4(uint16_t *p, f32x4 v, int n_left) {
    if (n_left >= 4 && ((uintptr_t)p & 7) == 0) { *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])); return; }
    for (int r = 0; r < 4 && r < n_left; r++) p[r] = (uint16_t)(pack_bf16(v[r], 0.0f) & 0xffffu);
}
/* scales: byte A_BYTE / B_BYTE of sa / sb; four bits an element on both sides */
template <int A_BYTE, int B_BYTE>
__device__ __forceinline__ f32x4 mfma(i32x4 a, i32x4 b, f32x4 c, int sa, int sb) {
    const i32x8 wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, A_BYTE, sa, B_BYTE, sb);
}

/* Any sizes: operands straight from memory, 64 x 64 outputs a wave, 2 x 2 waves. */
template <typename OUT, bool GROUPED>
__global__ void __launch_bounds__(256, 2)
k_mxfp4_any(OUT *__restrict__ y, const uint8_t *__restrict__ x, const uint8_t *__restrict__ xs, const uint8_t *__restrict__ W,
            const uint8_t *__restrict__ Ws, int M, int N, int nb, const int *__restrict__ first_row, int groups) {
    constexpr int TM = 128, TN = 128;
    const int tiles_n = (N + TN - 1) / TN, tm = blockIdx.x / tiles_n, n0 = (blockIdx.x - tm * tiles_n) * TN;
    RowTile t = {tm * TM, M, 0};
    if constexpr (GROUPED) {
        RowGroups<TM> all;
        if (tm >= all.count(first_row, groups, M)) return;
        t = all.tile(tm);
        W += (size_t)t.group * N * nb * 16;
        Ws += (size_t)t.group * N * nb;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4;
    const int mw = t.m0 + 64 * (wave & 1), nw = n0 + 64 * (wave >> 1);
    size_t xrow[4], wrow[4];                                   /* rows past the end repeat the last one, and are not stored */
#pragma unroll
    for (int i = 0; i < 4; i++) {
        xrow[i] = (size_t)min(mw + 16 * i + li, t.end - 1) * nb;
        wrow[i] = (size_t)min(nw + 16 * i + li, N - 1) * nb;
    }
    i32x4 a[4], b[4];
    int sa[4], sb[4];
    auto fetch = [&](int step) {
        const int blk = 4 * step + lg;
        const bool in = blk < nb;
        const int at = in ? blk : 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            a[i] = *reinterpret_cast<const i32x4 *>(W + (wrow[i] + at) * 16);
            b[i] = *reinterpret_cast<const i32x4 *>(x + (xrow[i] + at) * 16);
            sa[i] = Ws[wrow[i] + at];
            sb[i] = xs[xrow[i] + at];
            if (!in) { a[i] = i32x4{0, 0, 0, 0}; b[i] = a[i]; sa[i] = 127; sb[i] = 127; }
        }
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0, 0, 0, 0};
    const int steps = (nb + 3) / 4;
    for (int s = 0; s < steps; s++) {
        fetch(s);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = mfma<0, 0>(a[i], b[j], acc[i][j], sa[i], sb[j]);
    }
    /* acc[a][b][r] = y[mw + 16 b + li][nw + 16 a + 4 lg + r] */
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int m = mw + 16 * j + li;
        if (m >= t.end) continue;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int n = nw + 16 * i + 4 * lg;
            if (n < N) store4(y + (size_t)m * N + n, acc[i][j], N - n);
        }
    }
}

template <typename OUT>
int linear(void *stream, OUT *y, const uint8_t *x, const uint8_t *xs, const uint8_t *W, const uint8_t *Ws, const int *first_row, int groups, int rows, int in,
           int out) {
    const int nb = (int)(((long)in + 31) / 32);
    const long wgs = (first_row ? row_tiles_at_most(rows, groups, 128) : ((long)rows + 127) / 128) * ((out + 127L) / 128);
    if (wgs >> 31) return (int)hipErrorInvalidValue;
    if (first_row)
        hipLaunchKernelGGL((k_mxfp4_any<OUT, true>), dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream, y, x, xs, W, Ws, rows, out, nb, first_row, groups);
    else
        hipLaunchKernelGGL((k_mxfp4_any<OUT, false>), dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream, y, x, xs, W, Ws, rows, out, nb, nullptr, 1);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

int iris_hip_linear_mxfp4_f32(void *stream, float *y, const uint8_t *x, const uint8_t *xs, const uint8_t *W, const uint8_t *Ws, const int *first_row, int groups,
                              int rows, int in, int out) {
    return linear(stream, y, x, xs, W, Ws, first_row, groups, rows, in, out);
}
int iris_hip_linear_mxfp4_bf16(void *stream, uint16_t *y, const uint8_t *x, const uint8_t *xs, const uint8_t *W, const uint8_t *Ws, const int *first_row, int groups,
                               int rows, int in, int out) {
    return linear(stream, y, x, xs, W, Ws, first_row, groups, rows, in, out);
}

}  // extern "C"
