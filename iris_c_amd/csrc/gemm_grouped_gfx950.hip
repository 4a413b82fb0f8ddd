/*
 * Linear layers over groups of rows, each with weights of its own (row_groups.h):
 *
 *   y[m, :] = x[m, :] W[g]^T for the rows m of group g      bf16 inputs, f32 accumulation, f32 or bf16 output
 *
 * k_grouped_any takes every size and alignment: 128 x 128 tiles on 2 x 2 waves of 64 x 64, K in steps of 64, one LDS stage of
 * [W tile | x tile] with rows padded to 160 B (the 16 lanes that the LDS serves together on a 128-bit read then fall in distinct bank
 * windows), the next step waiting in registers meanwhile. Its loads are 16 bytes wide at any alignment; where a row of K
 * ends inside one, single values are read and zeros stand behind them.
 */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iris_kernels_hip.h"
#include "row_groups.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));           /* 16 bytes at an address that suits one value */

namespace {

constexpr int TK = 64, LS = TK + 16;             /* K of a step, LDS row stride in elements */

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
/* 8 values from p, of which `left` exist */
__device__ __forceinline__ u32x4 load8(const uint16_t *p, int left) {
    if (left >= 8) return *reinterpret_cast<const u32x4_at2 *>(p);
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < left) v[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
    return v;
}

template <typename OUT>
__global__ void __launch_bounds__(256, 2)
k_grouped_any(OUT *__restrict__ y, const uint16_t *__restrict__ x, const uint16_t *__restrict__ W, int M, int N, int K, const int *__restrict__ first_row, int groups) {
    constexpr int TM = 128, TN = 128;
    __shared__ __align__(16) uint16_t lds[(TN + TM) * LS];
    uint16_t *Wl = lds, *Xl = lds + TN * LS;
    const int tiles_n = (N + TN - 1) / TN, tm = blockIdx.x / tiles_n, n0 = (blockIdx.x - tm * tiles_n) * TN;
    RowGroups<TM> all;
    if (tm >= all.count(first_row, groups, M)) return;         /* the same for the whole workgroup */
    const RowTile t = all.tile(tm);
    W += (size_t)t.group * N * K;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lg = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;
    /* this thread moves 16 B chunk tid % 8 of rows tid / 8 + 32 c of both tiles; rows past the end repeat the last one */
    const int srow = tid >> 3, scol = (tid & 7) * 8;
    const uint16_t *wsrc[4], *xsrc[4];
#pragma unroll
    for (int c = 0; c < 4; c++) {
        wsrc[c] = W + (size_t)min(n0 + srow + 32 * c, N - 1) * K;
        xsrc[c] = x + (size_t)min(t.m0 + srow + 32 * c, t.end - 1) * K;
    }
    u32x4 wreg[4], xreg[4];
    auto fetch = [&](int k0) {
        const int k = k0 + scol, left = K - k;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            wreg[c] = left > 0 ? load8(wsrc[c] + k, left) : u32x4{0, 0, 0, 0};
            xreg[c] = left > 0 ? load8(xsrc[c] + k, left) : u32x4{0, 0, 0, 0};
        }
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int a = 0; a < 4; a++)
#pragma unroll
        for (int b = 0; b < 4; b++) acc[a][b] = f32x4{0, 0, 0, 0};
    const int a_rd = (64 * wn + li) * LS + 8 * lg, b_rd = (64 * wm + li) * LS + 8 * lg;

    fetch(0);
    for (int k0 = 0; k0 < K; k0 += TK) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            *reinterpret_cast<u32x4 *>(&Wl[(srow + 32 * c) * LS + scol]) = wreg[c];
            *reinterpret_cast<u32x4 *>(&Xl[(srow + 32 * c) * LS + scol]) = xreg[c];
        }
        __syncthreads();
        if (k0 + TK < K) fetch(k0 + TK);
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            u32x4 av[4], bv[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                av[i] = *reinterpret_cast<const u32x4 *>(&Wl[a_rd + 16 * i * LS + 32 * ks]);
                bv[i] = *reinterpret_cast<const u32x4 *>(&Xl[b_rd + 16 * i * LS + 32 * ks]);
            }
#pragma unroll
            for (int a = 0; a < 4; a++)
#pragma unroll
                for (int b = 0; b < 4; b++)
                    acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, av[a]), __builtin_bit_cast(bf16x8, bv[b]), acc[a][b], 0, 0, 0);
        }
        __syncthreads();
    }
    /* acc[a][b][r] = y[m0 + 64 wm + 16 b + li][n0 + 64 wn + 16 a + 4 lg + r] */
#pragma unroll
    for (int b = 0; b < 4; b++) {
        const int m = t.m0 + 64 * wm + 16 * b + li;
        if (m >= t.end) continue;
#pragma unroll
        for (int a = 0; a < 4; a++) {
            const int n = n0 + 64 * wn + 16 * a + 4 * lg;
            if (n < N) store4(y + (size_t)m * N + n, acc[a][b], N - n);
        }
    }
}

template <typename OUT>
int grouped(void *stream, OUT *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    const long wgs = row_tiles_at_most(rows, groups, 128) * ((out + 127L) / 128);
    if (wgs >> 31) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((k_grouped_any<OUT>), dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream, y, x, W, rows, out, in, first_row, groups);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

int iris_hip_linear_f32_grouped(void *stream, float *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    return grouped(stream, y, x, W, first_row, groups, rows, in, out);
}
int iris_hip_linear_bf16_grouped(void *stream, uint16_t *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    return grouped(stream, y, x, W, first_row, groups, rows, in, out);
}

}  // extern "C"
