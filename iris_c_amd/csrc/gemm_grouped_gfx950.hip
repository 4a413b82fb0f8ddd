/*
 * Linear layers over groups of rows, each with weights of its own (row_groups.h):
 *
 *   y[m, :] = x[m, :] W[g]^T for the rows m of group g      bf16 inputs, f32 accumulation, f32 or bf16 output
 *
 * Groups of many rows run on the tiles of the plain layers (k_gemm_wide of gemm_conv_gfx950.hip, k_gemm_tiles of gemm_tiles_gfx950.hip, which take
 * their tile's rows and weights from row_groups.h), groups of a few rows on k_grouped_rows below.
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

/* ---- few rows a group: operands straight from memory into registers ----
 *
 * A wave owns 16 rows x 16 A columns and walks a range of K; KW waves of a workgroup share the outputs, take a range each and add their sums
 * through the LDS, in order. A step is 32 U columns of K: lane group g of the four holds chunks U g .. U g + U - 1 of 8, 64 contiguous bytes
 * of its row with U = 4, and U products follow each other. The operands of the next step are on their way while this one is
 * multiplied; in the last step of a row that is no multiple of 32 U long, chunks past the end are zeros. */
template <typename OUT, int A, int U, int KW>
__global__ void __launch_bounds__(64 * KW)
k_grouped_rows(OUT *__restrict__ y, const uint16_t *__restrict__ x, const uint16_t *__restrict__ W, int M, int N, int K, const int *__restrict__ first_row, int groups) {
    constexpr int TM = 16, TN = 16 * A;
    __shared__ __align__(16) f32x4 sums[KW][A][64];
    const int tiles_n = (N + TN - 1) / TN;
    RowGroups<TM> all;
    const int tiles_m = all.count(first_row, groups, M), total = tiles_m * tiles_n, per_xcd = (total + 7) / 8;
    const int work = (blockIdx.x % 8) * per_xcd + blockIdx.x / 8;            /* an XCD takes a contiguous range, row tiles fastest: those of a group share weights */
    if ((int)(blockIdx.x / 8) >= per_xcd || work >= total) return;
    const int tn = work / tiles_m;
    const RowTile t = all.tile(work - tn * tiles_m);
    const int lane = threadIdx.x & 63, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lg = lane >> 4, n0 = tn * TN;
    /* rows past the end repeat the last one, and are not stored */
    const uint16_t *wrow[A], *xrow = x + (size_t)min(t.m0 + li, t.end - 1) * K;
#pragma unroll
    for (int i = 0; i < A; i++) wrow[i] = W + ((size_t)t.group * N + min(n0 + 16 * i + li, N - 1)) * K;

    struct Step { u32x4 a[U][A], b[U]; };
    auto fetch = [&](Step &s, int k0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = k0 + 8 * (U * lg + u);
#pragma unroll
            for (int i = 0; i < A; i++) s.a[u][i] = *reinterpret_cast<const u32x4_at2 *>(wrow[i] + k);
            s.b[u] = *reinterpret_cast<const u32x4_at2 *>(xrow + k);
        }
    };
    auto fetch_last = [&](Step &s, int k0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = k0 + 8 * (U * lg + u), left = K - k;
#pragma unroll
            for (int i = 0; i < A; i++) s.a[u][i] = left > 0 ? load8(wrow[i] + k, left) : u32x4{0, 0, 0, 0};
            s.b[u] = left > 0 ? load8(xrow + k, left) : u32x4{0, 0, 0, 0};
        }
    };
    f32x4 acc[A];
#pragma unroll
    for (int i = 0; i < A; i++) acc[i] = f32x4{0, 0, 0, 0};
    auto multiply = [&](const Step &s) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < A; i++)
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, s.a[u][i]), __builtin_bit_cast(bf16x8, s.b[u]), acc[i], 0, 0, 0);
    };
    const int steps = (K + 32 * U - 1) / (32 * U), whole = K / (32 * U);
    const int from = (int)((long)steps * kw / KW), to = (int)((long)steps * (kw + 1) / KW), full = min(to, whole);
    Step s0, s1;
    int at = from;
    if (at < full) {
        fetch(s0, at * 32 * U);
        while (true) {
            if (at + 1 < full) fetch(s1, (at + 1) * 32 * U);
            multiply(s0);
            if (++at >= full) break;
            if (at + 1 < full) fetch(s0, (at + 1) * 32 * U);
            multiply(s1);
            if (++at >= full) break;
        }
    }
    if (at < to) {
        fetch_last(s0, at * 32 * U);
        multiply(s0);
    }
    /* acc[a][r] = y[m0 + li][n0 + 16 a + 4 lg + r]; each wave adds every KW-th block up */
#pragma unroll
    for (int i = 0; i < A; i++) sums[kw][i][lane] = acc[i];
    __syncthreads();
    const int m = t.m0 + li;
#pragma unroll
    for (int i = 0; i < A; i++) {
        const int n = n0 + 16 * i + 4 * lg;
        if (i % KW != kw || m >= t.end || n >= N) continue;
        f32x4 v = sums[0][i][lane];
#pragma unroll
        for (int k = 1; k < KW; k++) v += sums[k][i][lane];
        store4(y + (size_t)m * N + n, v, N - n);
    }
}

template <typename OUT, int A, int U, int KW>
int launch_rows(hipStream_t st, OUT *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    const long wgs = row_tiles_at_most(rows, groups, 16) * ((out + 16L * A - 1) / (16 * A));
    if (wgs >> 30) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((k_grouped_rows<OUT, A, U, KW>), dim3((unsigned)(wgs + 7) / 8 * 8), dim3(64 * KW), 0, st, y, x, W, rows, out, in, first_row, groups);
    return (int)hipGetLastError();
}

/* Which kernel, host arithmetic only, from the rows and groups there are; how the rows lie in them is only known on the device. 3: k_gemm_wide in
 * tiles of 32 `shape` columns, 2: k_gemm_tiles with its tile `shape` and `splits` ranges of K, 1: k_grouped_rows with 16 `shape` columns a
 * wave, 0: k_grouped_any. The least estimated time decides. k_grouped_rows reads a group's weights once for every 16 of its rows, at 6 TB/s
 * where they come from a cache (its loads are 16 rows of 64 bytes each) and 5 TB/s from HBM, the tiles at 4.7 from HBM. us, k_grouped_rows / the
 * best tiles: 16 groups of 8 rows, 2560 -> 2560 43.5 / 48.5, of 16 49.6 / 47.7, of 17 74.9 / 48.8, of 64 139 / 50; 4 groups of 1024 -> 1024, 1 row each 3.9 / 8.8,
 * 30 5.8 / 8.8, 64 8.6 / 10.0; 2 groups of 2560 -> 6144, 16 rows 16 / 17.5, 32 22.8 / 17.8. Two blocks of columns a wave halve the reads of x where there are
 * enough workgroups: the 16 groups 57.8 / 46.0 at 12 rows, but 1 row in each of 4 3.9 / 4.7. */
struct Plan { int kernel, shape, splits; };
Plan plan_grouped(int groups, int rows, int in, int out, int out_size, bool aligned16, size_t part_bytes) {
    const long some = groups < rows ? groups : rows, few_tiles = row_tiles_about(rows, groups, 16);
    const float weights = (float)out * (float)in * 2.0f, every = (float)some * weights;
    const float cached = (float)few_tiles * weights / 6.0e6f, fresh = every / 5.0e6f;
    float best = 3.0f + (cached > fresh ? cached : fresh);
    Plan plan = {1, few_tiles * ((out + 31L) / 32) >= 512 ? 2 : 1, 1};
    const float least = 4.0f + every / 4.7e6f;                 /* of the tiles */
    if (aligned16) {
        int shape = 0, splits = 1;
        float us = iris_hip_gemm_tiles_grouped_plan(groups, rows, out, in, out_size, part_bytes, &shape, &splits);
        if (us >= 0.0f && (us > least ? us : least) < best) { best = us > least ? us : least; plan = {2, shape, splits}; }
        us = iris_hip_gemm_wide_grouped_plan(groups, rows, out, in, out_size, &shape);
        if (us >= 0.0f && (us > least ? us : least) < best) { best = us > least ? us : least; plan = {3, shape, 1}; }
    }
    /* two workgroups a CU, a step of 64 columns 1.4 us in full rounds of them: 36 x 96 tiles of K = 4096 720 us, 1020 of 2560 114 */
    const long any_tiles = row_tiles_about(rows, groups, 128) * ((out + 127L) / 128);
    if (5.0f + (float)((any_tiles + 511) / 512) * (float)((in + 63) / 64) * 1.4f < best) plan = {0, 0, 1};
    return plan;
}

template <typename OUT>
int grouped(void *stream, float *part, OUT *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    hipStream_t st = (hipStream_t)stream;
    const bool aligned16 = (((uintptr_t)x | (uintptr_t)W | (uintptr_t)y) & 15) == 0;
    const Plan plan = plan_grouped(groups, rows, in, out, (int)sizeof(OUT), aligned16, part ? IRIS_LINEAR_PART_BYTES : 0);
    if (plan.kernel == 3) return iris_hip_gemm_wide_grouped(stream, y, (int)sizeof(OUT), x, W, first_row, groups, rows, out, in, plan.shape);
    if (plan.kernel == 2) return iris_hip_gemm_tiles_grouped(stream, y, (int)sizeof(OUT), x, W, first_row, groups, rows, out, in, plan.shape, plan.splits, part);
    if (plan.kernel == 1)
        return plan.shape == 2 ? launch_rows<OUT, 2, 2, 4>(st, y, x, W, first_row, groups, rows, in, out) : launch_rows<OUT, 1, 4, 4>(st, y, x, W, first_row, groups, rows, in, out);
    const long wgs = row_tiles_at_most(rows, groups, 128) * ((out + 127L) / 128);
    if (wgs >> 31) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((k_grouped_any<OUT>), dim3((unsigned)wgs), dim3(256), 0, st, y, x, W, rows, out, in, first_row, groups);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

/* plan[0..2]: the kernel a layer of these sizes takes with 16-byte aligned operands, its tile and its ranges of K, as plan_grouped has them. No GPU needed. */
void iris_hip_linear_grouped_plan(int groups, int rows, int in, int out, int out_bytes, int *plan) {
    const Plan p = plan_grouped(groups, rows, in, out, out_bytes, true, IRIS_LINEAR_PART_BYTES);
    plan[0] = p.kernel; plan[1] = p.shape; plan[2] = p.splits;
}

int iris_hip_linear_f32_grouped(void *stream, float *part, float *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    return grouped(stream, part, y, x, W, first_row, groups, rows, in, out);
}
int iris_hip_linear_bf16_grouped(void *stream, float *part, uint16_t *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    return grouped(stream, part, y, x, W, first_row, groups, rows, in, out);
}

}  // extern "C"
