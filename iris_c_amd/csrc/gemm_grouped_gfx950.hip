/*
 * Linear layers over groups of rows, each with weights of its own (row_groups.h):
 *
 *   y[m, :] = x[m, :] W[g]^T for the rows m of group g      bf16 inputs, f32 accumulation, f32 or bf16 output
 *
 * Groups of many rows run on the tiles of the plain layers (k_gemm_wide of gemm_conv_gfx950.hip, k_gemm_tiles of gemm_tiles_gfx950.hip, which take
 * their tile's rows and weights from row_groups.h), where rows are a multiple of 64 long, results a multiple of 8 and matrices 16-byte aligned; groups of a
 * few rows on k_grouped_rows below.
 *
 * k_grouped_any takes every size and alignment: tiles of 64 x 64 or 128 x 128 on 2 x 2 waves, K in steps of 64, two LDS stages of
 * [W tile | x tile] with rows padded to 160 B (the 16 lanes that the LDS serves together on a 128-bit read then fall in distinct bank
 * windows). The next step is put into one stage while the other is multiplied, and the one after it is on its way to registers. Its loads are 16
 * bytes wide at any alignment; where a row of K ends inside one, in the last step, single values are read and zeros stand behind them. Latency bounds it where
 * tiles are few (3556 rows, 1355 -> 256: 18.5 us in tiles of 64, 29.3 of 128, and 65 with one stage and a test at each load), the loads and the
 * LDS where they are many (4000 rows, 4097 -> 4097: 300 us, 448 TFLOP/s; tiles of 64 take 414).
 */
#include <hip/hip_runtime.h>

#include <cfloat>
#include <stdint.h>

#include "half_words.h"
#include "iris_kernels_hip.h"
#include "row_groups.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));           /* at an address that suits one value */
typedef unsigned u32x2_at2 __attribute__((ext_vector_type(2), aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
typedef f32x4 f32x4_at4 __attribute__((aligned(4)));

namespace {

constexpr int TK = 64, LS = TK + 16;             /* K of a step, LDS row stride in elements */

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    f32x2 p = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}
__device__ __forceinline__ void store4(float *p, f32x4 v, int n_left) {
    if (n_left >= 4) { *reinterpret_cast<f32x4_at4 *>(p) = v; return; }
    for (int r = 0; r < 4 && r < n_left; r++) p[r] = v[r];
}
__device__ __forceinline__ void store4(uint16_t *p, f32x4 v, int n_left) {
    if (n_left >= 4) { *reinterpret_cast<u32x2_at2 *>(p) = u32x2_at2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])}; return; }
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

template <typename OUT, int B>
__global__ void __launch_bounds__(256, 2)
k_grouped_any(OUT *__restrict__ y, const uint16_t *__restrict__ x, const uint16_t *__restrict__ W, int M, int N, int K, const int *__restrict__ first_row, int groups) {
    constexpr int T = 32 * B;
    __shared__ __align__(16) uint16_t lds[2][2 * T * LS];
    const int tiles_n = (N + T - 1) / T, tm = blockIdx.x / tiles_n, n0 = (blockIdx.x - tm * tiles_n) * T;
    RowGroups<T> all;
    if (tm >= all.count(first_row, groups, M)) return;         /* the same for the whole workgroup */
    const RowTile t = all.tile(tm);
    W += (size_t)t.group * N * K;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lg = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;
    /* this thread moves 16 B chunk tid % 8 of rows tid / 8 + 32 c of both tiles; rows past the end repeat the last one */
    const int srow = tid >> 3, scol = (tid & 7) * 8;
    const uint16_t *src[2][B];
#pragma unroll
    for (int c = 0; c < B; c++) {
        src[0][c] = W + (size_t)min(n0 + srow + 32 * c, N - 1) * K + scol;
        src[1][c] = x + (size_t)min(t.m0 + srow + 32 * c, t.end - 1) * K + scol;
    }
    const int steps = (K - 1) / TK + 1, whole = K / TK;
    struct Step { u32x4 v[2][B]; };
    auto fetch = [&](Step &s, int step) {
        if (step < whole) {
#pragma unroll
            for (int c = 0; c < 2 * B; c++) s.v[c % 2][c / 2] = *reinterpret_cast<const u32x4_at2 *>(src[c % 2][c / 2] + step * TK);
        } else if (step < steps) {
#pragma unroll
            for (int c = 0; c < 2 * B; c++) s.v[c % 2][c / 2] = K - step * TK > scol ? load8(src[c % 2][c / 2] + step * TK, K - step * TK - scol) : u32x4{0, 0, 0, 0};
        }
    };
    f32x4 acc[B][B];
#pragma unroll
    for (int a = 0; a < B; a++)
#pragma unroll
        for (int b = 0; b < B; b++) acc[a][b] = f32x4{0, 0, 0, 0};
    const int a_rd = (16 * B * wn + li) * LS + 8 * lg, b_rd = (T + 16 * B * wm + li) * LS + 8 * lg;
    /* the values of step + 2 are requested, and those of step + 1 put into the other stage, while those of this step are multiplied */
    auto put = [&](const Step &s, uint16_t *stage) {
#pragma unroll
        for (int c = 0; c < 2 * B; c++) *reinterpret_cast<u32x4 *>(&stage[(c % 2 * T + srow + 32 * (c / 2)) * LS + scol]) = s.v[c % 2][c / 2];
    };
    auto multiply = [&](const uint16_t *stage) {
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            u32x4 av[B], bv[B];
#pragma unroll
            for (int i = 0; i < B; i++) {
                av[i] = *reinterpret_cast<const u32x4 *>(&stage[a_rd + 16 * i * LS + 32 * ks]);
                bv[i] = *reinterpret_cast<const u32x4 *>(&stage[b_rd + 16 * i * LS + 32 * ks]);
            }
#pragma unroll
            for (int a = 0; a < B; a++)
#pragma unroll
                for (int b = 0; b < B; b++)
                    acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, av[a]), __builtin_bit_cast(bf16x8, bv[b]), acc[a][b], 0, 0, 0);
        }
    };
    Step s0, s1;
    fetch(s0, 0);
    fetch(s1, 1);
    put(s0, lds[0]);
    for (int step = 0;; step += 2) {
        __syncthreads();
        fetch(s0, step + 2);
        multiply(lds[0]);
        if (step + 1 >= steps) break;
        put(s1, lds[1]);
        __syncthreads();
        fetch(s1, step + 3);
        multiply(lds[1]);
        if (step + 2 >= steps) break;
        put(s0, lds[0]);
    }
    /* acc[a][b][r] = y[m0 + 16 (B wm + b) + li][n0 + 16 (B wn + a) + 4 lg + r] */
#pragma unroll
    for (int b = 0; b < B; b++) {
        const int m = t.m0 + 16 * (B * wm + b) + li;
        if (m >= t.end) continue;
#pragma unroll
        for (int a = 0; a < B; a++) {
            const int n = n0 + 16 * (B * wn + a) + 4 * lg;
            if (n < N) store4(y + (size_t)m * N + n, acc[a][b], N - n);
        }
    }
}

/* ---- few rows a group: operands straight from memory into registers ----
 *
 * A wave owns 16 rows x 16 A columns and walks a range of K; KW waves of a workgroup share the outputs, take a range each and add their sums
 * through the LDS, in order. A step is 32 U columns of K: lane group g of the four holds chunks U g .. U g + U - 1 of 8, 64 contiguous bytes
 * of its row with U = 4, and U products follow each other. The operands of the next step are on their way while this one is
 * multiplied; in the last step of a row that is no multiple of 32 U long, chunks past the end are zeros.
 *
 * Rows of an odd K start in the middle of 4 bytes every second time, and 16-byte loads from there take four times as long. HALVES: whole 4 bytes are loaded
 * instead, from those in which a run of values starts (half: 1 if in their middle) to those in which it ends, and shifted in registers. INSIDE: x or W starts in the middle of
 * 4 bytes itself; the steps whose words would reach past the matrices (half_words.h) are loaded as the last step is. A kernel of its own: in one for both the others took 5 % longer. us:
 * groups of 3, 4 and 1 rows, 8001 -> 1001, in 16-byte loads from anywhere 34.8, shifted 16.1 (8002 -> 1001 14.0); of 70 and 81 rows, 2817 -> 2661,
 * two blocks of columns, 104 / 42. (k_grouped_any loses by it: 2 x 1000 rows, 2561 -> 2561 88 / 101.)
 *
 * Bound by HBM: 16 rows over 128 groups, 2560 -> 1536 (126 MB) 27 us. */
__device__ __forceinline__ u32x4 load_run(const uint16_t *p, int half) { return *reinterpret_cast<const u32x4_at4 *>(run_start(p, half)); }
__device__ __forceinline__ uint32_t load_end(const uint16_t *end, int half) { return *reinterpret_cast<const uint32_t *>(run_last(end, half)); }
__device__ __forceinline__ u32x4 shifted(u32x4 v, uint32_t behind, int bits) {
    return u32x4{__builtin_amdgcn_alignbit(v[1], v[0], bits), __builtin_amdgcn_alignbit(v[2], v[1], bits), __builtin_amdgcn_alignbit(v[3], v[2], bits),
                 __builtin_amdgcn_alignbit(behind, v[3], bits)};
}

/* all rows start at 4 bytes; the matrices do, but rows are odd; x or W does not */
enum Starts { WORDS, HALVES, INSIDE };

template <typename OUT, int A, int U, int KW, Starts STARTS>
__global__ void __launch_bounds__(64 * KW)
k_grouped_rows(OUT *__restrict__ y, const uint16_t *__restrict__ x, const uint16_t *__restrict__ W, int M, int N, int K, const int *__restrict__ first_row, int groups) {
    constexpr int TM = 16, TN = 16 * A;
    constexpr bool SHIFTED = STARTS != WORDS;
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

    struct Step { u32x4 a[U][A], b[U]; uint32_t a_end[A], b_end; };
    auto fetch = [&](Step &s, int k0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = k0 + 8 * (U * lg + u);
#pragma unroll
            for (int i = 0; i < A; i++) s.a[u][i] = load_run(wrow[i] + k, SHIFTED ? half(wrow[i]) : 0);
            s.b[u] = load_run(xrow + k, SHIFTED ? half(xrow) : 0);
        }
        if constexpr (SHIFTED) {
            const int end = k0 + 8 * U * (lg + 1);
#pragma unroll
            for (int i = 0; i < A; i++) s.a_end[i] = load_end(wrow[i] + end, half(wrow[i]));
            s.b_end = load_end(xrow + end, half(xrow));
        }
    };
    auto shift = [&](Step &s) {
        if constexpr (SHIFTED) {
#pragma unroll
            for (int u = 0; u < U; u++) {
#pragma unroll
                for (int i = 0; i < A; i++) s.a[u][i] = shifted(s.a[u][i], u + 1 < U ? s.a[u + 1][i][0] : s.a_end[i], 16 * half(wrow[i]));
                s.b[u] = shifted(s.b[u], u + 1 < U ? s.b[u + 1][0] : s.b_end, 16 * half(xrow));
            }
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
    const HalfSteps inside = STARTS == INSIDE ? half_steps(x, W, K, 32 * U) : HalfSteps{0, K / (32 * U)};
    const int steps = (K - 1) / (32 * U) + 1;
    const int from = (int)((long)steps * kw / KW), to = (int)((long)steps * (kw + 1) / KW), full = min(to, inside.upto);
    Step s0, s1;
    int at = from;
    if (STARTS == INSIDE && at < min(inside.first, to)) {
        fetch_last(s0, at * 32 * U);
        multiply(s0);
        at++;
    }
    if (at < full) {
        fetch(s0, at * 32 * U);
        while (true) {
            if (at + 1 < full) fetch(s1, (at + 1) * 32 * U);
            shift(s0);
            multiply(s0);
            if (++at >= full) break;
            if (at + 1 < full) fetch(s0, (at + 1) * 32 * U);
            shift(s1);
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

bool halves(const uint16_t *x, const uint16_t *W, int in) { return (in & 1) || half(x) || half(W); }

template <typename OUT, int A, int U, int KW>
int launch_rows(hipStream_t st, OUT *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    const long wgs = row_tiles_at_most(rows, groups, 16) * ((out + 16L * A - 1) / (16 * A));
    if (!launch_fits(wgs, 64 * KW)) return (int)hipErrorInvalidValue;
    const dim3 grid((unsigned)(wgs + 7) / 8 * 8), block(64 * KW);
#define ROWS(STARTS) hipLaunchKernelGGL((k_grouped_rows<OUT, A, U, KW, STARTS>), grid, block, 0, st, y, x, W, rows, out, in, first_row, groups)
    if (half(x) || half(W)) ROWS(INSIDE);
    else if (in & 1) ROWS(HALVES);
    else ROWS(WORDS);
#undef ROWS
    return (int)hipGetLastError();
}

template <typename OUT, int B>
int launch_any(hipStream_t st, OUT *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    const long wgs = row_tiles_at_most(rows, groups, 32 * B) * ((out + 32L * B - 1) / (32 * B));
    if (!launch_fits(wgs, 256)) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((k_grouped_any<OUT, B>), dim3((unsigned)wgs), dim3(256), 0, st, y, x, W, rows, out, in, first_row, groups);
    return (int)hipGetLastError();
}

/* Which kernel, host arithmetic only, from the rows and groups there are; how the rows lie in them is only known on the device. 3: k_gemm_wide in
 * tiles of 32 `shape` columns, 2: k_gemm_tiles with its tile `shape` and `splits` ranges of K, 1: k_grouped_rows with 16 `shape` columns a
 * wave, 0: k_grouped_any in tiles of 32 `shape` x 32 `shape`. The least estimated time decides. k_grouped_rows reads a group's weights once for every 16 of its rows, at 6 TB/s
 * where they come from a cache (its loads are 16 rows of 64 bytes each) and 5 TB/s from HBM, the tiles at 4.7 from HBM. us, k_grouped_rows / the
 * best tiles: 16 groups of 8 rows, 2560 -> 2560 43.5 / 48.5, of 16 49.6 / 47.7, of 17 74.9 / 48.8, of 64 139 / 50; 4 groups of 1024 -> 1024, 1 row each 3.9 / 8.8,
 * 30 5.8 / 8.8, 64 8.6 / 10.0; 2 groups of 2560 -> 6144, 16 rows 16 / 17.5, 32 22.8 / 17.8. Two blocks of columns a wave halve the reads of x where there are
 * enough workgroups: the 16 groups 57.8 / 46.0 at 12 rows, but 1 row in each of 4 3.9 / 4.7. Kernels whose grid could pass the limit of a launch are left
 * out: k_grouped_rows has a thread for every 8 - 16 results, and k_grouped_any for every 16 - 64. (The tiles' operands fill the memory before theirs could.) */
struct Plan { int kernel, shape, splits; };
Plan plan_grouped(int groups, int rows, int in, int out, int out_size, bool aligned16, bool halves, size_t part_bytes) {
    const long some = groups < rows ? groups : rows, few_tiles = row_tiles_about(rows, groups, 16);
    const float weights = (float)out * (float)in * 2.0f, every = (float)some * weights;
    const float cached = (float)few_tiles * weights / (halves ? 4.2e6f : 6.0e6f), fresh = every / 5.0e6f;
    auto fits = [&](int tm, int tn) { return launch_fits(row_tiles_at_most(rows, groups, tm) * ((out + tn - 1L) / tn), 256); };
    float best = 3.0f + (cached > fresh ? cached : fresh);
    Plan plan = {1, few_tiles * ((out + 31L) / 32) >= 512 ? 2 : 1, 1};
    if (!fits(16, 16 * plan.shape)) { best = FLT_MAX; plan = {0, 4, 1}; }
    const float least = 4.0f + every / 4.7e6f;                 /* of the tiles */
    if (aligned16) {
        int shape = 0, splits = 1;
        float us = iris_hip_gemm_tiles_grouped_plan(groups, rows, out, in, out_size, part_bytes, &shape, &splits);
        if (us >= 0.0f && (us > least ? us : least) < best) { best = us > least ? us : least; plan = {2, shape, splits}; }
        us = iris_hip_gemm_wide_grouped_plan(groups, rows, out, in, out_size, &shape);
        if (us >= 0.0f && (us > least ? us : least) < best) { best = us > least ? us : least; plan = {3, shape, 1}; }
    }
    /* a step of 64 columns, alone on a CU and each of those that share it */
    for (int blocks = 2; blocks <= 4; blocks += 2) {
        const int tile = 32 * blocks;
        const float alone = blocks == 2 ? 0.62f : 1.1f, share = blocks == 2 ? 0.42f : 1.08f;
        const long wgs = row_tiles_about(rows, groups, tile) * ((out + tile - 1L) / tile);
        const float each = share * (float)((wgs + 255) / 256), us = 5.0f + (float)((in + 63L) / 64) * (each > alone ? each : alone);
        if (us < best && fits(tile, tile)) { best = us; plan = {0, blocks, 1}; }
    }
    return plan;
}

template <typename OUT>
int grouped(void *stream, float *part, OUT *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    hipStream_t st = (hipStream_t)stream;
    const bool aligned16 = (((uintptr_t)x | (uintptr_t)W | (uintptr_t)y) & 15) == 0;
    const Plan plan = plan_grouped(groups, rows, in, out, (int)sizeof(OUT), aligned16, halves(x, W, in), part ? IRIS_LINEAR_PART_BYTES : 0);
    if (plan.kernel == 3) return iris_hip_gemm_wide_grouped(stream, y, (int)sizeof(OUT), x, W, first_row, groups, rows, out, in, plan.shape);
    if (plan.kernel == 2) return iris_hip_gemm_tiles_grouped(stream, y, (int)sizeof(OUT), x, W, first_row, groups, rows, out, in, plan.shape, plan.splits, part);
    if (plan.kernel == 1)
        return plan.shape == 2 ? launch_rows<OUT, 2, 2, 4>(st, y, x, W, first_row, groups, rows, in, out) : launch_rows<OUT, 1, 4, 4>(st, y, x, W, first_row, groups, rows, in, out);
    return plan.shape == 2 ? launch_any<OUT, 2>(st, y, x, W, first_row, groups, rows, in, out) : launch_any<OUT, 4>(st, y, x, W, first_row, groups, rows, in, out);
}

}  // namespace

extern "C" {

/* plan[0..2]: the kernel a layer of these sizes takes with 16-byte aligned operands, its tile and its ranges of K, as plan_grouped has them. No GPU needed. */
void iris_hip_linear_grouped_plan(int groups, int rows, int in, int out, int out_bytes, int *plan) {
    const Plan p = plan_grouped(groups, rows, in, out, out_bytes, true, in & 1, IRIS_LINEAR_PART_BYTES);
    plan[0] = p.kernel; plan[1] = p.shape; plan[2] = p.splits;
}

int iris_hip_linear_f32_grouped(void *stream, float *part, float *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    return grouped(stream, part, y, x, W, first_row, groups, rows, in, out);
}
int iris_hip_linear_bf16_grouped(void *stream, float *part, uint16_t *y, const uint16_t *x, const uint16_t *W, const int *first_row, int groups, int rows, int in, int out) {
    return grouped(stream, part, y, x, W, first_row, groups, rows, in, out);
}

}  // extern "C"
