/*
 * Linear layers in microscaled 4-bit floating point (MXFP4, see mxfp4_ops.hip), of all rows or of groups of rows with weights of
 * their own:
 *
 *   y[m, n] = sum over blocks b of 2^(xs[m, b] + ws[n, b] - 254) sum over the 32 columns i of b of x[m, i] W[n, i]
 *
 * f32 sums, f32 or bf16 output. v_mfma_scale_f32_16x16x128_f8f6f4 and _32x32x64_ take both operands as they lie in memory: a lane holds the 32
 * codes (16 bytes) of a row in one block, and that block's scale in a byte of another register, the same byte for all lanes. Which block of
 * a k-step a lane group holds is free as long as both operands agree, and is chosen so that a lane's scales of several products
 * are neighbouring bytes. As in the bf16 layers the product is issued transposed (A = W rows, B = x rows), so that a lane holds
 * four consecutive n of one output row.
 *
 * Three kernels: k_mxfp4_rows for a few rows (bound by the reading of the weights), k_mxfp4_tiles in four tiles, k_mxfp4_wide in tiles of 256 rows.
 * plan_mxfp4 chooses. Times are medians, of several runs from the least to the largest; "from HBM": the weights of more layers in turn than the Infinity Cache (256 MB) holds, otherwise they may be in it.
 */
#include <hip/hip_runtime.h>

#include <cfloat>
#include <climits>
#include <stdint.h>
#include <type_traits>

#include "iris_kernels_hip.h"
#include "row_groups.h"
#include "write_through.h"

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
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
/* 16 bytes of results at p, of which the row has `left` values. THROUGH the L2s or STREAMING where all rows are aligned, and so none ends inside 16 bytes. ANY:
 * one plain store whatever the alignment (parts of lines are better put together in the L2s: 777 x 1000 -> 1111 5.2 us, 6.3 through them), single values
 * at the end of a row. */
enum Store { THROUGH, STREAMING, ANY };
typedef i32x4 i32x4_at2 __attribute__((aligned(2)));           /* at an address that suits one value */
template <Store KIND> using Kind = std::integral_constant<Store, KIND>;
template <Store KIND, typename OUT>
__device__ __forceinline__ void store16(OUT *p, i32x4 v, int left) {
    constexpr int VALUES = 16 / (int)sizeof(OUT);
    if constexpr (KIND == THROUGH) {
        store_through(p, v);
    } else if constexpr (KIND == STREAMING) {
        __builtin_nontemporal_store(v, reinterpret_cast<i32x4 *>(p));
    } else if (left >= VALUES) {
        *reinterpret_cast<i32x4_at2 *>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < VALUES - 1; i++)
            if (i < left) {
                if constexpr (VALUES == 8) p[i] = (OUT)((uint32_t)v[i / 2] >> (16 * (i & 1)));
                else p[i] = __int_as_float(v[i]);
            }
    }
}
/* scales: byte A_BYTE / B_BYTE of sa / sb; four bits an element on both sides */
template <int A_BYTE, int B_BYTE>
__device__ __forceinline__ f32x4 mfma(i32x4 a, i32x4 b, f32x4 c, int sa, int sb) {
    const i32x8 wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, A_BYTE, sa, B_BYTE, sb);
}

template <int A_BYTE, int B_BYTE>
__device__ __forceinline__ f32x16 mfma32(i32x4 a, i32x4 b, f32x16 c, int sa, int sb) {
    const i32x8 wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, wb, c, 4, 4, A_BYTE, sa, B_BYTE, sb);
}

/* ---- few rows: operands straight from memory into registers ----
 *
 * A workgroup owns 16 rows x 16 A columns; its KW waves walk a range of K each and add their sums through the LDS, in order. A step is 16 blocks of
 * 32: lane group g of the four holds blocks 4 g .. 4 g + 3, 64 contiguous bytes of its row, four products follow each other, and the
 * scales are the bytes of one register. The operands of the next step are on their way while this one is multiplied. In the last step of a row
 * that is no multiple of 16 blocks long, blocks past the end are zeros with scale 1. Any sizes. Bound by the reading of the weights: 1 row, 4096 -> 24576 (54 MB) 11.6 - 12.0 us
 * from HBM (4.5 TB/s), 10.4 - 10.8 from the Infinity Cache; 40 rows over 64 groups, 2560 -> 1536 (48 MB) 14.2 and 13.1. */
constexpr int ROWS_KW = 4;
typedef uint32_t uint32_at1 __attribute__((aligned(1)));

template <typename OUT, int A, bool GROUPED>
__global__ void __launch_bounds__(64 * ROWS_KW)
k_mxfp4_rows(OUT *__restrict__ y, const uint8_t *__restrict__ x, const uint8_t *__restrict__ xs, const uint8_t *__restrict__ W,
             const uint8_t *__restrict__ Ws, int M, int N, int nb, const int *__restrict__ first_row, int groups) {
    constexpr int TM = 16, TN = 16 * A, U = 4, KW = ROWS_KW;
    __shared__ __align__(16) f32x4 sums[KW][A][64];
    /* an XCD takes a contiguous range of the work list, row tiles fastest: those of a group read the same weights */
    const int tiles_n = (N + TN - 1) / TN;
    int tiles_m = (M + TM - 1) / TM;
    RowGroups<TM> all;
    if constexpr (GROUPED) tiles_m = all.count(first_row, groups, M);
    const int total = tiles_m * tiles_n, per_xcd = (total + 7) / 8, work = (blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
    if ((int)(blockIdx.x / 8) >= per_xcd || work >= total) return;
    const int tn = work / tiles_m, tm = work - tn * tiles_m;
    RowTile t = {tm * TM, M, 0};
    if constexpr (GROUPED) t = all.tile(tm);
    const int lane = threadIdx.x & 63, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lg = lane >> 4, n0 = tn * TN;
    /* rows past the end repeat the last one, and are not stored */
    const size_t xrow = (size_t)min(t.m0 + li, t.end - 1) * nb;
    size_t wrow[A];
#pragma unroll
    for (int i = 0; i < A; i++) wrow[i] = ((size_t)t.group * N + min(n0 + 16 * i + li, N - 1)) * nb;

    struct Step { i32x4 a[A][U], b[U]; int sa[A], sb; };
    auto fetch = [&](Step &s, int at) {                        /* at: first block of the step; all of it inside the row */
        const int blk = at + U * lg;
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int i = 0; i < A; i++) s.a[i][u] = *reinterpret_cast<const i32x4 *>(W + (wrow[i] + blk + u) * 16);
            s.b[u] = *reinterpret_cast<const i32x4 *>(x + (xrow + blk + u) * 16);
        }
#pragma unroll
        for (int i = 0; i < A; i++) s.sa[i] = (int)*reinterpret_cast<const uint32_at1 *>(Ws + wrow[i] + blk);
        s.sb = (int)*reinterpret_cast<const uint32_at1 *>(xs + xrow + blk);
    };
    auto fetch_last = [&](Step &s, int at) {
        const int blk = at + U * lg;
        s.sb = 0;
#pragma unroll
        for (int i = 0; i < A; i++) s.sa[i] = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool in = blk + u < nb;
            const int from = in ? blk + u : 0;
#pragma unroll
            for (int i = 0; i < A; i++) {
                s.a[i][u] = *reinterpret_cast<const i32x4 *>(W + (wrow[i] + from) * 16);
                s.sa[i] |= (in ? (int)Ws[wrow[i] + from] : 127) << (8 * u);
            }
            s.b[u] = *reinterpret_cast<const i32x4 *>(x + (xrow + from) * 16);
            if (!in) s.b[u] = i32x4{0, 0, 0, 0};
            s.sb |= (in ? (int)xs[xrow + from] : 127) << (8 * u);
        }
    };
    f32x4 acc[A];
#pragma unroll
    for (int i = 0; i < A; i++) acc[i] = f32x4{0, 0, 0, 0};
    auto multiply = [&](const Step &s) {
        auto one = [&](auto byte) {
            constexpr int u = decltype(byte)::value;
#pragma unroll
            for (int i = 0; i < A; i++) acc[i] = mfma<u, u>(s.a[i][u], s.b[u], acc[i], s.sa[i], s.sb);
        };
        one(std::integral_constant<int, 0>{});
        one(std::integral_constant<int, 1>{});
        one(std::integral_constant<int, 2>{});
        one(std::integral_constant<int, 3>{});
    };
    /* this wave's steps */
    const int steps = (nb + 4 * U - 1) / (4 * U), whole = nb / (4 * U);
    const int from = (int)((long)steps * kw / KW), to = (int)((long)steps * (kw + 1) / KW), full = min(to, whole);
    Step s0, s1;
    int at = from;
    if (at < full) {
        fetch(s0, at * 4 * U);
        while (true) {
            if (at + 1 < full) fetch(s1, (at + 1) * 4 * U);
            multiply(s0);
            if (++at >= full) break;
            if (at + 1 < full) fetch(s0, (at + 1) * 4 * U);
            multiply(s1);
            if (++at >= full) break;
        }
    }
    if (at < to) {
        fetch_last(s0, at * 4 * U);
        multiply(s0);
    }
    /* acc[a][r] = y[m0 + li][n0 + 16 a + 4 lg + r]; wave a adds block a up */
#pragma unroll
    for (int i = 0; i < A; i++) sums[kw][i][lane] = acc[i];
    __syncthreads();
    const int m = t.m0 + li, n = n0 + 16 * kw + 4 * lg;
    if (kw >= A || m >= t.end || n >= N) return;
    f32x4 v = sums[0][kw][lane];
#pragma unroll
    for (int k = 1; k < KW; k++) v += sums[k][kw][lane];
    store4(y + (size_t)m * N + n, v, N - n);
}

/* ---- tiles of 256 rows x 256 or 192 columns ----
 *
 * For k tiles of 256: 128 B of codes and 8 scales of every row. Eight waves, two per
 * SIMD, 4 (rows of 64) x 2 (columns of 16 NA): a wave owns 64 rows x 16 NA columns = NA x 4 accumulator blocks. A k tile is two
 * k-steps of v_mfma_scale_f32_16x16x128: in k-step ks lane group g of the four holds block 2 g + ks of its row, so that its two scales are
 * neighbouring bytes. (32x32x64 products draw more power: of registers with random codes the chip keeps up 6600 TFLOP/s of them and 7100 - 7400 of these.)
 *
 * Everything comes from memory straight into the LDS (160 KB at 256 columns): two stages of x, two and a half of W (a ring of five half tiles,
 * the columns of one wave column each), two of scales, which are fetched for two k tiles at a time (16 B a row). 16 B chunk c of row r sits
 * in slot c ^ swizzle(r): the 16 lanes that the LDS serves together on a 128-bit read are eight rows of each of two neighbouring lane
 * groups, with chunks that differ in bit 1. Two rows next to each other span the banks once; of each parity the four rows of one group
 * ((r >> 1) & 7 in {0, 1, 6, 7}) fill slots {0, 1, 2, 3} ^ c, those of the other {4, 5, 6, 7} ^ c ^ 2: all different.
 *
 * A k tile is four steps: k-step 0 with the first and the second half of the columns, then k-step 1; the operands of a step are read
 * during the step before, the scales of the next tile in steps 0 and 2. Codes of k tile t + 2: the first half of W in steps 0 and 2 of
 * tile t, the rest in step 3, behind the one barrier of a tile, which frees the stage. Every memory instruction stands in a gap between two
 * products. Requests past the end of K are issued all the same (a branch around each costs more, and the waits count them), but all lanes ask for
 * one 16 B of the last tile, into a stage that nobody reads.
 *
 * A k tile takes 1.7 us (256 tiles, K 4096 and 12288), its products at the rate above 1.16 - 1.21, and the first loads and the stores of a round of tiles 5.5 more, when nothing
 * else runs on a CU. 4608 x 4096 -> 36864 355 - 366 us (3.8 - 3.9 PFLOP/s; 2592 tiles are 10.1 rounds and take 11; the matrix cores are busy for half of the cycles, at 1.85 - 1.96 of
 * 2.4 GHz), 512 + 4096 rows in groups -> 12288 128 - 132 (from HBM 148), 512 x 2560 -> 19456 18.8 - 19.6 (21.0 - 21.4). f32 results, 4608 x 4096 -> 36864 395.
 *
 * Any number of columns: of an unaligned row the pieces are stored as they lie (bf16 results, 4608 x 4096 -> 9001 102 us; with tiles of 128 x 128 165). One k tile
 * is taken too (2327 x 256 -> 16384 25 us; 95).
 *
 * Rows that are no whole k tiles long, or whose scales are not 8-byte aligned: k_mxfp4_scales copies the scales into rows of 8 bytes a k tile. The last k
 * tile then is the last 8 blocks of a row, with scales 0 for those that the one before it has had: 2^-254 a product, nothing in f32, whatever the codes. us,
 * bf16 results, with it / tiles of 128 x 128: 2930 x 3793 -> 6325 60 / 97, 1158 x 896 -> 10821 19 / 48, 512 x 2500 -> 19457 26 / 51. */
template <int NA>
struct Wide {
    static constexpr int TM = 256, TN = 32 * NA, WP = (2 * NA + 7) / 8;                  /* WP: 8-row pieces of half of W per wave */
    static constexpr int XS = TM * 128, WH = TN / 2 * 128, SC = (TM + TN) * 16;          /* bytes: a stage of x, half of one of W, scales of two k tiles */
    static constexpr int W0 = 2 * XS, S0 = W0 + 5 * WH, NEED = S0 + 2 * SC;
    static constexpr int LDS = NEED > 128 * 1024 ? NEED : 128 * 1024;                    /* the epilogue takes 128 KB */
    static_assert(LDS <= 160 * 1024, "");
};

__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}
/* (r >> 1) & 7 = 0 1 2 3 4 5 6 7 -> 0 1 4 5 6 7 2 3 */
__device__ __forceinline__ int swizzle(int r) {
    const int j = r >> 1;
    return (j & 1) | ((j >> 1) & 2) | (((j << 1) ^ j) & 4);
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"                          /* M0 in a clobber list */
template <typename OUT, int NA, bool STREAM, bool GROUPED>
__global__ void __launch_bounds__(512, 2)
k_mxfp4_wide(OUT *__restrict__ y, const uint8_t *__restrict__ x, const uint8_t *__restrict__ xs, const uint8_t *__restrict__ W,
             const uint8_t *__restrict__ Ws, int M, int N, int nb, const int *__restrict__ first_row, int groups) {
    using T = Wide<NA>;
    constexpr int TM = T::TM, TN = T::TN, WP = T::WP, H0 = (NA + 1) / 2, H1 = NA / 2;
    static_assert(WP == 2 && H1 >= 3, "");
    extern __shared__ __align__(16) uint8_t lds[];
    /* Each XCD (own L2) takes a contiguous range of the tile list, which runs through bands of four tile rows, inside a band m fastest */
    const int tiles_n = (N + TN - 1) / TN;
    int tiles_m = (M + TM - 1) / TM;
    RowGroups<TM> all;
    if constexpr (GROUPED) tiles_m = all.count(first_row, groups, M);
    const int total = tiles_m * tiles_n, per_xcd = (total + 7) / 8, work = (blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
    if ((int)(blockIdx.x / 8) >= per_xcd || work >= total) return;
    constexpr int BAND = 4;
    const int band = work / (BAND * tiles_n), in_band = work - band * (BAND * tiles_n), band_rows = min(tiles_m - band * BAND, BAND);
    const int tm = band * BAND + in_band % band_rows, n0 = in_band / band_rows * TN;
    RowTile rows = {tm * TM, M, 0};
    const int nk = (nb + 7) / 8, ns = 8 * nk;                  /* k tiles, scales a row */
    if constexpr (GROUPED) {
        rows = all.tile(tm);
        W += (size_t)rows.group * N * nb * 16;
        Ws += (size_t)rows.group * N * ns;
    }
    const int m0 = rows.m0, m_end = rows.end;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4, wm = wave & 3, wn = wave >> 2;
    /* what this wave requests: 4 pieces of 8 rows of x, WP of each half of W, the scales of 64 rows of [x | W]; rows past the end of a matrix
     * repeat its last row (their outputs are never stored), pieces past the end of a stage its last piece */
    uint32_t xoff[4], woff[2][WP];
    int wpiece[WP];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int r = 8 * (4 * wave + j) + (lane >> 3);
        xoff[j] = (uint32_t)(min(m0 + r, m_end - 1) - m0) * (uint32_t)nb * 16u + 16u * ((lane & 7) ^ swizzle(r));
    }
#pragma unroll
    for (int j = 0; j < WP; j++) {
        wpiece[j] = min(WP * wave + j, 2 * NA - 1);
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int r = 8 * wpiece[j] + (lane >> 3);
            woff[half][j] = (uint32_t)(min(n0 + 16 * NA * half + r, N - 1) - n0) * (uint32_t)nb * 16u + 16u * ((lane & 7) ^ swizzle(r));
        }
    }
    const int srow = min(64 * wave, TM + TN - 64);             /* of [x | W] */
    uint32_t soff = (uint32_t)(64 * wave < TM ? min(m0 + srow + lane, m_end - 1) - m0 : min(n0 + srow - TM + lane, N - 1) - n0) * (uint32_t)ns;
    const uint8_t *x_tile = x + (size_t)m0 * nb * 16, *w_tile = W + (size_t)n0 * nb * 16;
    const int last = (nb - 8) * 16;                            /* codes of the last k tile */
    /* With one k tile a row has 8 scales, and the next row's come with them; behind the very last row there is none, it comes with the row in
     * front. (Offsets are not negative: the base is 8 bytes lower.) */
    const int one = nk == 1 ? 8 : 0, x_last = m_end == M ? M - 1 : INT_MAX, w_last = !GROUPED || rows.group == groups - 1 ? N - 1 : INT_MAX;
    const int s_most = nk == 1 ? 0 : nk - 2;
    const uint8_t *s_tile = (64 * wave < TM ? xs + (size_t)m0 * ns : Ws + (size_t)n0 * ns) - one;
    soff += (64 * wave < TM ? m0 + srow + lane >= x_last : n0 + srow - TM + lane >= w_last) ? 0 : one;
    const uint32_t lds0 = lds_address(lds);
    uint32_t lanes = ~0u;                                      /* 0 in the last two tiles, see above */
    auto load_lds = [&](uint32_t to, const uint8_t *from, uint32_t off) {
        off &= lanes;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds0 + to), "v"(off), "s"(from) : "memory", "m0");
    };
    auto request_x = [&](int j, int kt, int stage) { load_lds(stage * T::XS + (4 * wave + j) * 1024, x_tile + min(kt * 128, last), xoff[j]); };
    auto request_w = [&](int half, int j, int kt, int slot) {
        load_lds(T::W0 + slot * T::WH + wpiece[j] * 1024, w_tile + min(kt * 128, last), woff[half][j]);
    };
    /* scales of k tiles 2 p and 2 p + 1, or of the last two */
    auto request_s = [&](int p) { load_lds(T::S0 + (p & 1) * T::SC + srow * 16, s_tile + (size_t)min(2 * p, s_most) * 8, soff); };

    f32x4 acc[NA][4];                                          /* [16 columns][16 rows] */
#pragma unroll
    for (int a = 0; a < NA; a++)
#pragma unroll
        for (int b = 0; b < 4; b++) acc[a][b] = f32x4{0, 0, 0, 0};
    i32x4 av[NA], bv[2][4];                                    /* W operands of a k-step, x operands of both */
    int sa[2][NA], sb[2][4];                                   /* scales of this k tile and the next */
    int rd[2];                                                 /* bytes behind row 0 of 16 rows, by k-step */
#pragma unroll
    for (int ks = 0; ks < 2; ks++) rd[ks] = li * 128 + 16 * ((2 * lg + ks) ^ swizzle(li));
    auto read_a = [&](int ks, int a, int slot) { av[a] = *reinterpret_cast<const i32x4 *>(lds + T::W0 + slot * T::WH + 2048 * a + rd[ks]); };
    auto read_b = [&](int ks, int b, int stage) { bv[ks][b] = *reinterpret_cast<const i32x4 *>(lds + stage * T::XS + (64 * wm + 16 * b) * 128 + rd[ks]); };
    /* operand i of the first half of a k-step, in the order its products use them */
    auto read_first = [&](int ks, int i, int stage, int slot) {
        if (i == 0) read_a(ks, 0, slot);
        else if (i < 5) read_b(ks, i - 1, stage);
        else if (i < 4 + H0) read_a(ks, i - 4, slot);
    };
    const int s_rd = T::S0 + li * 16 + 2 * lg;
    auto read_scale = [&](int set, int i, int at) {            /* i: W blocks, then x blocks; at: bytes, stage and k tile of the two */
        if (i < NA) sa[set][i] = *reinterpret_cast<const uint16_t *>(lds + at + s_rd + (TM + 16 * NA * wn + 16 * i) * 16);
        else if (i < NA + 4) sb[set][i - NA] = *reinterpret_cast<const uint16_t *>(lds + at + s_rd + (64 * wm + 16 * (i - NA)) * 16);
    };
    auto products = [&](auto kstep, int set, int a0, int a1, auto &&gap) {
        constexpr int KS = decltype(kstep)::value;
#pragma unroll
        for (int g = 0; g < 4 * (a1 - a0); g++) {
            const int a = a0 + g / 4, b = g % 4;
            acc[a][b] = mfma<KS, KS>(av[a], bv[KS][b], acc[a][b], sa[set][a], sb[set][b]);
            gap(g);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    /* slot of half i of k tile t: (2 t + i) mod 5 */
    int w_slot = 0;
    auto next = [](int slot, int by) { slot += by; return slot >= 5 ? slot - 5 : slot; };
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
#pragma unroll
        for (int j = 0; j < 2 * WP; j++) request_w(j / WP, j % WP, kt, 2 * kt + j / WP);
#pragma unroll
        for (int j = 0; j < 4; j++) request_x(j, kt, kt);
        request_s(kt);
    }
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * WP + 5) : "memory");
#pragma unroll
    for (int i = 0; i < 4 + H0; i++) read_first(0, i, 0, wn);
#pragma unroll
    for (int i = 0; i < NA + 4; i++)
        read_scale(0, i, (i < NA ? n0 + 16 * (NA * wn + i) + li >= w_last : m0 + 64 * wm + 16 * (i - NA) + li >= x_last) ? one : 0);

    constexpr std::integral_constant<int, 0> k0{};
    constexpr std::integral_constant<int, 1> k1{};
    auto tile = [&](auto odd, int t) {
        constexpr int ODD = decltype(odd)::value, S1 = (NA + 4 + 1) / 2;                 /* scales read in step 0 */
        const int mine = next(w_slot, wn), far = next(w_slot, 4), after = next(w_slot, 2 + wn);
        lanes = t + 2 < nk ? ~0u : 0u;
        const int t1 = min(t + 1, nk - 1), s_at = ((t1 >> 1) & 1) * T::SC + 8 * (t1 - min(t1 & ~1, nk - 2));
        products(k0, ODD, 0, H0, [&](int g) {
            if (g < H1) read_a(0, H0 + g, mine);
            else if (g < H1 + S1) read_scale(ODD ^ 1, g - H1, s_at);
            else if (g == H1 + S1) request_w(0, 0, t + 2, far);
        });
        products(k0, ODD, H0, NA, [&](int g) {
            read_first(1, g, ODD, mine);
            if (g == 10 && ODD) request_s((t + 3) / 2);
        });
        products(k1, ODD, 0, H0, [&](int g) {
            if (g < H1) read_a(1, H0 + g, mine);
            else if (g < H1 + S1) read_scale(ODD ^ 1, S1 + g - H1, s_at);
            else if (g == H1 + S1) request_w(0, 1, t + 2, far);
        });
        /* This wave has read its last operands of the tile, and its share of the next one, and of the scales of the one after, has landed:
         * newer than that are only the requests of this tile. Behind the barrier the tile's stages are free. */
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 + ODD) : "memory");
        products(k1, ODD, H0, NA, [&](int g) {                 /* requests in the even gaps, reads in the odd ones and behind */
            if (g < 12 && g % 2 == 0) {
                if (g < 8) request_x(g / 2, t + 2, ODD);
                else request_w(1, g / 2 - 4, t + 2, w_slot);
            }
            const int i = g < 12 ? (g % 2 ? g / 2 : -1) : g - 6;
            if (i >= 0) read_first(0, i, ODD ^ 1, after);
            if (NA < 8 && g == 11) { read_first(0, 6, ODD ^ 1, after); read_first(0, 7, ODD ^ 1, after); }
        });
        w_slot = next(w_slot, 2);
    };
    int t = 0;
    for (; t + 1 < nk; t += 2) {
        tile(k0, t);
        tile(k1, t + 1);
    }
    if (t < nk) tile(k0, t);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");         /* the LDS is reused by the epilogue */

    /* acc[a][b][r] = y[m0 + 64 wm + 16 b + li][n0 + 16 NA wn + 16 a + 4 lg + r]. Through the LDS (16 KB a wave, its own region: no barrier), so
     * that a store instruction covers whole row segments. */
    constexpr int PER16 = 16 / (int)sizeof(OUT);               /* outputs per 16 B */
    const int mw = m0 + 64 * wm, nw = n0 + 16 * NA * wn;
    const bool aligned = N % PER16 == 0 && ((uintptr_t)y & 15) == 0;
    uint8_t *mine = lds + wave * 16384;
    if constexpr (sizeof(OUT) == 4) {
        float *buf = reinterpret_cast<float *>(mine);          /* 32 rows x 128 f32 at a time, chunk c of row r in slot (c & 16) | ((c ^ r) & 15) */
#pragma unroll
        for (int half = 0; half < 2; half++) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int a = 0; a < NA; a++) {
                    const int chunk = 4 * a + lg;
                    *reinterpret_cast<f32x4 *>(&buf[(16 * b + li) * 128 + 4 * ((chunk & 16) | ((chunk ^ li) & 15))]) = acc[a][2 * half + b];
                }
            auto store = [&](auto kind) {
#pragma unroll
                for (int it = 0; it < 16; it++) {
                    const int row = 2 * it + (lane >> 5), c = lane & 31, m = mw + 32 * half + row, n = nw + PER16 * c;
                    const i32x4 v = *reinterpret_cast<const i32x4 *>(&buf[row * 128 + 4 * ((c & 16) | ((c ^ row) & 15))]);
                    if (c < 4 * NA && m < m_end && n < N) store16<decltype(kind)::value>(y + (size_t)m * N + n, v, N - n);
                }
            };
            if constexpr (STREAM) store(Kind<STREAMING>{});
            else if (aligned) store(Kind<THROUGH>{});
            else store(Kind<ANY>{});
        }
    } else {
        uint16_t *buf = reinterpret_cast<uint16_t *>(mine);    /* 64 rows x 128 bf16, chunk c of row r in slot c ^ (r % 16) */
#pragma unroll
        for (int b = 0; b < 4; b++)
#pragma unroll
            for (int a = 0; a < NA; a++) {
                const int chunk = 2 * a + (lg >> 1);
                *reinterpret_cast<uint2 *>(&buf[(16 * b + li) * 128 + 8 * (chunk ^ li) + 4 * (lg & 1)]) =
                    make_uint2(pack_bf16(acc[a][b][0], acc[a][b][1]), pack_bf16(acc[a][b][2], acc[a][b][3]));
            }
        auto store = [&](auto kind) {
#pragma unroll
            for (int it = 0; it < 16; it++) {
                const int row = 4 * it + (lane >> 4), c = lane & 15, m = mw + row, n = nw + PER16 * c;
                const i32x4 v = *reinterpret_cast<const i32x4 *>(&buf[row * 128 + 8 * (c ^ (row & 15))]);
                if (c < 2 * NA && m < m_end && n < N) store16<decltype(kind)::value>(y + (size_t)m * N + n, v, N - n);
            }
        };
        if constexpr (STREAM) store(Kind<STREAMING>{});
        else if (aligned) store(Kind<THROUGH>{});
        else store(Kind<ANY>{});
    }
}

/* ---- smaller tiles ----
 *
 * WM x WN x KG waves, k tiles of 256: a wave owns 32 NB rows x 32 NA columns, and the KG waves that own the
 * same outputs take 4 / KG of the four steps of every k tile each (lanes 0 - 31 hold block s of their row in step s, lanes 32 - 63 block 4 + s,
 * so that a lane's scales are the bytes of one dword); their sums are added through the LDS at the end, in order. That keeps
 * the blocks of a wave large, i.e. few LDS reads a product, where the tile of a workgroup is small. Codes go from memory straight into a ring of
 * STAGES LDS stages, 128 B a row and k tile; 16 B chunk c of row r sits in slot c ^ ((r >> 1) & 7). Scales are fetched for eight k tiles at
 * a time, 64 B a row, into two stages of their own: what a CU can have in flight is lines, and 8 B of every row for each k tile were as many
 * lines as its codes. Part p of a row (two k tiles) sits in slot p ^ ((r >> 2) & 3). One barrier a k tile, in front of the last
 * step: behind it the tile's stage is free and is requested again, STAGES tiles ahead.
 *
 * Bound by latency, k tile after k tile: 777 x 1000 -> 1111 5.0 - 5.4 us, 512 x 9728 -> 2560 18 (from HBM 23).
 *
 * TAIL: any number of blocks, and scales at any address. Codes past the end of a row come from a line of zeros; scales go through
 * registers, 1 for blocks past the end. */
__device__ const uint4 zero_line[8] = {};                                /* what TAIL reads past the end of a row */
typedef i32x4 i32x4_at1 __attribute__((aligned(1)));

template <int NB, int NA, int WM, int WN, int KG, int STAGES>
struct Tile {
    static constexpr int TM = 32 * NB * WM, TN = 32 * NA * WN, ROWS = TM + TN, WAVES = WM * WN * KG, THREADS = 64 * WAVES;
    static constexpr int STAGE = ROWS * 128, SC = ROWS * 64, S0 = STAGES * STAGE;      /* bytes: codes of x and W of a k tile, their scales of eight */
    static constexpr int CP = (ROWS / 8 + WAVES - 1) / WAVES, SP = (ROWS / 16 + WAVES - 1) / WAVES;   /* requests of a wave: codes per k tile, scales per eight */
    static constexpr int SUMS = KG * TM * TN * 4, NEED = S0 + 2 * SC;
    static constexpr int LDS = NEED > SUMS ? NEED : SUMS;
    static_assert(LDS <= 160 * 1024 && ROWS % 32 == 0, "");
};

template <typename OUT, int NB, int NA, int WM, int WN, int KG, int STAGES, bool TAIL, bool GROUPED>
__global__ void __launch_bounds__(64 * WM * WN * KG, 2)
k_mxfp4_tiles(OUT *__restrict__ y, const uint8_t *__restrict__ x, const uint8_t *__restrict__ xs, const uint8_t *__restrict__ W,
              const uint8_t *__restrict__ Ws, int M, int N, int nb, const int *__restrict__ first_row, int groups) {
    using T = Tile<NB, NA, WM, WN, KG, STAGES>;
    constexpr int TM = T::TM, TN = T::TN, CP = T::CP, SP = T::SP, NSTEP = 4 / KG;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tiles_n = (N + TN - 1) / TN;
    int tiles_m = (M + TM - 1) / TM;
    RowGroups<TM> all;
    if constexpr (GROUPED) tiles_m = all.count(first_row, groups, M);
    const int total = tiles_m * tiles_n, per_xcd = (total + 7) / 8, work = (blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
    if ((int)(blockIdx.x / 8) >= per_xcd || work >= total) return;
    constexpr int BAND = 8;
    const int band = work / (BAND * tiles_n), in_band = work - band * (BAND * tiles_n), band_rows = min(tiles_m - band * BAND, BAND);
    const int tm = band * BAND + in_band % band_rows, n0 = in_band / band_rows * TN;
    RowTile t_rows = {tm * TM, M, 0};
    if constexpr (GROUPED) {
        t_rows = all.tile(tm);
        W += (size_t)t_rows.group * N * nb * 16;
        Ws += (size_t)t_rows.group * N * nb;
    }
    const int m0 = t_rows.m0, m_end = t_rows.end, nk = TAIL ? (nb + 7) / 8 : nb / 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l31 = lane & 31, h = lane >> 5, wm = wave % WM, wn = wave / WM % WN, kg = wave / (WM * WN);

    /* this wave's requests: 8-row pieces of codes, 16-row pieces of scales, of [x | W]; rows past the end of a matrix repeat its last row (their
     * outputs are never stored), pieces past the end of a stage its last piece */
    uint32_t coff[CP], soff[SP];
    int cpiece[CP], spiece[SP], spart;
    const uint8_t *x_tile = x + (size_t)m0 * nb * 16, *w_tile = W + (size_t)n0 * nb * 16, *xs_tile = xs + (size_t)m0 * nb, *ws_tile = Ws + (size_t)n0 * nb;
    auto row_off = [&](int r) { return (uint32_t)(r < TM ? min(m0 + r, m_end - 1) - m0 : min(n0 + r - TM, N - 1) - n0) * (uint32_t)nb; };
#pragma unroll
    for (int j = 0; j < CP; j++) {
        cpiece[j] = min(CP * wave + j, T::ROWS / 8 - 1);
        const int r = 8 * cpiece[j] + (lane >> 3);
        coff[j] = row_off(r) * 16u + 16u * ((lane & 7) ^ ((r >> 1) & 7));
    }
    spart = (lane & 3) ^ (lane >> 4);                          /* row lane / 4 of a piece, slot lane % 4 */
#pragma unroll
    for (int j = 0; j < SP; j++) {
        spiece[j] = min(SP * wave + j, T::ROWS / 16 - 1);
        soff[j] = row_off(16 * spiece[j] + (lane >> 2));
    }
    const uint32_t lds0 = lds_address(lds);
    auto request = [&](int i, int kt, int stage) {             /* piece i of this wave; past the end of K all lanes ask for one 16 B of the last tile */
        const uint32_t off = kt < nk ? coff[i] : 0u;
        if constexpr (TAIL) {
            kt = min(kt, nk - 1);
            const uint8_t *from = (cpiece[i] < TM / 8 ? x_tile : w_tile) + off + (size_t)kt * 128;
            const int r = 8 * cpiece[i] + (lane >> 3);
            if (8 * kt + ((lane & 7) ^ ((r >> 1) & 7)) >= nb) from = reinterpret_cast<const uint8_t *>(zero_line);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds0 + stage * T::STAGE + cpiece[i] * 1024), "v"(from) : "memory", "m0");
            return;
        }
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     ::"s"(lds0 + stage * T::STAGE + cpiece[i] * 1024), "v"(off), "s"((cpiece[i] < TM / 8 ? x_tile : w_tile) + (size_t)min(kt, nk - 1) * 128)
                     : "memory", "m0");
    };
    /* scales of k tiles 8 c .. 8 c + 7: part p is tiles 8 c + 2 p and the next, or the last two (there are two) */
    auto request_scales = [&](int c) {
        if constexpr (TAIL) {
            for (int i = tid; i < T::ROWS * 4; i += T::THREADS) {
                const int r = i >> 2, part = (i & 3) ^ ((r >> 2) & 3), b0 = 64 * c + 16 * part, left = nb - b0;
                const uint8_t *from = (r < TM ? xs_tile : ws_tile) + row_off(r) + b0;
                i32x4 v = {0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f};
                if (left >= 16) {
                    v = *reinterpret_cast<const i32x4_at1 *>(from);
                } else {
#pragma unroll
                    for (int k = 0; k < 16; k++)
                        if (k < left) v[k >> 2] ^= (0x7f ^ (int)from[k]) << (8 * (k & 3));
                }
                *reinterpret_cast<i32x4 *>(lds + T::S0 + (c & 1) * T::SC + i * 16) = v;
            }
            return;
        }
        const int part_off = min(8 * c + 2 * spart, nk - 2) * 8;
#pragma unroll
        for (int j = 0; j < SP; j++)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                         ::"s"(lds0 + T::S0 + (c & 1) * T::SC + spiece[j] * 1024), "v"(soff[j] + part_off), "s"(spiece[j] < TM / 16 ? xs_tile : ws_tile) : "memory", "m0");
    };

    f32x16 acc[NA][NB];
#pragma unroll
    for (int a = 0; a < NA; a++)
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[a][b][r] = 0.0f;
    i32x4 av[2][NA], bv[2][NB];
    int sa[2][NA], sb[2][NB];
    int rd[NSTEP];
#pragma unroll
    for (int s = 0; s < NSTEP; s++) rd[s] = l31 * 128 + 16 * ((4 * h + NSTEP * kg + s) ^ ((l31 >> 1) & 7));
    const int s_rd = T::S0 + l31 * 64 + 4 * h, s_slot = ((l31 >> 2) & 3) * 16;
    constexpr int OPS = NA + NB;
    auto read_operand = [&](int set, int s, int i, int stage) {
        const uint8_t *from = lds + stage * T::STAGE + rd[s];
        if (i < NB) bv[set][i] = *reinterpret_cast<const i32x4 *>(from + 32 * (NB * wm + i) * 128);
        else av[set][i - NB] = *reinterpret_cast<const i32x4 *>(from + (TM + 32 * (NA * wn + i - NB)) * 128);
    };
    auto scales_at = [&](int kt) {                             /* bytes to row 0's scales of a k tile */
        kt = min(kt, nk - 1);
        return s_rd + ((kt >> 3) & 1) * T::SC + (((kt >> 1) & 3) * 16 ^ s_slot) + 8 * (TAIL ? kt & 1 : kt - min(kt & ~1, nk - 2));
    };
    auto read_scale = [&](int set, int i, int at) {
        if (i < NB) sb[set][i] = *reinterpret_cast<const int *>(lds + at + 32 * (NB * wm + i) * 64) >> (8 * NSTEP * kg);
        else sa[set][i - NB] = *reinterpret_cast<const int *>(lds + at + (TM + 32 * (NA * wn + i - NB)) * 64) >> (8 * NSTEP * kg);
    };
    auto step = [&](auto which, int set, int sset, auto &&gap) {
        constexpr int S = decltype(which)::value;
#pragma unroll
        for (int g = 0; g < NA * NB; g++) {
            acc[g / NB][g % NB] = mfma32<S, S>(av[set][g / NB], bv[set][g % NB], acc[g / NB][g % NB], sa[sset][g / NB], sb[sset][g % NB]);
            gap(g);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    request_scales(0);
#pragma unroll
    for (int t = 0; t < STAGES; t++)
#pragma unroll
        for (int i = 0; i < CP; i++) request(i, t, t);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 1) * CP) : "memory");
    {
        const int at = scales_at(0);
#pragma unroll
        for (int i = 0; i < OPS; i++) { read_operand(0, 0, i, 0); read_scale(0, i, at); }
    }
    int cur = 0;
    /* NSTEP is 1, 2 or 4: operand sets alternate by step, so by tile where there is one step, and scale sets by tile */
    auto tile = [&](auto odd, int t) {
        constexpr int ODD = decltype(odd)::value;
        const int nxt = cur + 1 == STAGES ? 0 : cur + 1, s_at = scales_at(t + 1);
        auto inner = [&](auto s) {
            constexpr int S = decltype(s)::value;
            if constexpr (S + 1 < NSTEP)
                step(s, S & 1, ODD, [&](int g) {
#pragma unroll
                    for (int i = g * OPS / (NA * NB); i < (g + 1) * OPS / (NA * NB); i++) read_operand((S & 1) ^ 1, S + 1, i, cur);
                });
        };
        inner(std::integral_constant<int, 0>{});
        inner(std::integral_constant<int, 1>{});
        inner(std::integral_constant<int, 2>{});
        /* This wave has read its last operands of the tile, and its share of the next one has landed: of its requests only those for later tiles
         * are newer, and scales for much later ones. Those of eight tiles on are requested in the first of eight, when the stage's last readers
         * have passed the barrier. */
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * CP) : "memory");
        if ((t & 7) == 0 && t + 8 < nk) request_scales((t >> 3) + 1);
        constexpr int LAST = NSTEP - 1, SET = NSTEP == 1 ? ODD : LAST & 1, ALL = 2 * OPS + CP;
        step(std::integral_constant<int, LAST>{}, SET, ODD, [&](int g) {
#pragma unroll
            for (int i = g * ALL / (NA * NB); i < (g + 1) * ALL / (NA * NB); i++) {
                if (i < OPS) read_operand(NSTEP == 1 ? ODD ^ 1 : 0, 0, i, nxt);
                else if (i < 2 * OPS) read_scale(ODD ^ 1, i - OPS, s_at);
                else request(i - 2 * OPS, t + STAGES, cur);
            }
        });
        cur = nxt;
    };
    int t = 0;
    for (; t + 1 < nk; t += 2) {
        tile(std::integral_constant<int, 0>{}, t);
        tile(std::integral_constant<int, 1>{}, t + 1);
    }
    if (t < nk) tile(std::integral_constant<int, 0>{}, t);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");         /* the ring is free */

    /* acc[a][b][4 q + r] = y[32 (NB wm + b) + l31][32 (NA wn + a) + 8 q + 4 h + r]: as f32 rows of the tile, one copy per k group, chunk c of four
     * of row r in slot c ^ (r % 16), c ^ (r % 8) where a row has 8 */
    constexpr int SWZ = TN >= 64 ? 15 : 7;
    float *sums = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int a = 0; a < NA; a++)
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int row = 32 * (NB * wm + b) + l31, c = 8 * (NA * wn + a) + 2 * q + h;
                *reinterpret_cast<f32x4 *>(&sums[(kg * TM + row) * TN + 4 * (c ^ (row & SWZ))]) =
                    f32x4{acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]};
            }
    __syncthreads();
    auto sum = [&](int row, int c) {
        const float *from = &sums[row * TN + 4 * (c ^ (row & SWZ))];
        f32x4 v = *reinterpret_cast<const f32x4 *>(from);
#pragma unroll
        for (int k = 1; k < KG; k++) v += *reinterpret_cast<const f32x4 *>(from + k * TM * TN);
        return v;
    };
    constexpr int CHUNKS = sizeof(OUT) == 4 ? 1 : 2, ACROSS = TN / 4 / CHUNKS;        /* chunks of four a thread stores at a time */
    const bool aligned = N % (4 * CHUNKS) == 0 && ((uintptr_t)y & 15) == 0;
    auto store = [&](auto kind) {
#pragma unroll 4
        for (int i = tid; i < TM * ACROSS; i += T::THREADS) {
            const int row = i / ACROSS, c = i % ACROSS * CHUNKS, m = m0 + row, n = n0 + 4 * c;
            if (m >= m_end || n >= N) continue;
            const f32x4 v = sum(row, c);
            i32x4 r = __builtin_bit_cast(i32x4, v);
            if constexpr (CHUNKS == 2) {
                const f32x4 w = sum(row, c + 1);
                r = i32x4{(int)pack_bf16(v[0], v[1]), (int)pack_bf16(v[2], v[3]), (int)pack_bf16(w[0], w[1]), (int)pack_bf16(w[2], w[3])};
            }
            store16<decltype(kind)::value>(y + (size_t)m * N + n, r, N - n);
        }
    };
    if (aligned) store(Kind<THROUGH>{});
    else store(Kind<ANY>{});
}
#pragma clang diagnostic pop

/* rows of nb scales to rows of 8 bytes a k tile: M of xs, behind them those of Ws, `rows` in all; see k_mxfp4_wide */
__global__ void __launch_bounds__(256)
k_mxfp4_scales(uint64_t *__restrict__ to, const uint8_t *__restrict__ xs, const uint8_t *__restrict__ Ws, int M, size_t rows, int nb) {
    const int nk = (nb + 7) / 8, over = 8 * nk - nb;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, row = i / nk;
    if (row >= rows) return;
    const int kt = (int)(i - row * nk), skip = kt == nk - 1 ? over : 0;
    const uint8_t *from = (row < (size_t)M ? xs + row * nb : Ws + (row - M) * nb) + (kt == nk - 1 ? nb - 8 : 8 * kt);
    uint64_t v = 0;
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (j >= skip) v |= (uint64_t)from[j] << (8 * j);
    to[i] = v;
}

/* the arguments of every kernel here */
#define KERNEL_ARGS y, x, xs, W, Ws, M, N, nb, first_row, groups
#define KERNEL_PARAMS OUT *y, const uint8_t *x, const uint8_t *xs, const uint8_t *W, const uint8_t *Ws, int M, int N, int nb, const int *first_row, int groups

template <bool GROUPED>
long tiles_at_most(int M, int N, int groups, int tm, int tn) {
    return (GROUPED ? row_tiles_at_most(M, groups, tm) : ((long)M + tm - 1) / tm) * ((N + tn - 1L) / tn);
}

/* Results leave the L2s as they are stored (write_through.h), those of 100 MB and more past the Infinity Cache (256 MB) too, with the streaming hint: it then
 * keeps the operands. us, plain / through, and with the conversion of the result to MXFP4 behind: 512 x 2560 -> 19456 19.0 / 18.2 and 25.2 / 24.6,
 * 2115 x 4096 -> 4096 25.2 / 24.4 and 30.8 / 29.9, 1000 x 1024 -> 9216 11.7 / 10.4 and 17.6 / 16.9, 300 x 512 -> 4096 6.0 / 6.0 and 10.4 / 10.2. Through / streaming:
 * 4608 x 4096 -> 36864 (340 MB) 387 / 363 (weights from HBM 380 / 366) and 446 / 440, -> 12288 (113 MB) 133 / 129 (131 / 131) and 154 / 155, in two groups 150 / 130 (150 / 149); f32
 * 36864 450 / 413, 9000 x 1024 -> 4096 (147 MB) 51.4 / 49.0; unaligned rows not: 4608 x 2560 -> 16001 130 / 142. Kernels of their own: of a test in front of two stores to one place the compiler keeps one, the plain one. */
constexpr size_t STREAM_BYTES = (size_t)100 << 20;

/* part: room for the copy of the scales, NULL where they can be read as they are */
template <typename OUT, int NA, bool GROUPED, bool STREAM = false>
int launch_wide(hipStream_t st, void *part, KERNEL_PARAMS) {
    if constexpr (!STREAM)
        if ((size_t)M * N * sizeof(OUT) >= STREAM_BYTES && N % (16 / sizeof(OUT)) == 0 && ((uintptr_t)y & 15) == 0) return launch_wide<OUT, NA, GROUPED, true>(st, part, KERNEL_ARGS);
    using T = Wide<NA>;
    static bool configured = false;
    if (!configured) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(k_mxfp4_wide<OUT, NA, STREAM, GROUPED>), hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
        if (e != hipSuccess) return (int)e;
        configured = true;
    }
    const long most = tiles_at_most<GROUPED>(M, N, groups, T::TM, T::TN);
    if (!launch_fits(most, 512)) return (int)hipErrorInvalidValue;
    if (part) {
        const size_t all = (size_t)M + (size_t)groups * N, nk = (size_t)(nb + 7) / 8;
        hipLaunchKernelGGL(k_mxfp4_scales, dim3((unsigned)((all * nk + 255) / 256)), dim3(256), 0, st, (uint64_t *)part, xs, Ws, M, all, nb);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
        xs = (const uint8_t *)part;
        Ws = xs + M * nk * 8;
    }
    hipLaunchKernelGGL((k_mxfp4_wide<OUT, NA, STREAM, GROUPED>), dim3((unsigned)(most + 7) / 8 * 8), dim3(512), T::LDS, st, KERNEL_ARGS);
    return (int)hipGetLastError();
}

template <typename OUT, bool TAIL, bool GROUPED, int NB, int NA, int WM, int WN, int KG, int STAGES>
int launch_tiles(hipStream_t st, KERNEL_PARAMS) {
    using T = Tile<NB, NA, WM, WN, KG, STAGES>;
    static bool configured = false;
    if (!configured) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(k_mxfp4_tiles<OUT, NB, NA, WM, WN, KG, STAGES, TAIL, GROUPED>),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
        if (e != hipSuccess) return (int)e;
        configured = true;
    }
    const long most = tiles_at_most<GROUPED>(M, N, groups, T::TM, T::TN);
    if (!launch_fits(most, T::THREADS)) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((k_mxfp4_tiles<OUT, NB, NA, WM, WN, KG, STAGES, TAIL, GROUPED>), dim3((unsigned)(most + 7) / 8 * 8), dim3(T::THREADS), T::LDS, st, KERNEL_ARGS);
    return (int)hipGetLastError();
}

template <typename OUT, int A, bool GROUPED>
int launch_rows(hipStream_t st, KERNEL_PARAMS) {
    const long most = tiles_at_most<GROUPED>(M, N, groups, 16, 16 * A);
    if (!launch_fits(most, 64 * ROWS_KW)) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((k_mxfp4_rows<OUT, A, GROUPED>), dim3((unsigned)(most + 7) / 8 * 8), dim3(64 * ROWS_KW), 0, st, KERNEL_ARGS);
    return (int)hipGetLastError();
}

/* Estimated times in us. A workgroup's k tile takes `step` where workgroups have a CU to themselves and `share` for each of those on its CU where they
 * are more; `fixed` is the launch, the first tiles and the end, `again` what a further round of the resident ones takes more. Fitted to
 * 190 sizes (1 - 4608 rows, 512 -> 512 to 16384 -> 1024 and 2560 -> 19456): what is chosen takes 1.7 % longer on average than the best of 17 tiles,
 * 20 % at worst, with operands from the caches. The times are there to be compared: as the clock falls with the work, large layers take longer (4608 x 4096 -> 36864
 * 280, measured 359; 512 + 4096 rows -> 12288 101, 130). us, best others / chosen: 512 x 9728 -> 2560 (64 x 128) 23.2 / 18.3, 64 x 9728 -> 2560 (32 x 32) 11.2 / 8.8, 512 x 4096 ->
 * 12288 (256 x 192) 30.8 / 23.2, 2115 x 4096 -> 12288 (256 x 256) 73.4 / 61.6. */
struct Shape { int tm, tn, threads, resident; float fixed, step, share, again; };
constexpr Shape SHAPES[] = {{32, 32, 256, 4, 3.36f, 0.129f, 0.098f, 1.6f},   {64, 64, 256, 2, 3.87f, 0.257f, 0.214f, 2.5f},  {64, 128, 256, 1, 4.16f, 0.344f, 0.354f, 3.2f},
                            {128, 128, 512, 1, 4.85f, 0.205f, 0.455f, 5.5f}, {256, 192, 512, 1, 5.0f, 0.326f, 0.973f, 6.0f}, {256, 256, 512, 1, 5.16f, 0.635f, 1.22f, 6.0f}};
constexpr int NSHAPES = sizeof(SHAPES) / sizeof(SHAPES[0]), FIRST_WIDE = 4;

/* -1 and -2: k_mxfp4_rows with that many blocks of columns, 0 - 3: k_mxfp4_tiles, 4 and 5: k_mxfp4_wide, in the order of SHAPES. whole: rows of whole k tiles
 * and aligned scales; otherwise k_mxfp4_wide needs part_bytes of workspace for a copy of the scales and 4 us more, and, as with one k tile, k_mxfp4_tiles runs
 * in its form for rows of any length, whose k tiles take a third and whose further rounds twice as long. */
int plan_mxfp4(int groups, int M, int N, int nb, bool whole, size_t part_bytes) {
    const bool tail = !whole || nb < 16;
    const size_t copy = ((size_t)M + (size_t)groups * N) * ((nb + 7) / 8 * 8);
    const bool wide = M >= 256 && N >= 192 && nb >= 8 && (whole || copy <= part_bytes);
    const float first = whole ? 0.0f : 4.0f + 2.0f * (float)copy / 2.5e6f;
    const long some = groups < M ? groups : M;
    auto row_tiles = [&](int tm) { return groups == 1 ? ((long)M + tm - 1) / tm : row_tiles_about(M, groups, tm); };
    const float weights = 17.0f * (float)nb * (float)N, fresh = (float)some * weights / 5.0e6f;    /* HBM's 5 TB/s */
    /* k_mxfp4_rows: a step of a wave 1 us, W once for every 16 rows at 5.5 TB/s (from the Infinity Cache), a workgroup 1.15 ns */
    const float steps = (float)(((nb + 15) / 16 + ROWS_KW - 1) / ROWS_KW), read = (float)row_tiles(16) * weights / 5.5e6f;
    const float starts = 1.15e-3f * (float)row_tiles(16) * (float)((N + 15L) / 16), most = steps > read ? steps : read;
    float best = 2.2f + (most > starts ? most : starts);
    if (best < 2.2f + fresh) best = 2.2f + fresh;
    /* two blocks of columns: 40 rows over 64 weight matrices of 2560 -> 1536 13.9 us with one, 12.7 with two; 1 row, 4096 -> 4096 3.7 / 4.9 */
    int plan = row_tiles(16) * ((N + 31L) / 32) >= 512 ? -2 : -1;
    /* kernels whose grid could pass the limit of a launch are left out */
    auto fits = [&](int tm, int tn, int threads) { return launch_fits(row_tiles_at_most(M, groups, tm) * ((N + tn - 1L) / tn), threads); };
    if (!fits(16, -16 * plan, 64 * ROWS_KW)) best = FLT_MAX;
    /* the tiles' offsets inside a tile of rows have 32 bits */
    for (int i = 0; i < (nb >> 20 ? 0 : wide ? NSHAPES : FIRST_WIDE); i++) {
        const Shape &s = SHAPES[i];
        const long wgs = row_tiles(s.tm) * ((N + s.tn - 1L) / s.tn), each = (wgs + 255) / 256, rounds = (wgs + 256L * s.resident - 1) / (256L * s.resident);
        const float shared = s.share * (float)each, step = shared > s.step ? shared : s.step;
        const bool slower = tail && i < FIRST_WIDE;
        float us = s.fixed + (float)((nb + 7) / 8) * step * (slower ? 1.3f : 1.0f) + (float)(rounds - 1) * s.again * (slower ? 2.0f : 1.0f);
        if (us < s.fixed + fresh) us = s.fixed + fresh;
        if (i >= FIRST_WIDE) us += first;
        if (us < best && fits(s.tm, s.tn, s.threads)) { best = us; plan = i; }
    }
    return plan;
}

template <typename OUT, bool TAIL, bool GROUPED>
int launch_shape(int shape, hipStream_t st, KERNEL_PARAMS) {
    switch (shape) {
    case 0: return launch_tiles<OUT, TAIL, GROUPED, 1, 1, 1, 1, 4, 4>(st, KERNEL_ARGS);
    case 1: return launch_tiles<OUT, TAIL, GROUPED, 2, 2, 1, 1, 4, 3>(st, KERNEL_ARGS);
    case 2: return launch_tiles<OUT, TAIL, GROUPED, 2, 2, 1, 2, 2, 3>(st, KERNEL_ARGS);
    case 3: return launch_tiles<OUT, TAIL, GROUPED, 2, 2, 2, 2, 2, 3>(st, KERNEL_ARGS);
    default: return (int)hipErrorInvalidValue;
    }
}

template <typename OUT, bool GROUPED>
int linear(hipStream_t st, void *part, KERNEL_PARAMS) {
    const bool whole = nb % 8 == 0 && (((uintptr_t)xs | (uintptr_t)Ws) & 7) == 0;
    const int plan = plan_mxfp4(groups, M, N, nb, whole, part ? IRIS_LINEAR_PART_BYTES : 0);
    if (plan == -1) return launch_rows<OUT, 1, GROUPED>(st, KERNEL_ARGS);
    if (plan == -2) return launch_rows<OUT, 2, GROUPED>(st, KERNEL_ARGS);
    if (whole) part = nullptr;
    if (plan == 5) return launch_wide<OUT, 8, GROUPED>(st, part, KERNEL_ARGS);
    if (plan == 4) return launch_wide<OUT, 6, GROUPED>(st, part, KERNEL_ARGS);
    return !whole || nb < 16 ? launch_shape<OUT, true, GROUPED>(plan, st, KERNEL_ARGS) : launch_shape<OUT, false, GROUPED>(plan, st, KERNEL_ARGS);
}

template <typename OUT>
int linear(void *stream, void *part, OUT *y, const uint8_t *x, const uint8_t *xs, const uint8_t *W, const uint8_t *Ws, const int *first_row, int groups, int rows, int in, int out) {
    const int nb = (int)(((long)in + 31) / 32);
    return first_row ? linear<OUT, true>((hipStream_t)stream, part, y, x, xs, W, Ws, rows, out, nb, first_row, groups)
                     : linear<OUT, false>((hipStream_t)stream, part, y, x, xs, W, Ws, rows, out, nb, nullptr, 1);
}

}  // namespace

extern "C" {

/* The kernel a layer of these sizes takes with aligned operands, as plan_mxfp4 numbers them. No GPU needed. */
int iris_hip_linear_mxfp4_plan(int groups, int rows, int in, int out) {
    const int nb = (int)(((long)in + 31) / 32);
    return plan_mxfp4(groups, rows, out, nb, nb % 8 == 0, IRIS_LINEAR_PART_BYTES);
}

int iris_hip_linear_mxfp4_f32(void *stream, float *part, float *y, const uint8_t *x, const uint8_t *xs, const uint8_t *W, const uint8_t *Ws, const int *first_row,
                              int groups, int rows, int in, int out) {
    return linear(stream, part, y, x, xs, W, Ws, first_row, groups, rows, in, out);
}
int iris_hip_linear_mxfp4_bf16(void *stream, float *part, uint16_t *y, const uint8_t *x, const uint8_t *xs, const uint8_t *W, const uint8_t *Ws, const int *first_row, int groups,
                               int rows, int in, int out) {
    return linear(stream, part, y, x, xs, W, Ws, first_row, groups, rows, in, out);
}

}  // extern "C"
