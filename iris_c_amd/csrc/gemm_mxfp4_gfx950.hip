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
#include <type_traits>

#include "iris_kernels_hip.h"
#include "row_groups.h"

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


/* ---- tiles of 256 rows x 256 or 192 columns ----
 *
 * For whole k tiles of 256 (in a multiple of 256, two at least): a k tile is 128 B of codes and 8 scales of every row. Eight waves, two per
 * SIMD, 4 (rows of 64) x 2 (columns of 32 NA): a wave owns 64 rows x 32 NA columns = NA x 2 accumulator blocks of 32 x 32. A k tile is
 * four steps of v_mfma_scale_f32_32x32x64: in step s lanes 0 - 31 hold block s of their row, lanes 32 - 63 block 4 + s, so that a
 * lane's four scales are the bytes of one dword.
 *
 * Everything comes from memory straight into the LDS (160 KB at 256 columns): two stages of x, two and a half of W (a ring of five half
 * tiles, the columns of one wave column each), two of scales, which are fetched for two k tiles at a time (16 B a row). 16 B chunk c of row r
 * sits in slot c ^ ((r >> 1) & 7): the 16 lanes that the LDS serves together on a 128-bit read (eight pairs of neighbouring rows, of
 * different slots) fall on different banks. Codes of k tile t + 2: the first half of W in steps 0 and 1 of tile t, the rest in step 3,
 * behind the one barrier of a tile, which frees the stage. The operands of a step are read during the step before, the scales of the
 * next tile during steps 0 - 2. Every memory instruction stands in a gap between two products; requests past the
 * end of K ask for the last tile again, into a stage that nobody reads. */
template <int NA>
struct Wide {
    static constexpr int TM = 256, TN = 64 * NA;
    static constexpr int XS = TM * 128, WH = TN / 2 * 128, SC = (TM + TN) * 16;      /* bytes: a stage of x, half of one of W, scales of two k tiles */
    static constexpr int W0 = 2 * XS, S0 = W0 + 5 * WH, LDS = S0 + 2 * SC;
    static_assert(LDS <= 160 * 1024 && LDS >= 128 * 1024, "the epilogue takes 128 KB");
};

__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"                          /* M0 in a clobber list */
template <typename OUT, int NA, bool GROUPED>
__global__ void __launch_bounds__(512, 2)
k_mxfp4_wide(OUT *__restrict__ y, const uint8_t *__restrict__ x, const uint8_t *__restrict__ xs, const uint8_t *__restrict__ W,
             const uint8_t *__restrict__ Ws, int M, int N, int nb, const int *__restrict__ first_row, int groups) {
    using T = Wide<NA>;
    constexpr int TM = T::TM, TN = T::TN;
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
    RowTile t_rows = {tm * TM, M, 0};
    if constexpr (GROUPED) {
        t_rows = all.tile(tm);
        W += (size_t)t_rows.group * N * nb * 16;
        Ws += (size_t)t_rows.group * N * nb;
    }
    const int m0 = t_rows.m0, m_end = t_rows.end, nk = nb / 8;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l31 = lane & 31, h = lane >> 5, wm = wave & 3, wn = wave >> 2;
    /* the 8-row pieces of codes and the 64 rows of scales that this wave fetches; rows past the end of a matrix repeat its last row (their
     * outputs are never stored), pieces past the end of a stage its last piece */
    constexpr int WP = (4 * NA + 7) / 8;                       /* pieces of half of W per wave */
    uint32_t xoff[4], woff[2][WP], soff;
    int wpiece[WP];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int r = 8 * (4 * wave + j) + (lane >> 3);
        xoff[j] = (uint32_t)(min(m0 + r, m_end - 1) - m0) * (uint32_t)nb * 16u + 16u * ((lane & 7) ^ ((r >> 1) & 7));
    }
#pragma unroll
    for (int j = 0; j < WP; j++) {
        wpiece[j] = min(WP * wave + j, 4 * NA - 1);
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int r = 32 * NA * half + 8 * wpiece[j] + (lane >> 3);
            woff[half][j] = (uint32_t)(min(n0 + r, N - 1) - n0) * (uint32_t)nb * 16u + 16u * ((lane & 7) ^ ((r >> 1) & 7));
        }
    }
    const int srow = min(64 * wave, TM + TN - 64);             /* of [x | W] */
    soff = (uint32_t)(srow < TM ? min(m0 + srow + lane, m_end - 1) - m0 : min(n0 + srow - TM + lane, N - 1) - n0) * (uint32_t)nb;
    const uint8_t *x_tile = x + (size_t)m0 * nb * 16, *w_tile = W + (size_t)n0 * nb * 16;
    const uint8_t *s_tile = srow < TM ? xs + (size_t)m0 * nb : Ws + (size_t)n0 * nb;
    const uint32_t lds0 = lds_address(lds);
    auto load_lds = [&](uint32_t to, const uint8_t *from, uint32_t off) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds0 + to), "v"(off), "s"(from) : "memory", "m0");
    };
    auto request_x = [&](int j, int kt) { load_lds((kt & 1) * T::XS + (4 * wave + j) * 1024, x_tile + (size_t)min(kt, nk - 1) * 128, xoff[j]); };
    auto request_w = [&](int half, int j, int kt, int slot) {
        load_lds(T::W0 + slot * T::WH + wpiece[j] * 1024, w_tile + (size_t)min(kt, nk - 1) * 128, woff[half][j]);
    };
    /* scales of k tiles 2 p and 2 p + 1, or of the last two */
    auto request_s = [&](int p) { load_lds(T::S0 + (p & 1) * T::SC + srow * 16, s_tile + (size_t)min(2 * p, nk - 2) * 8, soff); };

    f32x16 acc[NA][2];                                         /* [32 columns][32 rows] */
#pragma unroll
    for (int a = 0; a < NA; a++)
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[a][b][r] = 0.0f;
    i32x4 av[2][NA], bv[2][2];                                 /* of this step and the next */
    int sa[2][NA], sb[2][2];                                   /* of this k tile and the next */
    int rd[4];                                                 /* bytes behind row 0 of a block of 32 rows, by step */
#pragma unroll
    for (int s = 0; s < 4; s++) rd[s] = l31 * 128 + 16 * ((4 * h + s) ^ ((l31 >> 1) & 7));
    /* operand i of a step, in the order the products use them: W block 0, both x blocks, the other W blocks */
    auto read_operand = [&](int set, int s, int i, int xstage, int wslot) {
        if (i == 1 || i == 2) bv[set][i - 1] = *reinterpret_cast<const i32x4 *>(lds + xstage * T::XS + (64 * wm + 32 * (i - 1)) * 128 + rd[s]);
        else av[set][i ? i - 2 : 0] = *reinterpret_cast<const i32x4 *>(lds + T::W0 + wslot * T::WH + (i ? i - 2 : 0) * 4096 + rd[s]);
    };
    const int s_rd = l31 * 16 + 4 * h;
    auto read_scale = [&](int set, int i, int kt) {            /* i: W blocks, then x blocks */
        kt = min(kt, nk - 1);
        const int start = min(kt & ~1, nk - 2), at = T::S0 + ((kt >> 1) & 1) * T::SC + 8 * (kt - start) + s_rd;
        if (i < NA) sa[set][i] = *reinterpret_cast<const int *>(lds + at + (TM + 32 * NA * wn + 32 * i) * 16);
        else sb[set][i - NA] = *reinterpret_cast<const int *>(lds + at + (64 * wm + 32 * (i - NA)) * 16);
    };
    auto product = [&](auto step, int set, int sset, int a, int b) {
        constexpr int S = decltype(step)::value;
        acc[a][b] = mfma32<S, S>(av[set][a], bv[set][b], acc[a][b], sa[sset][a], sb[sset][b]);
    };
    auto step = [&](auto which, int set, int sset, auto &&gap) {
#pragma unroll
        for (int g = 0; g < 2 * NA; g++) {
            product(which, set, sset, g / 2, g % 2);
            gap(g);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr int OPS = NA + 2;                                /* operands of a step, scales of a tile */

    /* slot of half i of k tile t: (2 t + i) mod 5 */
    int w_slot = 0;
    auto next = [](int slot, int by) { slot += by; return slot >= 5 ? slot - 5 : slot; };
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int j = 0; j < WP; j++) request_w(half, j, kt, 2 * kt + half);
#pragma unroll
        for (int j = 0; j < 4; j++) request_x(j, kt);
        request_s(kt);
    }
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * WP + 5) : "memory");
#pragma unroll
    for (int i = 0; i < OPS; i++) read_operand(0, 0, i, 0, wn);
#pragma unroll
    for (int i = 0; i < OPS; i++) read_scale(0, i, 0);

    auto tile = [&](auto odd, int t) {
        constexpr int ODD = decltype(odd)::value;
        const int mine = next(w_slot, wn), far = next(w_slot, 4), then = next(w_slot, 2 + wn);
        step(std::integral_constant<int, 0>{}, 0, ODD, [&](int g) {
            if (g < OPS) read_operand(1, 1, g, t & 1, mine);
            else if (g == OPS) request_w(0, 0, t + 2, far);
            if (g < 2) read_scale(ODD ^ 1, g, t + 1);
        });
        step(std::integral_constant<int, 1>{}, 1, ODD, [&](int g) {
            if (g < OPS) read_operand(0, 2, g, t & 1, mine);
            else if (g == OPS && WP > 1) request_w(0, 1, t + 2, far);
            if (g < 2) read_scale(ODD ^ 1, 2 + g, t + 1);
        });
        step(std::integral_constant<int, 2>{}, 0, ODD, [&](int g) {
            if (g < OPS) read_operand(1, 3, g, t & 1, mine);
            else if (g == OPS && ODD) request_s((t + 1) / 2 + 1);
            if (g < 2 && 4 + g < OPS) read_scale(ODD ^ 1, 4 + g, t + 1);
        });
        /* This wave has read its last operands of the tile, and its share of the next one, and of the scales of the one after, has landed:
         * newer than that are only the requests of this tile. Behind the barrier the tile's stages are free. */
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(WP + ODD) : "memory");
        step(std::integral_constant<int, 3>{}, 1, ODD, [&](int g) {
            if (g < 4) request_x(g, t + 2);
            else if (g < 4 + WP) request_w(1, g - 4, t + 2, w_slot);
            if (g < OPS) read_operand(0, 0, g, (t & 1) ^ 1, then);
        });
        w_slot = next(w_slot, 2);
    };
    int t = 0;
    for (; t + 1 < nk; t += 2) {
        tile(std::integral_constant<int, 0>{}, t);
        tile(std::integral_constant<int, 1>{}, t + 1);
    }
    if (t < nk) tile(std::integral_constant<int, 0>{}, t);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");         /* the LDS is reused by the epilogue */

    /* acc[a][b][4 q + r] = y[m0 + 64 wm + 32 b + l31][n0 + 32 NA wn + 32 a + 8 q + 4 h + r]. Through the LDS (16 KB a wave, its own region: no
     * barrier), so that a store instruction covers whole row segments. */
    constexpr int PER16 = 16 / (int)sizeof(OUT);               /* outputs per 16 B; the launcher has N a multiple of it */
    const int mw = m0 + 64 * wm, nw = n0 + 32 * NA * wn;
    uint8_t *mine = lds + wave * 16384;
    if constexpr (sizeof(OUT) == 4) {
        float *buf = reinterpret_cast<float *>(mine);          /* 32 rows x 128 f32 at a time, chunk c of row r in slot (c & 16) | ((c ^ r) & 15) */
#pragma unroll
        for (int b = 0; b < 2; b++) {
#pragma unroll
            for (int a = 0; a < NA; a++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int chunk = 8 * a + 2 * q + h;
                    *reinterpret_cast<f32x4 *>(&buf[l31 * 128 + 4 * ((chunk & 16) | ((chunk ^ l31) & 15))]) =
                        f32x4{acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]};
                }
#pragma unroll
            for (int it = 0; it < 16; it++) {
                const int row = 2 * it + (lane >> 5), c = lane & 31, m = mw + 32 * b + row, n = nw + PER16 * c;
                const f32x4 v = *reinterpret_cast<const f32x4 *>(&buf[row * 128 + 4 * ((c & 16) | ((c ^ row) & 15))]);
                if (c < 8 * NA && m < m_end && n < N) *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(y) + (size_t)m * N + n) = v;
            }
        }
    } else {
        uint16_t *buf = reinterpret_cast<uint16_t *>(mine);    /* 64 rows x 128 bf16, chunk c of row r in slot c ^ (r % 16) */
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int a = 0; a < NA; a++)
#pragma unroll
                for (int q = 0; q < 4; q++)
                    *reinterpret_cast<uint2 *>(&buf[(32 * b + l31) * 128 + 8 * ((4 * a + q) ^ (l31 & 15)) + 4 * h]) =
                        make_uint2(pack_bf16(acc[a][b][4 * q], acc[a][b][4 * q + 1]), pack_bf16(acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]));
#pragma unroll
        for (int it = 0; it < 16; it++) {
            const int row = 4 * it + (lane >> 4), c = lane & 15, m = mw + row, n = nw + PER16 * c;
            const i32x4 v = *reinterpret_cast<const i32x4 *>(&buf[row * 128 + 8 * (c ^ (row & 15))]);
            if (c < 4 * NA && m < m_end && n < N) *reinterpret_cast<i32x4 *>(reinterpret_cast<uint16_t *>(y) + (size_t)m * N + n) = v;
        }
    }
}
#pragma clang diagnostic pop

template <typename OUT, int NA, bool GROUPED>
int launch_wide(hipStream_t st, OUT *y, const uint8_t *x, const uint8_t *xs, const uint8_t *W, const uint8_t *Ws, int M, int N, int nb, const int *first_row, int groups) {
    static bool configured = false;
    if (!configured) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(k_mxfp4_wide<OUT, NA, GROUPED>), hipFuncAttributeMaxDynamicSharedMemorySize, Wide<NA>::LDS);
        if (e != hipSuccess) return (int)e;
        configured = true;
    }
    const long most = (GROUPED ? row_tiles_at_most(M, groups, 256) : ((long)M + 255) / 256) * ((N + Wide<NA>::TN - 1L) / Wide<NA>::TN);
    if (most >> 30) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((k_mxfp4_wide<OUT, NA, GROUPED>), dim3((unsigned)(most + 7) / 8 * 8), dim3(512), Wide<NA>::LDS, st, y, x, xs, W, Ws, M, N, nb, first_row, groups);
    return (int)hipGetLastError();
}

template <typename OUT>
int linear(void *stream, OUT *y, const uint8_t *x, const uint8_t *xs, const uint8_t *W, const uint8_t *Ws, const int *first_row, int groups, int rows, int in,
           int out) {
    const int nb = (int)(((long)in + 31) / 32);
    const long wgs = (first_row ? row_tiles_at_most(rows, groups, 128) : ((long)rows + 127) / 128) * ((out + 127L) / 128);
    if (wgs >> 31) return (int)hipErrorInvalidValue;
    hipStream_t st = (hipStream_t)stream;
    if (rows >= 256 && out >= 192 && nb % 8 == 0 && nb >= 16 && out % (16 / (int)sizeof(OUT)) == 0 && (((uintptr_t)y | (uintptr_t)xs | (uintptr_t)Ws) & 15) == 0)
        return first_row ? launch_wide<OUT, 4, true>(st, y, x, xs, W, Ws, rows, out, nb, first_row, groups)
                         : launch_wide<OUT, 4, false>(st, y, x, xs, W, Ws, rows, out, nb, nullptr, 1);
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
