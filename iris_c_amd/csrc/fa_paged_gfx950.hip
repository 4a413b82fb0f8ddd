/*
 * Attention of one query row a sequence over the paged cache (paged_cache.h), head_dim 128, on the matrix cores.
 *
 *     out = sum_j p_j v_j / sum_j p_j,   p_j = 2^(scale log2(e) q . k_j - max)
 *
 * Every K and V row is read once and used for the few query heads that share it, so memory bounds it. What it needs is bytes in flight:
 * a wave on its own (a workgroup of one, four to a CU) walks a range of keys in tiles of 16 KB, K and V, that go from memory straight
 * into its part of the LDS, two tiles ahead and without a register or a barrier in between; 128 KB are in flight on a CU.
 *
 * The work of a call is one list of tiles: sequence by sequence, in it kv head by kv head (and, with more than 16 query heads to a kv
 * head, block of 16 by block). It is cut into as many equal ranges as there are waves, wherever that falls: the balance does not depend
 * on how long the sequences are, which the host does not know. A wave finds its range from the lengths (64 sequences at a time, one to a
 * lane). A list entry that lies in one range as a whole is finished there; of one that is cut, each part leaves its unnormalised sums
 * and their maximum in the workspace and a second launch joins them. A range cuts its first and its last entry at most: two places each.
 *
 * In a tile S^T = K Q^T (A = K, a key a row; B = Q, a query head a column, 16 of them, zeros behind the last) and O^T += V^T P^T
 * (A = V^T from the transposing LDS read), so that a lane holds one query's scores for 4 keys of every 16, and P^T in bf16 is the
 * second product's B operand as it lies. Codes of 8 bits become bf16, which holds them exactly, behind the LDS reads; the scales of
 * the keys multiply the scores, those of the values the probabilities.
 *
 * LDS: the 16-byte piece c of row r is kept in place c ^ swizzle(r) of its row (the loads' source addresses are permuted), so that
 * neither the K reads (16 rows at a time) nor the transposing reads (8 rows) meet in a bank: rows of 256 bytes 2 (r % 8), rows of 128
 * bytes (r & 6) + (r / 16 % 2).
 *
 * Rows behind a sequence's last token, and pages that are not there, are read from a row of zeros in their place: whatever lies in the
 * cache there has no part in the result.
 */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iris_kernels_hip.h"
#include "paged_cache.h"
#include "sequences.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

constexpr int HD = 128, COLS = 16, STAGES = 2;
constexpr int MOST_WAVES = 1024;                                     /* ranges: four waves on each of 256 CUs */
constexpr int PART = COLS * HD + 2 * COLS;                           /* floats of a place in the workspace: sums, maxima, denominators */
constexpr float RAISE = 8.0f;                                        /* the maximum is raised by more than 2^8 only: p stays below that */
constexpr unsigned NO_ROW = 0xffffffffu;

template <bool FP8> struct Shape {
    static constexpr int KEYS = FP8 ? 64 : 32, ROW = FP8 ? HD : 2 * HD;                       /* keys of a tile, bytes of a row */
    static constexpr int HALF = KEYS * ROW, SCALES = FP8 ? 2 * 4 * KEYS : 0, STAGE = 2 * HALF + SCALES;
    static constexpr int LOADS = 2 * HALF / 1024 + (FP8 ? 2 : 0);                             /* of a tile, a wave each */
};

__device__ __align__(256) const unsigned char zeros[256] = {};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const f32x2 p = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}
template <bool FP8> __device__ __forceinline__ int swizzle(int row) { return FP8 ? (row & 6) | ((row >> 4) & 1) : 2 * (row & 7); }

/* over the four lanes l % 16, + 16, + 32, + 48 */
template <class F> __device__ __forceinline__ float over_column(float v, F f) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float t = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(t), __float_as_uint(t), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

/* The list of tiles: sequence g has tiles(g) * per of them, per = kv_heads * blocks of 16 query heads */
struct Work {
    PagedArg cache;
    int n, per, keys;                            /* keys of a tile */
    int lane_tiles, upto, total;                 /* this lane's sequence of the last 64 looked at */

    __device__ __forceinline__ void look(int base) {
        const int g = base + (threadIdx.x & 63);
        lane_tiles = g < n ? (int)(((long)paged_length(cache, g) + keys - 1) / keys) : 0;
        upto = total + wave_sum_upto(lane_tiles * per);
        total = __builtin_amdgcn_readlane(upto, 63);
    }
    __device__ __forceinline__ int count(const PagedArg &c, int sequences, int per_tile, int tile_keys) {
        cache = c; n = sequences; per = per_tile; keys = tile_keys; total = 0;
        for (int base = 0; base < n; base += 64) look(base);
        return total;
    }
    /* the sequence of tile u < count(): its number, tiles, and the tiles in front of it */
    __device__ __forceinline__ void find(int u, int *g, int *tiles, int *before) {
        int base = 0;
        if (n > 64) {
            total = 0;
            for (; base < n; base += 64) {
                look(base);
                if (u < total) break;
            }
        }
        const unsigned long long past = __ballot(upto > u);
        const int at = past ? __ffsll(past) - 1 : 0;
        *g = base + at;
        *tiles = __builtin_amdgcn_readlane(lane_tiles, at);
        *before = __builtin_amdgcn_readlane(upto, at) - *tiles * per;
    }
};

/* the tiles of wave w of `waves`, and the wave that has tile u */
__device__ __forceinline__ int range_begin(int total, int w, int waves) { return (int)((long)total * w / waves); }
__device__ __forceinline__ int range_of(int total, int u, int waves) { return (int)((((long)u + 1) * waves - 1) / total); }
/* every range has two tiles at least, where there are as many */
__device__ __forceinline__ int ranges(int total, int most) { return min(most, max(1, total / 2)); }

struct Args {
    uint16_t *out;
    const uint16_t *q;
    const unsigned char *k, *v;
    const uint8_t *ks, *vs;
    PagedArg cache;
    int ldo, ldq, n, group, blocks;              /* group: query heads of a kv head, in blocks of 16 */
    float scale_log2, *part;
};

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_16(uint32_t lds, const unsigned char *src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
/* a byte of each lane, to 4 bytes of the LDS each */
__device__ __forceinline__ void load_byte(uint32_t lds, const unsigned char *src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

/* The sums of 16 columns over keys: O^T as dims 16 db + 4 lg + r of column li, its maximum, and this lane's part of the denominator */
struct State { f32x4 o[8]; float top, sum; };

/* The keys [tile0, tile1) * KEYS of a sequence's kv head */
template <bool FP8>
__device__ __forceinline__ void walk(State &st, const Args &a, unsigned char *lds, int g, int kvh, int block, int tile0, int tile1) {
    typedef Shape<FP8> S;
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    const int length = paged_length(a.cache, g), shift = a.cache.shift;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)lds);

    /* Q^T: lane (li, lg) holds 8 dims of column li for each of four steps of 32: dims 32 ks + 8 lg, and with rows of 8 bits, whose 16-byte
     * reads carry two steps, 64 (ks / 2) + 16 lg + 8 (ks % 2) */
    bf16x8 qb[4];
    {
        const int col = block * COLS + li;
        const uint16_t *qp = a.q + (size_t)g * a.ldq + (size_t)(kvh * a.group + min(col, a.group - 1)) * HD;
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            u32x4 w = *reinterpret_cast<const u32x4 *>(qp + (FP8 ? 64 * (ks >> 1) + 16 * lg + 8 * (ks & 1) : 32 * ks + 8 * lg));
            if (col >= a.group) w = u32x4{0, 0, 0, 0};
            qb[ks] = __builtin_bit_cast(bf16x8, w);
        }
    }

    /* the pages of the next 64 page-fuls of tokens, one to a lane, from the one that the tile asked for begins in */
    int page_base = (tile0 * S::KEYS) >> shift, page_id;
    auto look_up = [&]() {
        const int at = page_base + lane;
        page_id = at < a.cache.ld ? a.cache.table[(size_t)g * a.cache.ld + at] : -1;
    };
    look_up();

    unsigned long long seen[STAGES];                                 /* the keys of the tile in each stage that count */
    auto request = [&](int tile, int stage) {
        const int k0 = tile * S::KEYS;
        if (((k0 + S::KEYS - 1) >> shift) - page_base >= 64) {
            page_base = k0 >> shift;
            look_up();
        }
        const int pos = k0 + (lane & (S::KEYS - 1));
        const int page = __shfl(page_id, (pos >> shift) - page_base, 64);
        const bool there = pos < length && (unsigned)page < (unsigned)a.cache.pages;
        const unsigned row = there ? (((unsigned)page * (unsigned)a.cache.kv_heads + (unsigned)kvh) << shift) + ((unsigned)pos & ((1u << shift) - 1)) : NO_ROW;
        const unsigned long long word = __ballot(there);
        seen[stage] = S::KEYS == 64 ? word : word & 0xffffffffu;
        const uint32_t dst = lds0 + stage * S::STAGE;
        constexpr int LANES = S::ROW / 16;                           /* to a row */
#pragma unroll
        for (int j = 0; j < S::HALF / 1024; j++) {
            const int r = j * (64 / LANES) + lane / LANES;
            const unsigned from = (unsigned)__shfl((int)row, r, 64);
            const unsigned piece = 16u * ((lane & (LANES - 1)) ^ swizzle<FP8>(r));
            const size_t at = (size_t)from * S::ROW + piece;
            load_16(dst + 1024 * j, from == NO_ROW ? zeros + piece : a.k + at);
            load_16(dst + S::HALF + 1024 * j, from == NO_ROW ? zeros + piece : a.v + at);
        }
        if (FP8) {
            load_byte(dst + 2 * S::HALF, row == NO_ROW ? zeros : a.ks + row);
            load_byte(dst + 2 * S::HALF + 256, row == NO_ROW ? zeros : a.vs + row);
        }
    };

#pragma unroll
    for (int db = 0; db < 8; db++) st.o[db] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    st.top = -INFINITY; st.sum = 0.0f;
    float base = 0.0f;                                               /* the maximum, 0 where it is -infinity */

    /* where a lane reads, from the start of K or V in a stage */
    int k_rd[4], v_rd[8];
#pragma unroll
    for (int i = 0; i < (FP8 ? 2 : 4); i++) k_rd[i] = li * S::ROW + 16 * ((4 * i + lg) ^ swizzle<FP8>(li));
    {
        const int half = li >> (FP8 ? 1 : 2), row = FP8 ? 4 * lg + (half & 3) + 16 * (half >> 2) : 4 * lg + half;
#pragma unroll
        for (int db = 0; db < 8; db++)
            v_rd[db] = S::HALF + row * S::ROW + (FP8 ? 16 * (db ^ swizzle<FP8>(row)) + 8 * (li & 1)
                                                     : 16 * ((2 * db + ((li & 3) >> 1)) ^ swizzle<FP8>(row)) + 8 * (li & 1));
    }

    request(tile0, 0);
    if (tile0 + 1 < tile1) request(tile0 + 1, 1);
    for (int t = tile0; t < tile1; t++) {
        const int stage = (t - tile0) & 1;
        const unsigned char *cur = lds + stage * S::STAGE;
        if (t + 1 < tile1) wait_loads<S::LOADS>();
        else wait_loads<0>();
        constexpr int MB = S::KEYS / 16;
        f32x4 s[MB];
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (FP8) {
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    const u32x4 w = *reinterpret_cast<const u32x4 *>(cur + (k_rd[p] ^ 16 * (mb & 1)) + 16 * mb * S::ROW);     /* swizzle(16 mb + li) */
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const bf16x2 c0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[2 * e], 1.0f, false), c1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[2 * e], 1.0f, true);
                        const bf16x2 c2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[2 * e + 1], 1.0f, false), c3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[2 * e + 1], 1.0f, true);
                        const bf16x8 ka = {c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, qb[2 * p + e], acc, 0, 0, 0);
                    }
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < 4; ks++)
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8 *>(cur + k_rd[ks] + 16 * mb * S::ROW), qb[ks], acc, 0, 0, 0);
            }
            s[mb] = acc;
        }
        /* key 16 mb + 4 lg + r against column li, in units of log2 */
        float high = -INFINITY, vscale[MB][4];
#pragma unroll
        for (int mb = 0; mb < MB; mb++) {
            float f[4] = {a.scale_log2, a.scale_log2, a.scale_log2, a.scale_log2};
            if constexpr (FP8) {
                const u32x4 kb = *reinterpret_cast<const u32x4 *>(cur + 2 * S::HALF + 4 * (16 * mb + 4 * lg));
                const u32x4 vb = *reinterpret_cast<const u32x4 *>(cur + 2 * S::HALF + 256 + 4 * (16 * mb + 4 * lg));
#pragma unroll
                for (int r = 0; r < 4; r++) { f[r] *= paged_scale(kb[r]); vscale[mb][r] = paged_scale(vb[r]); }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) s[mb][r] *= f[r];
        }
        const unsigned long long all = S::KEYS == 64 ? ~0ull : 0xffffffffull, mine = seen[stage];
        if (mine != all) {
#pragma unroll
            for (int mb = 0; mb < MB; mb++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (!((mine >> (16 * mb + 4 * lg + r)) & 1ull)) s[mb][r] = -INFINITY;
        }
#pragma unroll
        for (int mb = 0; mb < MB; mb++) high = fmaxf(fmaxf(fmaxf(high, s[mb][0]), fmaxf(s[mb][1], s[mb][2])), s[mb][3]);
        if (__any(high > st.top + RAISE)) {                          /* the first tile: -infinity + 8 */
            const float now = fmaxf(st.top, over_column(high, [](float x, float y) { return fmaxf(x, y); }));
            base = now == -INFINITY ? 0.0f : now;
            const float alpha = __builtin_amdgcn_exp2f(st.top - base);
            st.top = now;
            st.sum *= alpha;
#pragma unroll
            for (int db = 0; db < 8; db++) st.o[db] *= alpha;
        }
        u32x4 pw[MB / 2];
#pragma unroll
        for (int kg = 0; kg < MB / 2; kg++) {
            float p[8];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                p[r] = __builtin_amdgcn_exp2f(s[2 * kg][r] - base);
                p[4 + r] = __builtin_amdgcn_exp2f(s[2 * kg + 1][r] - base);
            }
            st.sum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            if constexpr (FP8) {
#pragma unroll
                for (int r = 0; r < 4; r++) { p[r] *= vscale[2 * kg][r]; p[4 + r] *= vscale[2 * kg + 1][r]; }
            }
            pw[kg] = u32x4{pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]), pack_bf16(p[4], p[5]), pack_bf16(p[6], p[7])};
        }
#pragma unroll
        for (int kg = 0; kg < MB / 2; kg++)
#pragma unroll
            for (int db = 0; db < 8; db++) {
                bf16x8 va;
                const unsigned char *vp = cur + v_rd[db] + 32 * kg * S::ROW;
                if constexpr (FP8) {
                    const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2 *)vp);
                    const bf16x2 c0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], 1.0f, false), c1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], 1.0f, true);
                    const bf16x2 c2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], 1.0f, false), c3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], 1.0f, true);
                    va = bf16x8{c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
                } else {
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)vp);
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(vp + 16 * S::ROW));
                    va = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                }
                st.o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(bf16x8, pw[kg]), st.o[db], 0, 0, 0);
            }
        wait_lds();                                                  /* this stage has been read */
        if (t + 2 < tile1) request(t + 2, stage);
    }
    st.sum = over_column(st.sum, [](float x, float y) { return x + y; });
}

template <bool FP8>
__global__ void __launch_bounds__(64, 1)
k_paged_hd128(Args a) {
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x, li = lane & 15, lg = lane >> 4, w = blockIdx.x, per = a.cache.kv_heads * a.blocks;
    Work work;
    const int total = work.count(a.cache, a.n, per, Shape<FP8>::KEYS), waves = ranges(total, gridDim.x);
    for (int g = w; g < a.n; g += gridDim.x)                         /* sequences without keys */
        if (paged_length(a.cache, g) == 0)
            for (int c = lane; c < a.group * a.cache.kv_heads * (HD / 4); c += 64)
                *reinterpret_cast<uint2 *>(a.out + (size_t)g * a.ldo + 4 * (size_t)c) = make_uint2(0, 0);
    if (w >= waves) return;
    int u = range_begin(total, w, waves);
    const int end = range_begin(total, w + 1, waves);
    while (u < end) {
        int g, tiles, before;
        work.find(u, &g, &tiles, &before);
        do {                                                         /* the list entries of this sequence */
            const int entry = (u - before) / tiles, tile0 = u - before - entry * tiles, tile1 = min(tiles, tile0 + end - u);
            const int kvh = entry / a.blocks, block = entry - kvh * a.blocks, cols = min(COLS, a.group - block * COLS);
            State st;
            walk<FP8>(st, a, lds, g, kvh, block, tile0, tile1);
            if (li < cols) {
                if (tile1 - tile0 == tiles) {
                    const float inv = st.sum > 0.0f ? 1.0f / st.sum : 0.0f;
                    uint16_t *op = a.out + (size_t)g * a.ldo + (size_t)(kvh * a.group + block * COLS + li) * HD + 4 * lg;
#pragma unroll
                    for (int db = 0; db < 8; db++)
                        *reinterpret_cast<uint2 *>(op + 16 * db) = make_uint2(pack_bf16(st.o[db][0] * inv, st.o[db][1] * inv), pack_bf16(st.o[db][2] * inv, st.o[db][3] * inv));
                } else {
                    float *pp = a.part + (size_t)(2 * w + (tile0 == 0)) * PART;
#pragma unroll
                    for (int db = 0; db < 8; db++) *reinterpret_cast<f32x4 *>(pp + li * HD + 16 * db + 4 * lg) = st.o[db];
                    if (lg == 0) { pp[COLS * HD + li] = st.top; pp[COLS * HD + COLS + li] = st.sum; }
                }
            }
            u += tile1 - tile0;
        } while (u < end && u - before < tiles * per);
    }
}

/* Workgroup w joins the list entry that the end of range w cuts, if it is the first end in it. 32 lanes take 4 dims each of a column and
 * every so many-th part, eight at a time so that their loads are under way together; the LDS joins what several groups of 32 have. */
constexpr int JOIN = 512;
__global__ void __launch_bounds__(JOIN)
k_paged_join(Args a, int keys) {
    __shared__ f32x4 sums[JOIN];
    __shared__ float tops[JOIN / 32], dens[JOIN / 32];
    const int w = blockIdx.x, per = a.cache.kv_heads * a.blocks;
    Work work;
    const int total = work.count(a.cache, a.n, per, keys), waves = ranges(total, gridDim.x);
    if (w + 1 >= waves) return;
    const int u = range_begin(total, w + 1, waves);
    int g, tiles, before;
    work.find(u, &g, &tiles, &before);
    const int entry = (u - before) / tiles, first = before + entry * tiles;
    if (first == u || first < range_begin(total, w, waves)) return;
    const int last = range_of(total, first + tiles - 1, waves);
    const int kvh = entry / a.blocks, block = entry - kvh * a.blocks, cols = min(COLS, a.group - block * COLS);
    const int places = cols <= 1 ? 1 : cols <= 2 ? 2 : cols <= 4 ? 4 : cols <= 8 ? 8 : 16, groups = JOIN / 32 / places;     /* per column */
    const int unit = threadIdx.x >> 5, c = unit & (places - 1), part = unit / places, at = threadIdx.x & 31;
    float top = -INFINITY, den = 0.0f;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < cols) {
        for (int i0 = w + part; i0 <= last; i0 += 8 * groups) {
            float t[8], d[8];
            f32x4 o[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int i = min(i0 + j * groups, last);
                const float *pp = a.part + (size_t)(2 * i + (i == w)) * PART;
                t[j] = i0 + j * groups <= last ? pp[COLS * HD + c] : -INFINITY;
                d[j] = pp[COLS * HD + COLS + c];
                o[j] = *reinterpret_cast<const f32x4 *>(pp + c * HD + 4 * at);
            }
            float now = top;
#pragma unroll
            for (int j = 0; j < 8; j++) now = fmaxf(now, t[j]);
            const float base = now == -INFINITY ? 0.0f : now, alpha = __builtin_amdgcn_exp2f(top - base);
            sum *= alpha;
            den *= alpha;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (i0 + j * groups > last) break;
                const float f = __builtin_amdgcn_exp2f(t[j] - base);
                sum += o[j] * f;
                den += d[j] * f;
            }
            top = now;
        }
    }
    sums[threadIdx.x] = sum;
    if (at == 0) { tops[unit] = top; dens[unit] = den; }
    __syncthreads();
    if (part == 0 && c < cols) {
        float now = top;
        for (int j = 1; j < groups; j++) now = fmaxf(now, tops[c + j * places]);
        const float base = now == -INFINITY ? 0.0f : now, alpha = __builtin_amdgcn_exp2f(top - base);
        sum *= alpha;
        den *= alpha;
        for (int j = 1; j < groups; j++) {
            const float f = __builtin_amdgcn_exp2f(tops[c + j * places] - base);
            sum += sums[threadIdx.x + 32 * places * j] * f;
            den += dens[c + j * places] * f;
        }
        const float inv = den > 0.0f ? 1.0f / den : 0.0f;
        *reinterpret_cast<uint2 *>(a.out + (size_t)g * a.ldo + (size_t)(kvh * a.group + block * COLS + c) * HD + 4 * at) =
            make_uint2(pack_bf16(sum[0] * inv, sum[1] * inv), pack_bf16(sum[2] * inv, sum[3] * inv));
    }
}

}  // namespace

extern "C" size_t iris_hip_paged_workspace(void) { return (size_t)2 * MOST_WAVES * PART * sizeof(float); }

/* 1 where iris_hip_paged_hd128 takes these sizes: row numbers and the number of tiles in 32 bits */
extern "C" int iris_hip_paged_hd128_takes(int pages, int page_shift, int table_ld, int n, int heads, int kv_heads) {
    const __int128 rows = ((__int128)pages * kv_heads) << page_shift;
    const __int128 tiles = ((((__int128)table_ld << page_shift) + 31) / 32 + 1) * n * kv_heads * ((heads / kv_heads + COLS - 1) / COLS);
    return rows < NO_ROW && tiles < (1LL << 31) && ((__int128)table_ld << page_shift) < (1LL << 31) - 64;
}

extern "C" int iris_hip_paged_hd128(void *stream, float *part, uint16_t *out, int ldo, const uint16_t *q, int ldq, const void *k, const void *v,
                                    const uint8_t *ks, const uint8_t *vs, int pages, int page_shift, const int *table, int table_ld,
                                    const int *lengths, int n, int heads, int kv_heads, float scale) {
    const int group = heads / kv_heads, blocks = (group + COLS - 1) / COLS, keys = ks ? Shape<true>::KEYS : Shape<false>::KEYS;
    const Args a = {out, q, (const unsigned char *)k, (const unsigned char *)v, ks, vs, {table, lengths, table_ld, pages, page_shift, kv_heads, HD},
                    ldo, ldq, n, group, blocks, scale * 1.4426950408889634f, part};
    const long tiles = ((((long)table_ld << page_shift) + keys - 1) / keys) * n * kv_heads * blocks;
    const int waves = tiles / 2 < 1 ? 1 : tiles / 2 < MOST_WAVES ? (int)(tiles / 2) : MOST_WAVES;
    if (ks) hipLaunchKernelGGL(k_paged_hd128<true>, dim3(waves), dim3(64), STAGES * Shape<true>::STAGE, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(k_paged_hd128<false>, dim3(waves), dim3(64), STAGES * Shape<false>::STAGE, (hipStream_t)stream, a);
    if (waves > 1) hipLaunchKernelGGL(k_paged_join, dim3(waves), dim3(JOIN), 0, (hipStream_t)stream, a, keys);
    return (int)hipGetLastError();
}
