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
 * on how long the sequences are, which the host does not know. A wave finds its range from the lengths (256 sequences at a time, four to a
 * lane). A list entry that lies in one range as a whole is finished there; of one that is cut, each part leaves its unnormalised sums
 * and their maximum in the workspace and a second launch joins them. It finds what a range's end cuts in the workspace too, written while the range's wave waits for its
 * first pages: looked up from the lengths again the second launch takes 1 to 2 us more. A range cuts its first and its last entry at most: two places each.
 *
 * In a tile S^T = K Q^T (A = K, a key a row; B = Q, a query head a column, 16 of them, zeros behind the last) and O^T += V^T P^T
 * (A = V^T from the transposing LDS read), so that a lane holds one query's scores for 4 keys of every 16, and P^T in bf16 is the
 * second product's B operand as it lies. There is room for more products than memory lets be used: P goes in two bf16 parts of 8 bits,
 * and the result is as exact as its own rounding. Keys in 8 bits are multiplied as they are, with their scales, by scaled products of
 * 128 dims: Q is cut into two parts of 4 bits, which together hold its 8 (to 2^-18 of its largest value). Values in 8 bits become bf16,
 * which holds them exactly, behind the LDS reads, and their scales multiply the probabilities.
 *
 * What bounds it: memory in long texts: 131072 + 70001 + 4097 tokens of 8 kv heads in 8 bits (424 MB) take 80 us, 5.3 TB/s, and 6 to join;
 * 64 texts of 4096 in bf16 (1.07 GB) 189 us, 5.7 TB/s (with the join). In short ones the instructions around a list entry, some 2 us
 * of a wave that is alone on its SIMD (two waves of half the tile are no faster): 256 texts of up to 2048 in 8 bits (157 MB) 44 us + 5. Calls of one text are a
 * chain of launches and dependent reads (lengths, pages, tiles): 300 tokens 5.5 us + 4.
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
#include <type_traits>

#include "iris_kernels_hip.h"
#include "join_parts.h"
#include "paged_cache.h"
#include "sequences.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

constexpr int HD = 128, COLS = 16, STAGES = 2;
constexpr int MOST_WAVES = 1024;                                     /* ranges: four waves on each of 256 CUs, as the LDS holds */
constexpr int PART = part_floats(COLS, HD);                          /* floats of a place in the workspace: sums, maxima, denominators */
/* The list entry that the end of a range cuts: its first tile and their number (0: none is cut); and the tiles of the call */
struct Cut { int g, head, cols, first, tiles, total, unused[2]; };
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

/* The list of tiles: sequence g has tiles(g) * per of them, per = kv_heads * blocks of 16 query heads. Looked at 256 sequences at a time,
 * four to a lane, so that their lengths are one trip to memory. */
struct Work {
    PagedArg cache;
    int n, per, keys;                            /* keys of a tile */
    bool empty;                                  /* there are sequences without tokens */
    int length[4], upto[4], total;               /* this lane's sequences of the last 256 looked at: tokens, and tiles with all in front */

    __device__ __forceinline__ void look(int base) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int g = base + 64 * i + (threadIdx.x & 63);
            length[i] = cache.lengths[min(g, n - 1)];
        }
        const long most = (long)cache.ld << cache.shift;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            upto[i] = total;
            if (base + 64 * i < n) {
                const bool there = base + 64 * i + (int)(threadIdx.x & 63) < n;
                length[i] = there ? (int)min((long)max(length[i], 0), most) : 0;
                empty = empty || __any(there && length[i] == 0);
                upto[i] += wave_sum_upto(tiles(length[i]) * per);
                total = __builtin_amdgcn_readlane(upto[i], 63);
            }
        }
    }
    __device__ __forceinline__ int tiles(int tokens) const { return (tokens + keys - 1) / keys; }
    __device__ __forceinline__ int count(const PagedArg &c, int sequences, int per_tile, int tile_keys) {
        cache = c; n = sequences; per = per_tile; keys = tile_keys; total = 0; empty = false;
        for (int base = 0; base < n; base += 256) look(base);
        return total;
    }
    /* the sequence of tile u < count(): its number, tokens, the tiles of a list entry, and those in front of it */
    __device__ __forceinline__ void find(int u, int *g, int *tokens, int *entry, int *before) {
        int base = 0;
        if (n > 256) {
            total = 0;
            for (; base < n; base += 256) {
                look(base);
                if (u < total) break;
            }
        }
        *g = *before = *tokens = 0; *entry = 1;
        bool found = false;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned long long past = __ballot(upto[i] > u);
            if (past && !found) {
                const int at = __ffsll(past) - 1;
                found = true;
                *g = base + 64 * i + at;
                *tokens = __builtin_amdgcn_readlane(length[i], at);
                *entry = tiles(*tokens);
                *before = __builtin_amdgcn_readlane(upto[i], at) - *entry * per;
            }
        }
    }
};

/* The tiles in `waves` ranges: `each` or, the first `more` of them, one more. In 32 bits: a 64-bit division takes half a microsecond. */
struct Ranges {
    int each, more;
    __device__ __forceinline__ Ranges(int total, int waves) : each(total / waves) { more = total - each * waves; }
    __device__ __forceinline__ int begin(int w) const { return w * each + min(w, more); }
    __device__ __forceinline__ int of(int u) const {                 /* the range that tile u is in */
        const int front = more * (each + 1);
        return u < front ? u / (each + 1) : more + (u - front) / each;
    }
};
__device__ __forceinline__ int ranges(int total, int most) { return min(most, max(1, total)); }

struct Args {
    uint16_t *out;
    const uint16_t *q;
    const unsigned char *k, *v;
    const uint8_t *ks, *vs;
    PagedArg cache;
    int ldo, ldq, n, group, blocks;              /* group: query heads of a kv head, in blocks of 16 */
    float scale_log2, *part;                     /* part: two places a range, then a Cut each */
};
__device__ __forceinline__ Cut *cut_at(const Args &a, int w) { return reinterpret_cast<Cut *>(a.part + (size_t)2 * MOST_WAVES * PART) + w; }

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_16(uint32_t lds, const unsigned char *src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
/* a byte of each lane, to 4 bytes of the LDS each */
__device__ __forceinline__ void load_byte(uint32_t lds, const unsigned char *src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
/* a dword of each lane */
__device__ __forceinline__ void load_word(uint32_t lds, const void *src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop
/* Stores that are counted with the loads behind which they are issued; the compiler might make fewer of them */
__device__ __forceinline__ void store_8(void *p, uint2 v) {
    const u32x2 w = {v.x, v.y};
    asm volatile("global_store_dwordx2 %0, %1, off" ::"v"(p), "v"(w) : "memory");
}
__device__ __forceinline__ void store_16(void *p, f32x4 v) {         /* the wait states in front of the next write of its registers */
    asm volatile("global_store_dwordx4 %0, %1, off\n\ts_nop 1" ::"v"(p), "v"(v) : "memory");
}
constexpr int STORES = 8;                                            /* of a column's result, at least */
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

/* A tile that has been asked for: the keys of it that count, and what it belongs to */
struct Tile {
    unsigned long long seen;
    int g, head, cols;                           /* sequence, first query head, query heads (at most 16) */
    bool begin, end, from_start, whole;          /* first and last of its list entry in this range; the entry began here; and ended here */
};

template <bool FP8, int QROWS>
__global__ void __launch_bounds__(64, 2)                              /* 256 registers: the products then leave their results in vector registers */
k_paged_hd128(Args a) {
    typedef Shape<FP8> S;
    extern __shared__ __align__(16) unsigned char lds[];              /* two stages, Q of two list entries, pages of two runs of 64 */
    constexpr int Q0 = STAGES * S::STAGE, Q_BYTES = QROWS * 2 * HD, P0 = Q0 + 2 * Q_BYTES;
    const int lane = threadIdx.x, li = lane & 15, lg = lane >> 4, w = blockIdx.x, per = a.cache.kv_heads * a.blocks, shift = a.cache.shift;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)lds);
    Work work;
    const int total = work.count(a.cache, a.n, per, S::KEYS), waves = ranges(total, gridDim.x);
    if (w >= total && lane == 0) cut_at(a, w)->tiles = 0;
    for (int g = work.empty ? w : a.n; g < a.n; g += gridDim.x)
        if (paged_length(a.cache, g) == 0)
            for (int c = lane; c < a.group * a.cache.kv_heads * (HD / 4); c += 64)
                *reinterpret_cast<uint2 *>(a.out + (size_t)g * a.ldo + 4 * (size_t)c) = make_uint2(0, 0);
    const Ranges range(total, waves);
    const int begin = range.begin(w), end = range.begin(w + 1);
    if (w >= waves || begin == end) return;                          /* no keys at all */

    /* The tile that is asked for next, and the pages of 64 page-fuls of tokens from the one that it begins in. */
    int u = begin - 1, g = 0, length = 0, tiles = 1, before = 0, tile = 0, kvh = 0, block = 0, q_turn = 0;
    int run_g = -1, run_page = 0, run = 0;
    bool from_start = false, asked = false;
    /* steps to the next tile, and asks for its pages where they are not those that are here */
    auto step = [&]() {
        u++; tile++;
        if (u == begin || tile == tiles) {
            tile = 0;
            if (++block == a.blocks) { block = 0; kvh++; }
            if (u == begin || kvh == a.cache.kv_heads) {
                work.find(u, &g, &length, &tiles, &before);
                const int entry = (u - before) / tiles;              /* 0 but for the range's first */
                tile = u - before - entry * tiles;
                kvh = entry / a.blocks;
                block = entry - kvh * a.blocks;
            }
        }
        const int from = tile * S::KEYS >> shift, to = (tile * S::KEYS + S::KEYS - 1) >> shift;
        if (g != run_g || from < run_page || to >= run_page + 64) {
            run_g = g; run_page = from; run ^= 1;
            asked = true;
            const int at = run_page + lane;
            load_word(lds0 + P0 + 256 * run, at < a.cache.ld ? (const void *)(a.cache.table + (size_t)run_g * a.cache.ld + at) : (const void *)zeros);
        }
    };

    /* Asks for tile u and steps to the next one, whose pages are asked for in front of this one's loads: whoever waits for this tile has them. */
    auto request = [&](Tile &t, int stage) {
        const int k0 = tile * S::KEYS, head = kvh;
        t.g = g;
        t.head = kvh * a.group + block * COLS;
        t.cols = min(COLS, a.group - block * COLS);
        t.begin = u == begin || tile == 0;
        if (t.begin) from_start = tile == 0;
        t.from_start = from_start;
        t.end = u + 1 == end || tile + 1 == tiles;
        t.whole = from_start && tile + 1 == tiles;

        const int pos = k0 + (lane & (S::KEYS - 1));
        const unsigned page = reinterpret_cast<const unsigned *>(lds + P0 + 256 * run)[(pos >> shift) - run_page];
        const bool there = pos < length && page < (unsigned)a.cache.pages;
        const unsigned row = there ? ((page * (unsigned)a.cache.kv_heads + (unsigned)head) << shift) + ((unsigned)pos & ((1u << shift) - 1)) : NO_ROW;
        const unsigned long long word = __ballot(there);
        t.seen = S::KEYS == 64 ? word : word & 0xffffffffu;
        if (u + 1 < end) step();
        if (t.begin) {
#pragma unroll
            for (int j = 0; j < QROWS / 4; j++) {
                const int r = 4 * j + (lane >> 4);
                load_16(lds0 + Q0 + Q_BYTES * q_turn + 1024 * j,
                        r < t.cols ? (const unsigned char *)(a.q + (size_t)t.g * a.ldq + (size_t)(t.head + r) * HD + 8 * (lane & 15)) : zeros);
            }
            q_turn ^= 1;
        }
        const uint32_t dst = lds0 + stage * S::STAGE;
        constexpr int LANES = S::ROW / 16, ROWS = 64 / LANES;        /* lanes to a row, rows to a load */
#pragma unroll
        for (int j = 0; j < S::HALF / 1024; j++) {
            const int r = j * ROWS + lane / LANES;
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

    /* O^T: dims 16 db + 4 lg + r of column li; the column's maximum, and this lane's part of the denominator */
    f32x4 o[8];
    float top = 0.0f, sum = 0.0f, base = 0.0f;                       /* base: the maximum, 0 where it is -infinity */
    unsigned worst = 0;                                              /* the largest scale byte of the V rows this lane has looked at */
    bf16x8 qb[4];                                                    /* Q^T in bf16, or in two parts of 8 bits and their scale */
    i32x8 q_hi, q_lo;
    int q_scale = 0, q_read = 0;

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

    Tile now, next;
    bool stored = false;
    step();
    {
        /* meanwhile, for the second launch: the entry that the range ends in */
        int g1, length1, tiles1, before1;
        work.find(end - 1, &g1, &length1, &tiles1, &before1);
        const int entry1 = (end - 1 - before1) / tiles1, first1 = before1 + entry1 * tiles1, kvh1 = entry1 / a.blocks, c1 = (entry1 - kvh1 * a.blocks) * COLS;
        if (lane == 0) *cut_at(a, w) = Cut{g1, kvh1 * a.group + c1, min(COLS, a.group - c1), first1, first1 + tiles1 > end ? tiles1 : 0, total, {}};
    }
    wait_loads<1>();                                                 /* all but that store */
    asked = false;
    /* The first two turns only ask (one place in the code for it: a short call is as long as its instructions take to come from memory). */
    for (int t = begin - 2, stage = 0; t < end; t++, stage ^= 1) {
        /* all but the next tile's, and the stores of the last result if there was one: this tile, its Q, the pages of the one after the next */
        if (t + 1 >= end) wait_loads<0>();
        else if (stored) wait_loads<S::LOADS + STORES>();
        else if (t >= begin || asked) wait_loads<S::LOADS>();
        const unsigned char *cur = lds + stage * S::STAGE;
        if (t >= begin) {
            stored = now.end;
            if (now.begin) {
                const unsigned char *qp = lds + Q0 + Q_BYTES * q_read + (li & (QROWS - 1)) * 2 * HD;
                if constexpr (FP8) {
                    /* lane (li, lg) holds dims 16 lg .. + 15 and 64 + 16 lg .. + 15 of column li */
                    u32x4 x[4];
                    unsigned most = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        x[i] = *reinterpret_cast<const u32x4 *>(qp + 128 * (i >> 1) + 32 * lg + 16 * (i & 1));
                        if (QROWS < COLS && li >= QROWS) x[i] = u32x4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < 4; j++) most = max(most, max(x[i][j] & 0x7fff, (x[i][j] >> 16) & 0x7fff));
                    }
                    most = max(most, (unsigned)__shfl_xor((int)most, 16, 64));      /* one scale for the column: a lane's 32 values are of two blocks */
                    most = max(most, (unsigned)__shfl_xor((int)most, 32, 64));
                    float factor;
                    q_scale = (int)scale_byte(most, &factor);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        int hi = 0, lo = 0;
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint32_t word = x[i >> 1][2 * (i & 1) + h];
                            const float c0 = __uint_as_float(word << 16) * factor, c1 = __uint_as_float(word & 0xffff0000u) * factor;
                            hi = h ? __builtin_amdgcn_cvt_pk_fp8_f32(c0, c1, hi, true) : __builtin_amdgcn_cvt_pk_fp8_f32(c0, c1, hi, false);
                            const f32x2 back = h ? __builtin_amdgcn_cvt_pk_f32_fp8(hi, true) : __builtin_amdgcn_cvt_pk_f32_fp8(hi, false);
                            lo = h ? __builtin_amdgcn_cvt_pk_fp8_f32(c0 - back[0], c1 - back[1], lo, true) : __builtin_amdgcn_cvt_pk_fp8_f32(c0 - back[0], c1 - back[1], lo, false);
                        }
                        q_hi[i] = hi; q_lo[i] = lo;
                    }
                } else {
                    /* lane (li, lg) holds dims 32 ks + 8 lg .. + 7 of column li */
#pragma unroll
                    for (int ks = 0; ks < 4; ks++) {
                        u32x4 x = *reinterpret_cast<const u32x4 *>(qp + 64 * ks + 16 * lg);
                        if (QROWS < COLS && li >= QROWS) x = u32x4{0, 0, 0, 0};
                        qb[ks] = __builtin_bit_cast(bf16x8, x);
                    }
                }
                q_read ^= 1;
#pragma unroll
                for (int db = 0; db < 8; db++) o[db] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                top = -INFINITY; sum = 0.0f; base = 0.0f; worst = 0;
            }
            constexpr int MB = S::KEYS / 16;
            f32x4 s[MB];                                                 /* key 16 mb + 4 lg + r against column li, in units of log2 */
#pragma unroll
            for (int mb = 0; mb < MB; mb++) {
                f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (FP8) {
                    const u32x4 k0 = *reinterpret_cast<const u32x4 *>(cur + (k_rd[0] ^ 16 * (mb & 1)) + 16 * mb * S::ROW);        /* swizzle(16 mb + li) */
                    const u32x4 k1 = *reinterpret_cast<const u32x4 *>(cur + (k_rd[1] ^ 16 * (mb & 1)) + 16 * mb * S::ROW);
                    const i32x8 ka = __builtin_bit_cast(i32x8, __builtin_shufflevector(k0, k1, 0, 1, 2, 3, 4, 5, 6, 7));
                    const int scale = *reinterpret_cast<const int *>(cur + 2 * S::HALF + 4 * (16 * mb + li));
                    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(ka, q_lo, acc, 0, 0, 0, scale, 0, q_scale);
                    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(ka, q_hi, acc, 0, 0, 0, scale, 0, q_scale);
                } else {
#pragma unroll
                    for (int ks = 0; ks < 4; ks++)
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8 *>(cur + k_rd[ks] + 16 * mb * S::ROW), qb[ks], acc, 0, 0, 0);
                }
                s[mb] = acc * a.scale_log2;
            }
            const unsigned long long all = S::KEYS == 64 ? ~0ull : 0xffffffffull, mine = now.seen;
            if (mine != all) {
#pragma unroll
                for (int mb = 0; mb < MB; mb++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (!((mine >> (16 * mb + 4 * lg + r)) & 1ull)) s[mb][r] = -INFINITY;
            }
            float high = -INFINITY;
#pragma unroll
            for (int mb = 0; mb < MB; mb++) high = fmaxf(fmaxf(fmaxf(high, s[mb][0]), fmaxf(s[mb][1], s[mb][2])), s[mb][3]);
            if (__any(high > top + RAISE)) {                          /* the first tile: -infinity + 8 */
                const float peak = fmaxf(top, over_column(high, [](float x, float y) { return fmaxf(x, y); }));
                base = peak == -INFINITY ? 0.0f : peak;
                const float alpha = __builtin_amdgcn_exp2f(top - base);
                top = peak;
                sum *= alpha;
#pragma unroll
                for (int db = 0; db < 8; db++) o[db] *= alpha;
            }
            u32x4 pw[MB / 2], rest[MB / 2];                               /* p in bf16 and what is left of it: together 16 bits */
#pragma unroll
            for (int kg = 0; kg < MB / 2; kg++) {
                float p[8];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    p[r] = __builtin_amdgcn_exp2f(s[2 * kg][r] - base);
                    p[4 + r] = __builtin_amdgcn_exp2f(s[2 * kg + 1][r] - base);
                }
                sum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                if constexpr (FP8) {
                    const u32x4 v0 = *reinterpret_cast<const u32x4 *>(cur + 2 * S::HALF + 256 + 4 * (32 * kg + 4 * lg)), v1 = *reinterpret_cast<const u32x4 *>(cur + 2 * S::HALF + 256 + 4 * (32 * kg + 16 + 4 * lg));
#pragma unroll
                    for (int r = 0; r < 4; r++) { p[r] = ldexpf(p[r], (int)v0[r] - 127); p[4 + r] = ldexpf(p[4 + r], (int)v1[r] - 127); }
                }
                /* The upper part is cut off and not rounded. An infinity in V times both has to be that infinity, so that the rest of a p in bf16 is not 0 either:
                 * its last bit is set (2^-23 of it; a p below 2^-110 of the maximum may still have none, and makes the infinity NaN). Codes of 8 bits have no
                 * infinities. */
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t b0 = __float_as_uint(p[2 * i]), b1 = __float_as_uint(p[2 * i + 1]), c0 = b0 & 0xffff0000u, c1 = b1 & 0xffff0000u, last = FP8 ? 0 : 1;
                    pw[kg][i] = (c0 >> 16) | c1;
                    rest[kg][i] = pack_bf16(__uint_as_float(b0 | last) - __uint_as_float(c0), __uint_as_float(b1 | last) - __uint_as_float(c1));
                }
            }
            /* The two products of a sum are not one behind the other, where the second would wait for the first (256 texts take 2.4 us longer so) */
            constexpr int TOGETHER = 2;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kg = 0; kg < MB / 2; kg++)
#pragma unroll
                for (int d0 = 0; d0 < 8; d0 += TOGETHER) {
                    bf16x8 va[TOGETHER];
#pragma unroll
                    for (int d = 0; d < TOGETHER; d++) {
                        const unsigned char *vp = cur + v_rd[d0 + d] + 32 * kg * S::ROW;
                        if constexpr (FP8) {
                            const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2 *)vp);
                            const bf16x2 c0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], 1.0f, false), c1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], 1.0f, true);
                            const bf16x2 c2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], 1.0f, false), c3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], 1.0f, true);
                            va[d] = bf16x8{c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
                        } else {
                            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)vp);
                            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(vp + 16 * S::ROW));
                            va[d] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                        }
                    }
#pragma unroll
                    for (int d = 0; d < TOGETHER; d++) o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[d], __builtin_bit_cast(bf16x8, rest[kg]), o[d0 + d], 0, 0, 0);
#pragma unroll
                    for (int d = 0; d < TOGETHER; d++) o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[d], __builtin_bit_cast(bf16x8, pw[kg]), o[d0 + d], 0, 0, 0);
                }
            if (FP8) worst = max(worst, *reinterpret_cast<const unsigned *>(cur + 2 * S::HALF + 256 + 4 * lane));      /* the scale of key `lane` */
            wait_lds();                                                  /* this stage has been read */
        }
        const Tile done = now;
        now = next;
        if (t + 2 < end) request(next, stage);
        if (t < begin || !done.end) continue;
        /* A V row of scale 255 is not a number, whatever its codes, and so is what it has part in. (A K row's scale is the product's, which makes the
         * score NaN.) Asked of every p, or of the scores of every tile, 256 texts take 3 us longer. */
        const float den = FP8 && __any(worst == 255) ? __builtin_nanf("") : over_column(sum, [](float x, float y) { return x + y; });
        if (li < done.cols && done.whole) {
            const float inv = den == 0.0f ? 0.0f : 1.0f / den;
            uint16_t *op = a.out + (size_t)done.g * a.ldo + (size_t)(done.head + li) * HD + 4 * lg;
#pragma unroll
            for (int db = 0; db < 8; db++)
                store_8(op + 16 * db, make_uint2(pack_bf16(o[db][0] * inv, o[db][1] * inv), pack_bf16(o[db][2] * inv, o[db][3] * inv)));
        } else if (li < done.cols) {
            float *pp = a.part + (size_t)(2 * w + done.from_start) * PART;
            /* the products have left the matrix cores: the compiler places no wait states in front of an asm statement */
            asm volatile("s_nop 15\n\ts_nop 3" : "+v"(o[0]), "+v"(o[1]), "+v"(o[2]), "+v"(o[3]), "+v"(o[4]), "+v"(o[5]), "+v"(o[6]), "+v"(o[7]));
#pragma unroll
            for (int db = 0; db < 8; db++) store_16(pp + li * HD + 16 * db + 4 * lg, o[db]);
            if (lg == 0) { pp[COLS * HD + li] = top; pp[COLS * HD + COLS + li] = den; }
        }
    }
}

/* Workgroup w stands for the end of range w. Those whose ends cut the same list entry share its columns: the entry's parts are those of
 * the ranges w0 .. last, and w takes every (last - w0)-th column from w - w0 on. */
template <int JOIN>
__global__ void __launch_bounds__(JOIN)
k_paged_join(Args a) {
    const int w = blockIdx.x;
    const Cut cut = *cut_at(a, w);
    if (!cut.tiles) return;
    const Ranges range(cut.total, ranges(cut.total, gridDim.x));
    const int w0 = range.of(cut.first), sharers = range.of(cut.first + cut.tiles - 1) - w0;
    join_parts<JOIN, COLS, HD>(
        (cut.cols - (w - w0) + sharers - 1) / sharers, sharers + 1, [&](int i) { return a.part + (size_t)(2 * (w0 + i) + (i == 0)) * PART; },      /* (perhaps no columns) */
        [&](int n) { return w - w0 + n * sharers; }, [&](int n) { return a.out + (size_t)cut.g * a.ldo + (size_t)(cut.head + w - w0 + n * sharers) * HD; });
}

}  // namespace

extern "C" size_t iris_hip_paged_workspace(void) { return MOST_WAVES * (2 * PART * sizeof(float) + sizeof(Cut)); }

/* 1 where iris_hip_paged_hd128 takes these sizes: row numbers and the number of tiles in 32 bits */
extern "C" int iris_hip_paged_hd128_takes(int pages, int page_shift, int table_ld, int n, int heads, int kv_heads) {
    const __int128 rows = ((__int128)pages * kv_heads) << page_shift;
    const __int128 tiles = ((((__int128)table_ld << page_shift) + 31) / 32 + 1) * n * kv_heads * ((heads / kv_heads + COLS - 1) / COLS);
    return rows < NO_ROW && tiles < (1LL << 31) && ((__int128)table_ld << page_shift) < (1LL << 31) - 64;
}

/* The launches for these sizes: waves of the first, and threads of a workgroup of the second (0: there is none). Host arithmetic only */
extern "C" void iris_hip_paged_plan(int fp8, int page_shift, int table_ld, int n, int heads, int kv_heads, int *waves, int *join) {
    const int group = heads / kv_heads, blocks = (group + COLS - 1) / COLS, keys = fp8 ? Shape<true>::KEYS : Shape<false>::KEYS;
    const long tiles = ((((long)table_ld << page_shift) + keys - 1) / keys) * n * kv_heads * blocks;
    const int most = group > 8 ? MOST_WAVES / 4 * 3 : MOST_WAVES;     /* with 16 rows of Q for two list entries three waves have room in a CU's LDS */
    *waves = tiles < 1 ? 1 : tiles < most ? (int)tiles : most;
    /* Entries of many parts are joined by more threads: one text of 30000, 8 heads on one kv head, 29.5 us and 21.5 with 512; 16 on 2, 23.5 and 19.6; where the
     * parts are few the threads only have to be started: 48 texts of 1 to 4096, 32 on 8, 24 and 26 */
    *join = *waves >= 160L * n * kv_heads * blocks ? 512 : *waves > 1 ? 256 : 0;
}

extern "C" int iris_hip_paged_hd128(void *stream, float *part, uint16_t *out, int ldo, const uint16_t *q, int ldq, const void *k, const void *v,
                                    const uint8_t *ks, const uint8_t *vs, int pages, int page_shift, const int *table, int table_ld,
                                    const int *lengths, int n, int heads, int kv_heads, float scale) {
    const int group = heads / kv_heads, blocks = (group + COLS - 1) / COLS;
    const Args a = {out, q, (const unsigned char *)k, (const unsigned char *)v, ks, vs, {table, lengths, table_ld, pages, page_shift, kv_heads, HD},
                    ldo, ldq, n, group, blocks, scale * 1.4426950408889634f, part};
    const int q_rows = group <= 4 ? 4 : group <= 8 ? 8 : 16;
    int waves, join;
    iris_hip_paged_plan(ks != nullptr, page_shift, table_ld, n, heads, kv_heads, &waves, &join);
    auto run = [&](auto fp8, auto rows) {
        constexpr int QROWS = decltype(rows)::value, LDS = STAGES * Shape<decltype(fp8)::value>::STAGE + 2 * QROWS * 2 * HD + 512;
        hipLaunchKernelGGL((k_paged_hd128<decltype(fp8)::value, QROWS>), dim3(waves), dim3(64), LDS, (hipStream_t)stream, a);
    };
    auto run_rows = [&](auto fp8) {
        if (q_rows == 4) run(fp8, std::integral_constant<int, 4>{});
        else if (q_rows == 8) run(fp8, std::integral_constant<int, 8>{});
        else run(fp8, std::integral_constant<int, 16>{});
    };
    if (ks) run_rows(std::true_type{});
    else run_rows(std::false_type{});
    if (join == 512) hipLaunchKernelGGL(k_paged_join<512>, dim3(waves), dim3(512), 0, (hipStream_t)stream, a);
    else if (join) hipLaunchKernelGGL(k_paged_join<256>, dim3(waves), dim3(256), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}
