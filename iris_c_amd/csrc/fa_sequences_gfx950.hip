/*
 * Attention over packed sequences (sequences.h), head_dim 128, bf16 on the matrix cores.
 *
 *     out[c] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(scale log2(e) q_c . k_j - max),   j < limit(c)
 *
 * limit(c): the keys m of the column's sequence; causal, of a column of row i of n: i + 1 + m - n. A column is one query row of one head,
 * and the columns of a tile are those of the query heads that share a kv head, row by row: K and V are fetched once for all of them, and
 * with four heads to a kv head a workgroup of 256 columns spans 64 rows, so that few of its products lie behind the causal limit, and a
 * prompt of 40 rows still fills 160 columns.
 *
 * A workgroup is WAVES waves of NB blocks of 16 columns; K and V tiles of 64 keys go from memory straight into the LDS, one group of GROUP
 * tiles ahead of the group in use, with one barrier a group. In a tile S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32_bf16: a
 * lane holds one column of each block, 16 of its 64 scores, and exp2(S^T) in bf16 is the second product's B operand as it lies. The row
 * sums are a product with ones; they are those of the rounded p. The maximum is raised by more than 2^8 only. The LDS keeps the 16-byte
 * piece c of row r in place c ^ 2 (r % 8) (the source addresses of the loads are permuted): neither kind of read meets in a bank.
 *
 * What a column does not see: rows behind the sequence's last key are read from a row of zeros; scores behind the causal limit are set to
 * -infinity, so that their p is zero; and because zero times an infinity is not a number, the tile that the limit passes through is
 * multiplied by zeros first, and if that gives anything but zeros its infinities and NaN are taken out of V, and put into the sums of the
 * columns that see them at the end (keys in parts: by the part that holds the tile).
 *
 * Workgroups: eight kv heads at a time (one to an XCD, whose L2 then holds the K and V of one head); with a causal limit from the last tile
 * of the last sequence down, so that of each sequence the longest come first (those of all sequences first is no faster), otherwise
 * sequence by sequence from the one with the most keys down.
 *
 * What bounds it: 12001 + 4096 + 700 + 1 causal rows, 32 heads on 8, take 1.18 - 1.24 ms, 1.07 - 1.12 PFLOP/s; pictures of 4608,
 * 1536, 2627 and 576 rows, 24 heads, 360 - 414 us (0.92 - 1.05 PFLOP/s). The matrix cores are busy 52 and 45 % of the cycles of all SIMDs, no LDS
 * access conflicts, 95 and 86 % of the requests are served by the L2s; as in the kernel for one sequence the rest is the softmax's vector
 * instructions (a thousand cycles beside 1088 of products per wave and tile) and what the chip's power leaves of the clock. 24 prompts of 4
 * to 512 rows take 20 us: workgroups of about 4 us of dependent reads (bounds, first tiles) and up to 8 tiles of 1.1 us and more, two on a CU.
 *
 * Where there are few columns and many keys, the keys of every workgroup's columns are cut into parts, of as many key blocks each as gives about
 * two workgroups to a CU; the lengths are in device memory, so the kernel itself finds how many (sequences.h). Each part leaves its unnormalised
 * sums, their maximum and denominator in a workspace, and a second launch joins them, as many workgroups as there are parts, which find what
 * they join in the workspace too (looked up anew it would take 3 us more): 64 + 1 + 200 + 17 rows over 8294 keys, 32 heads on 8, 67 us whole, 36 to 39 cut
 * (7 of them to join 30 MB); 32 rows over 16000 keys 227 and 31. Equal numbers of parts for all sequences, as many as the host can tell from their
 * average, leave the longest to be waited for: 46 and 53.
 */
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "iris_kernels_hip.h"
#include "join_parts.h"
#include "sequences.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

constexpr int HD = 128, KEYS = 64, TILE = KEYS * HD, STAGE = 2 * TILE;      /* elements of K or V; of a stage, 32 KB */
constexpr float RAISE = 8.0f;
constexpr int MOST_PARTS = 512;                                     /* two workgroups on each of 256 CUs */

__device__ __align__(256) const uint16_t zeros[HD] = {};

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const f32x2 p = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}
__device__ __forceinline__ float max3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }
/* over the four lanes l % 16, + 16, + 32, + 48 */
__device__ __forceinline__ float column_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float t = max3(__uint_as_float(a[0]), __uint_as_float(a[1]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(t), __float_as_uint(t), false, false);
    return max3(__uint_as_float(b[0]), __uint_as_float(b[1]), __uint_as_float(b[1]));
}
__device__ __forceinline__ int swizzle(int row) { return 2 * (row & 7); }
__device__ __forceinline__ uint32_t lds_address(const uint16_t *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p; }

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
/* K and V rows of a tile -> a stage: 32 pieces of four rows (1 KB), 32 / WAVES to a wave. Rows from `there` on are zeros. */
template <int WAVES>
__device__ __forceinline__ void load_tile(uint16_t *stage, const uint16_t *kt, const uint16_t *vt, size_t ld, int there, const uint32_t (&lane_off)[2], int wave) {
    constexpr int PIECES = 32 / WAVES;
    if (there >= KEYS) {
#pragma unroll
        for (int j = 0; j < PIECES; j++) {
            const int p = wave * PIECES + j;                          /* 0 .. 15: K, 16 .. 31: V */
            const uint64_t from = (uint64_t)(uintptr_t)((p < 16 ? kt : vt) + (size_t)(4 * (p & 15)) * ld);
            const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)from), hi = __builtin_amdgcn_readfirstlane((uint32_t)(from >> 32));
            const uint16_t *src = (const uint16_t *)(uintptr_t)(((uint64_t)hi << 32) | lo);
            const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_address(stage + (p < 16 ? 0 : TILE) + 4 * (p & 15) * HD));
            /* the wait states between a vector instruction that writes a scalar register and a memory instruction that reads it */
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(lane_off[p & 1]), "s"(src) : "memory", "m0");
        }
    } else {
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));                              /* the last tile's own addresses are not kept either */
#pragma unroll
        for (int j = 0; j < PIECES; j++) {
            const int p = wave * PIECES + j, row = 4 * (p & 15) + (lane >> 4), piece = 8 * ((lane & 15) ^ swizzle(row));
            const uint16_t *src = row < there ? (p < 16 ? kt : vt) + (size_t)row * ld + piece : zeros + piece;
            const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_address(stage + (p < 16 ? 0 : TILE) + 4 * (p & 15) * HD));
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory", "m0");
        }
    }
}
#pragma clang diagnostic pop

/* without what is an infinity or not a number */
__device__ __forceinline__ s16x8 only_numbers(s16x8 v) {
    u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t lo = (w[i] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu, hi = (w[i] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u;
        w[i] &= lo | hi;
    }
    return __builtin_bit_cast(s16x8, w);
}

struct Args {
    uint16_t *out;
    const uint16_t *q, *k, *v;
    int ldo, ldq, ldkv, kv_heads;
    SequencesArg seqs;
    float scale_log2, *part;                     /* part: partial results, where the keys are cut */
};

/* tiles between two barriers: two where only one workgroup has room on a CU anyway */
constexpr int group_of(int waves, int blocks) { return waves * blocks >= 16 ? 2 : 1; }

/* What a workgroup works on */
struct Place { bool there; int kvh, tile; };
__device__ __forceinline__ Place place(const Args &a, int count, bool last_first) {
    const int together = a.kv_heads % 8 == 0 ? 8 : a.kv_heads;       /* kv heads whose tiles are dealt out in turn */
    const unsigned round = (unsigned)together * (unsigned)count, number = blockIdx.x;
    if (round == 0 || number / round >= (unsigned)(a.kv_heads / together)) return {false, 0, 0};
    const unsigned rest = number % round;
    return {true, (int)(number / round) * together + (int)(rest % together), last_first ? count - 1 - (int)(rest / together) : (int)(rest / together)};
}
/* What the second launch finds about a workgroup of the first: part `part` of `parts` of `columns` columns from c0 on; place: of part 0 */
struct Cut { int parts, part, place, row0, c0, columns, kvh, unused; };
__device__ __forceinline__ float *part_at(const Args &a, int place) { return a.part + (size_t)place * part_floats(128, HD); }
__device__ __forceinline__ Cut *cut_at(const Args &a, int wg) { return reinterpret_cast<Cut *>(part_at(a, MOST_PARTS)) + wg; }

template <int WAVES, int NB, bool CAUSAL, bool CUT>
__global__ void __launch_bounds__(64 * WAVES, 2)
k_sequences_hd128(Args a) {
    extern __shared__ __align__(16) uint16_t lds[];                  /* 2 GROUP stages */
    constexpr int COLUMNS = 16 * NB * WAVES, GROUP = group_of(WAVES, NB);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lg = lane >> 4;
    const int group = a.seqs.per_row;

    SequenceTiles<!CAUSAL && !CUT, CUT> tiles;
    int count = tiles.count(a.seqs, COLUMNS);
    if constexpr (CUT) count = tiles.cut(a.kv_heads, MOST_PARTS);
    const Place at = place(a, count, CAUSAL);
    if (!at.there) {
        if (CUT && threadIdx.x == 0) cut_at(a, blockIdx.x)->parts = 0;
        return;
    }
    const SequenceTile s = tiles.tile(at.tile);
    const int kvh = at.kvh;
    if (CUT && threadIdx.x == 0)
        *cut_at(a, blockIdx.x) = Cut{s.parts, s.part, kvh * count + at.tile - s.part, s.row0, s.c0, min(COLUMNS, s.n * group - s.c0), kvh, 0};

    /* this lane's columns, one in each block; those behind the sequence's last are computed like it and not stored */
    const int columns = s.n * group, wc0 = s.c0 + wave * 16 * NB, ahead = s.m - s.n;
    int row[NB], head[NB], limit[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        const int c = min(wc0 + 16 * nb + li, columns - 1);
        row[nb] = c / group;
        head[nb] = kvh * group + c - row[nb] * group;
        limit[nb] = CAUSAL ? row[nb] + 1 + ahead : s.m;
    }
    const int last = min(s.c0 + COLUMNS, columns) - 1, k_end = CAUSAL ? max(last / group + 1 + ahead, 0) : s.m;      /* no column of the workgroup sees more */
    const int all_tiles = (k_end + KEYS - 1) / KEYS;
    const int each = CUT ? (all_tiles + s.parts - 1) / s.parts : all_tiles, tile0 = CUT ? min(s.part * each, all_tiles) : 0, ntiles = min(tile0 + each, all_tiles);
    const bool busy = wc0 < columns;
    /* the wave's columns see all of the tiles in front of the first limit, and nothing from the last one on */
    const int see_all = CAUSAL ? wc0 / group + 1 + ahead : s.m, see_any = CAUSAL ? min(wc0 + 16 * NB - 1, columns - 1) / group + 1 + ahead : s.m;

    const uint16_t *kbase = a.k + (size_t)s.key0 * a.ldkv + (size_t)kvh * HD, *vbase = a.v + (size_t)s.key0 * a.ldkv + (size_t)kvh * HD;
    uint32_t lane_off[2];
#pragma unroll
    for (int odd = 0; odd < 2; odd++) lane_off[odd] = 2u * (uint32_t)((lane >> 4) * a.ldkv + 8 * ((lane & 15) ^ swizzle(4 * odd + (lane >> 4))));
    auto request = [&](int tile, int stage) {
        if (tile >= ntiles) return;
        const size_t at = (size_t)tile * KEYS * a.ldkv;
        load_tile<WAVES>(lds + stage * STAGE, kbase + at, vbase + at, a.ldkv, s.m - tile * KEYS, lane_off, wave);
    };
#pragma unroll
    for (int t = 0; t < GROUP; t++) request(tile0 + t, t);

    bf16x8 qb[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        const uint16_t *qp = a.q + (size_t)(s.row0 + row[nb]) * a.ldq + (size_t)head[nb] * HD + 8 * lg;
#pragma unroll
        for (int ks = 0; ks < 4; ks++) qb[nb][ks] = *reinterpret_cast<const bf16x8 *>(qp + 32 * ks);
    }
    /* complete here: the compiler does not count the tile requests, and a wait of its own inside the loop would be for all of them */
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            u32x4 t = __builtin_bit_cast(u32x4, qb[nb][ks]);
            asm volatile("" : "+v"(t));
            qb[nb][ks] = __builtin_bit_cast(bf16x8, t);
        }

    const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
    /* where a lane reads K (key li, dims 8 lg of step 0) and V (row 4 lg + li / 4, dims 4 (li % 4) of block 0); the swizzle is an exclusive or,
     * so step ks is 32 ks, block db 16 db away by exclusive or */
    int k_rd = li * HD + 8 * (lg ^ swizzle(li)), v_rd;
    {
        const int vrow = 4 * lg + (li >> 2);
        v_rd = TILE + vrow * HD + 8 * (((li & 3) >> 1) ^ swizzle(vrow)) + 4 * (li & 1);
    }
    f32x4 o[8][NB], den[NB];                                          /* O^T: dims 16 db + 4 lg + r; the sum of p in every row */
    float top[NB], neg[NB], bound[NB];                                /* the maximum, minus it (0 while it is -infinity), (it + 8) / scale */
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
        for (int db = 0; db < 8; db++) o[db][nb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        den[nb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        top[nb] = -INFINITY; neg[nb] = 0.0f; bound[nb] = -INFINITY;
    }
    const float inv_scale = 1.0f / a.scale_log2;
    bool put_back = false;
    wait_loads<0>();
    lds_barrier();

    /* Tiles that all of the wave's columns see as a whole have a loop of their own: in one loop, where they jump over what the others need, 512 rows
     * take 15.8 us and not 13.2, 12001 + 4096 + 700 + 1 rows 1350 and not 1240 (32 heads on 8). The loops' turns have the same barriers. */
    const int whole = min(max(see_all, 0) / KEYS, ntiles);
    int t0 = tile0, half = 0;
    auto group_of_tiles = [&](auto is_cut) {
#pragma unroll
        for (int step = 0; step < GROUP; step++) {
            const int k0 = (t0 + step) * KEYS;
            const uint16_t *cur = lds + (half * GROUP + step) * STAGE;
            /* wave-uniform; every wave passes the same barriers and asks for its share of the tiles */
            const bool work = busy && t0 + step < ntiles && k0 < see_any;
            asm volatile("" : "+v"(k_rd), "+v"(v_rd));              /* their sums are made here and not kept in registers all the time */
            f32x4 sc[4][NB];
            if (work) {
                u32x4 ka[2][4];
                auto read_k = [&](int ks) {
#pragma unroll
                    for (int mb = 0; mb < 4; mb++) ka[ks & 1][mb] = *reinterpret_cast<const u32x4 *>(&cur[(k_rd ^ 32 * ks) + 16 * mb * HD]);
                };
                read_k(0);
                __builtin_amdgcn_sched_barrier(0);
                const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < 4; ks++) {
                    if (ks < 3) read_k(ks + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int mb = 0; mb < 4; mb++)
#pragma unroll
                        for (int nb = 0; nb < NB; nb++)
                            sc[mb][nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ka[ks & 1][mb]), qb[nb][ks],
                                                                                ks == 0 ? zero : sc[mb][nb], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (step == 0) {                                          /* behind the first product, so that the matrix cores have work meanwhile */
#pragma unroll
                for (int t = 0; t < GROUP; t++) request(t0 + GROUP + t, (half ^ 1) * GROUP + t);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (!work) continue;

            /* key k0 + 16 mb + 4 lg + r against column li of block nb */
            const bool cut = is_cut && k0 + KEYS > see_all;
            if (cut) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    const int behind = limit[nb] - k0 - 4 * lg;
#pragma unroll
                    for (int mb = 0; mb < 4; mb++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (16 * mb + r >= behind) sc[mb][nb][r] = -INFINITY;
                }
            }
            float high[NB];
            bool raise = false;
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                const float x = max3(max3(sc[0][nb][0], sc[0][nb][1], sc[0][nb][2]), max3(sc[0][nb][3], sc[1][nb][0], sc[1][nb][1]), max3(sc[1][nb][2], sc[1][nb][3], sc[2][nb][0]));
                const float y = max3(max3(sc[2][nb][1], sc[2][nb][2], sc[2][nb][3]), max3(sc[3][nb][0], sc[3][nb][1], sc[3][nb][2]), sc[3][nb][3]);
                high[nb] = fmaxf(x, y);
                raise = raise || high[nb] > bound[nb];
            }
            if (__any(raise)) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    const float now = fmaxf(top[nb], column_max(high[nb]) * a.scale_log2);
                    const float alpha = __builtin_amdgcn_exp2f(top[nb] - (now == -INFINITY ? 0.0f : now));
                    top[nb] = now;
                    neg[nb] = now == -INFINITY ? 0.0f : -now;
                    bound[nb] = (now + RAISE) * inv_scale;
                    den[nb] *= alpha;
#pragma unroll
                    for (int db = 0; db < 8; db++) o[db][nb] *= alpha;
                }
            }
            /* P^T: of keys 32 ks .. + 31 this lane has 32 ks + 4 lg + r and 32 ks + 16 + 4 lg + r */
            u32x4 pw[2][NB];
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    float p[8];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        p[r] = __builtin_amdgcn_exp2f(fmaf(sc[2 * ks][nb][r], a.scale_log2, neg[nb]));
                        p[4 + r] = __builtin_amdgcn_exp2f(fmaf(sc[2 * ks + 1][nb][r], a.scale_log2, neg[nb]));
                    }
                    pw[ks][nb] = u32x4{pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]), pack_bf16(p[4], p[5]), pack_bf16(p[6], p[7])};
                }
            auto value = [&](int ks, int db) -> s16x8 {
                const uint16_t *vp = &cur[(v_rd ^ 16 * db) + 32 * ks * HD];
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(vp));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(vp + 16 * HD));
                return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            };
            bool numbers = true;
            if (CAUSAL && cut) {
                const bf16x8 none = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0});
                f32x4 bad[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    bad[i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, value(i >> 3, i & 7)), none, bad[i & 1], 0, 0, 0);
                    if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
                bad[0] += bad[1];
                numbers = !__any(!(bad[0][0] + bad[0][1] + bad[0][2] + bad[0][3] == 0.0f));
                put_back = put_back || !numbers;
            }
            s16x8 va[2][4];
            auto read_v = [&](int g) {
#pragma unroll
                for (int d = 0; d < 4; d++) va[g & 1][d] = value(g >> 1, 4 * (g & 1) + d);
            };
            read_v(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g < 4; g++) {
                if (g < 3) read_v(g + 1);
                __builtin_amdgcn_sched_barrier(0);
                const int ks = g >> 1;
                if (CAUSAL && !numbers) {
#pragma unroll
                    for (int d = 0; d < 4; d++) va[g & 1][d] = only_numbers(va[g & 1][d]);
                }
                if ((g & 1) == 0)
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
                        den[nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(bf16x8, pw[ks][nb]), den[nb], 0, 0, 0);
#pragma unroll
                for (int d = 0; d < 4; d++)
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
                        o[4 * (g & 1) + d][nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va[g & 1][d]), __builtin_bit_cast(bf16x8, pw[ks][nb]),
                                                                                         o[4 * (g & 1) + d][nb], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        wait_loads<0>();                                              /* the next group has landed, this wave's pieces; behind the barrier everybody's */
        lds_barrier();
        t0 += GROUP;
        half ^= 1;
    };
    while (t0 + GROUP <= whole) group_of_tiles(std::false_type{});
    while (t0 < ntiles) group_of_tiles(std::true_type{});

    if (CAUSAL && put_back) {
        /* What was left out of the tiles that a limit passes through, for the columns that see it. Of this part's tiles alone: a column that sees
         * no key of the part has weight 0 in the join, where an infinity of another part's would be 0 times an infinity. */
        for (int key = max(max(see_all, 0) / KEYS, tile0) * KEYS; key < min(min(see_any, s.m), ntiles * KEYS); key++) {
            const uint16_t *vp = vbase + (size_t)key * a.ldkv + 4 * lg;
#pragma unroll
            for (int db = 0; db < 8; db++) {
                const uint2 w = *reinterpret_cast<const uint2 *>(vp + 16 * db);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t bits = r % 2 ? (r < 2 ? w.x : w.y) & 0xffff0000u : (r < 2 ? w.x : w.y) << 16;
                    const float v = (bits & 0x7f800000u) == 0x7f800000u ? __uint_as_float(bits) : 0.0f;
#pragma unroll
                    for (int nb = 0; nb < NB; nb++) o[db][nb][r] += key < limit[nb] ? v : 0.0f;
                }
            }
        }
    }

    if (CUT && s.parts > 1) {
        static_assert(!CUT || COLUMNS == 128, "");
        float *pp = part_at(a, kvh * count + at.tile);
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            const int c = wave * 16 * NB + 16 * nb + li;
            if (s.c0 + c >= columns) continue;
#pragma unroll
            for (int db = 0; db < 8; db++) *reinterpret_cast<f32x4 *>(pp + c * HD + 16 * db + 4 * lg) = o[db][nb];
            if (lg == 0) { pp[COLUMNS * HD + c] = top[nb]; pp[COLUMNS * (HD + 1) + c] = den[nb][0]; }
        }
        return;
    }
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        const float inv = den[nb][0] == 0.0f ? 0.0f : 1.0f / den[nb][0];
        if (wc0 + 16 * nb + li < columns) {
            uint16_t *op = a.out + (size_t)(s.row0 + row[nb]) * a.ldo + (size_t)head[nb] * HD + 4 * lg;
#pragma unroll
            for (int db = 0; db < 8; db++)
                *reinterpret_cast<uint2 *>(op + 16 * db) = make_uint2(pack_bf16(o[db][nb][0] * inv, o[db][nb][1] * inv), pack_bf16(o[db][nb][2] * inv, o[db][nb][3] * inv));
        }
    }
}

/* The parts of a workgroup's columns joined, by as many workgroups as there are parts: each takes every parts-th column */
constexpr int JOIN = 512;
__global__ void __launch_bounds__(JOIN)
k_sequences_join(Args a) {
    const Cut cut = *cut_at(a, blockIdx.x);
    if (cut.parts < 2) return;
    const int group = a.seqs.per_row;
    join_parts<JOIN, 128, HD>(
        (cut.columns - cut.part + cut.parts - 1) / cut.parts, cut.parts, [&](int i) { return part_at(a, cut.place + i); },
        [&](int n) { return cut.part + n * cut.parts; },
        [&](int n) {
            const int c = cut.c0 + cut.part + n * cut.parts, row = c / group;
            return a.out + (size_t)(cut.row0 + row) * a.ldo + (size_t)(cut.kvh * group + c - row * group) * HD;
        });
}

template <int WAVES, int NB, bool CAUSAL, bool CUT = false>
int launch(hipStream_t stream, const Args &a) {
    constexpr int LDS = 2 * group_of(WAVES, NB) * STAGE * (int)sizeof(uint16_t);
    static bool configured = false;
    if (!configured) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(k_sequences_hd128<WAVES, NB, CAUSAL, CUT>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) return (int)e;
        configured = true;
    }
    const long wgs = CUT ? MOST_PARTS : sequence_tiles_at_most(a.seqs, 16 * NB * WAVES) * a.kv_heads;
    if (!wgs) return 0;
    if (wgs > ((1L << 32) - 1) / (64 * WAVES)) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((k_sequences_hd128<WAVES, NB, CAUSAL, CUT>), dim3((unsigned)wgs), dim3(64 * WAVES), LDS, stream, a);
    if constexpr (CUT) hipLaunchKernelGGL(k_sequences_join, dim3((unsigned)wgs), dim3(JOIN), 0, stream, a);
    return (int)hipGetLastError();
}

}  // namespace

/* Which workgroups a call takes: waves x blocks of 16 columns a wave; and whether it cuts their keys where it has a workspace (4 x 2 then), into at
 * most `parts` for all of them; 1: it does not. Host arithmetic only */
extern "C" void iris_hip_sequences_plan(int n, int rows, int keys, int heads, int kv_heads, int causal, int own_keys, int *waves, int *blocks, int *parts) {
    const int group = heads / kv_heads;
    const long some = n < rows ? n : rows, blocks16 = ((long)rows * group + some * 8) / 16 * kv_heads, each = (long)rows * group / some;
    /* Measured, us, by waves x blocks, with 32 query heads on 8 unless noted. Causal: 31 rows 5.9 with 2 x 1, 6.4 with 4 x 1; 118 rows 7.4 / 7.5, 8 x 1 9.1, 4 x 2 9.6;
     * 512 rows 13.6 / 13.0, 4 x 2 17.3; 1000 rows 31.1 / 22.6, 4 x 2 28.0; 24 prompts of 4 to 512 21.8 with 4 x 1, 18.9 with 4 x 2; 61 of 40 rows 21.8 / 20.6; 4608 rows
     * 231 / 180, 8 x 2 188. Not causal, 4 x 1 / 8 x 1 / 4 x 2 / 8 x 2: 1000 rows 28.4 / 25.4 / 28.7 / -; the 24 prompts 27.8 / 22.8 / 22.5 / 26.2; 11 of 200 rows, 24 heads on 24,
     * 23.5 / 19.0 / 19.8 / 24.4; 4608 rows so 339 / 299 / 288 / 262. Sequences of few columns leave waves of large workgroups without any: 101 of 16 rows, 24 on 24, 23.3 with
     * 4 x 1, 25.3 with 8 x 1, 26.7 with 4 x 2; one wave alone is slower for every one of these (its loads wait for each other). */
    *parts = 1;
    *waves = causal || blocks16 <= 1024 ? 4 : 8;
    *blocks = (causal ? blocks16 > 3500 : blocks16 > 2048 && each >= 1024) ? 2 : 1;
    if (each <= 64) { *waves = 4; *blocks = 1; }
    if (blocks16 <= 128 && keys / some <= KEYS) { *waves = 2; *blocks = 1; }
    /* Whether the key blocks of a workgroup are cut into parts: where few workgroups walk long. tiles: workgroups of 128 columns, chain: key
     * blocks that one walks, on the average of the sequences. us, whole and cut, causal / not:
     *     tiles  16, chain  8  12.6 18.9 /  11.6 17.8         16  19.5 17.2 /  18.8 16.3         32  32.9 17.0 / 32.2 16.4
     *     tiles  64, chain 16  20.2 23.0 /  19.7 23.1         32  34.1 30.0 /  33.2 30.5         64  61.6 38.6 / 60.6 38.6
     *     tiles 128, chain 16  21.1 26.6 /  20.7 27.5         32  36.2 35.4 /  35.2 36.0         64  65.2 52.0 / 63.0 50.8
     *     tiles 232, chain 31  40.2 47.1 /  41.1 51.5         93   114  106 /   106  109
     * Where sequences with keys of their own may differ in length, which the host does not know, the longest is waited for: 32 of 16 rows, 376 tiles,
     * over 500 keys but one of 8000 (chain 11) 116 29, over 100 to 4000 (11) 59 32, of 20000 (17) 288 35; 10 of 100 rows, 328 tiles, over 200 to 16000
     * keys 139 98, 24 heads on 24 189 94. They are cut sooner, though all of one length lose by it: 32 of 16 rows over 734 keys each (11) 21 30,
     * 4 of 64 rows 17 21, 32 of 16 over 1024 27 35, over 2048 52 57.
     * Nothing is cut where there might be more tiles than leave an eighth of the parts to cut with, or more than the 256 sequences that a wave looks
     * at at once. */
    const long tiles = sequence_tiles_at_most({nullptr, nullptr, n, rows, keys, group}, 128) * kv_heads, chain = (long)keys / some / KEYS / (causal && own_keys ? 2 : 1);
    static_assert(MOST_PARTS * (part_floats(128, HD) * sizeof(float) + sizeof(Cut)) <= IRIS_LINEAR_PART_BYTES, "");
    const bool differ = some > 1 && !own_keys;
    if (n <= 256 && tiles <= MOST_PARTS / 8 * 7 && tiles * ((long)keys / KEYS + 1) < 1L << 30 && (differ ? chain >= 11 : chain * (360 - tiles) >= 4800)) *parts = MOST_PARTS;
}

/* part: IRIS_LINEAR_PART_BYTES of private workspace, 16-byte aligned, or null: the keys of a workgroup are then not cut */
extern "C" int iris_hip_sequences_hd128(void *stream, float *part, uint16_t *out, int ldo, const uint16_t *q, int ldq, const uint16_t *k, const uint16_t *v,
                                        int ldkv, const int *first_row, const int *first_key, int n, int rows, int keys, int heads, int kv_heads, float scale,
                                        int causal) {
    Args a = {out, q, k, v, ldo, ldq, ldkv, kv_heads, {first_row, first_key, n, rows, keys, heads / kv_heads}, scale * 1.4426950408889634f, part};
    const hipStream_t st = (hipStream_t)stream;
    int waves, blocks, parts;
    iris_hip_sequences_plan(n, rows, keys, heads, kv_heads, causal, first_key == nullptr, &waves, &blocks, &parts);
    if (part && parts > 1) return causal ? launch<4, 2, true, true>(st, a) : launch<4, 2, false, true>(st, a);
    if (causal) return blocks == 2 ? launch<4, 2, true>(st, a) : waves == 4 ? launch<4, 1, true>(st, a) : launch<2, 1, true>(st, a);
    if (waves == 8) return blocks == 2 ? launch<8, 2, false>(st, a) : launch<8, 1, false>(st, a);
    return waves == 4 ? launch<4, 1, false>(st, a) : launch<2, 1, false>(st, a);
}
