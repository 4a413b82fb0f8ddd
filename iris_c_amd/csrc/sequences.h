/*
 * Rows of several sequences one behind the other: rows [first[g], first[g + 1]) of `rows` are sequence g, first: device int [n + 1], and
 * its keys are [first_key[g], first_key[g + 1]) of `keys` (first_key NULL: its own rows).
 *
 * Every row has `per_row` columns (the query heads that share a key-value head, or one), numbered row by row inside a sequence. The
 * kernels walk one list of tiles of `height` columns, sequence by sequence. No tile straddles two. The host knows an upper bound of their number; a
 * workgroup finds the true number and its own tile, 256 sequences at a time, four to a lane.
 *
 * Whatever the arrays hold, every tile lies inside [0, rows) and [0, keys): a value counts as the largest up to its place, limited to
 * 0 .. rows (keys). Rows outside [first[0], first[n]) are in no tile. first NULL: row g is sequence g.
 */
#ifndef IRIS_SEQUENCES_H
#define IRIS_SEQUENCES_H

struct SequencesArg { const int *first_row, *first_key; int n, rows, keys, per_row; };       /* the kernels' argument */

/* the tile's columns are c0 .. c0 + height - 1 of the sequence's n * per_row; column c is row row0 + c / per_row. Cut: part `part` of `parts` */
struct SequenceTile { int row0, n, c0, key0, m, g, part, parts; };        /* g: the sequence's number, in order */

/* inclusive sum and maximum over the lanes up to each one, in the vector registers (shifts inside rows of 16, then the rows' last
 * lanes to those behind them): a tenth of the time of six trips through the LDS */
template <int CTRL, int ROWS> __device__ __forceinline__ int seq_dpp(int other, int v) {
    return __builtin_amdgcn_update_dpp(other, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_sum_upto(int v) {
    v += seq_dpp<0x111, 0xf>(0, v);
    v += seq_dpp<0x112, 0xf>(0, v);
    v += seq_dpp<0x114, 0xf>(0, v);
    v += seq_dpp<0x118, 0xf>(0, v);
    v += seq_dpp<0x142, 0xa>(0, v);
    v += seq_dpp<0x143, 0xc>(0, v);
    return v;
}
__device__ __forceinline__ int wave_max_upto(int v) {                    /* of values >= 0 */
    v = max(v, seq_dpp<0x111, 0xf>(0, v));
    v = max(v, seq_dpp<0x112, 0xf>(0, v));
    v = max(v, seq_dpp<0x114, 0xf>(0, v));
    v = max(v, seq_dpp<0x118, 0xf>(0, v));
    v = max(v, seq_dpp<0x142, 0xa>(0, v));
    v = max(v, seq_dpp<0x143, 0xc>(0, v));
    return v;
}

/* Blocks of keys to a part, at least 4, within a 32nd the fewest that make no more than most_entries entries of `tiles` tiles (fewer than that)
 * with `work` blocks in all. entries(each) is their number with `each` blocks to a part: one a tile, and one more for every further part. There is such a
 * number: entries(each) <= work / each + tiles. Host code can call it. */
template <class Entries> __host__ __device__ __forceinline__ int part_blocks(int work, int tiles, int most_entries, Entries entries) {
    constexpr int LEAST = 4;
    const int more = most_entries - tiles;
    int few = (work / most_entries > LEAST ? work / most_entries : LEAST) - 1, many = (work + more - 1) / more;      /* too few, or not to be tried; enough */
    if (many < LEAST) many = LEAST;
    while (many - few > 1 + many / 32) {                                  /* at least 2: `each` lies between them, and takes the place of one */
        const int each = (few + many) / 2;
        if (entries(each) <= most_entries) many = each;
        else few = each;
    }
    return many;
}

/* BY_LENGTH: up to 64 sequences in the order of their keys, the most first, for kernels whose tiles take as long as the keys are many: the
 * last workgroups of a call are then short ones. CUT, up to 256 sequences: every tile is in the list as several parts of at most `each` key
 * blocks of 64, so many that there are about as many entries as wanted, and each about as long as the others. */
template <bool BY_LENGTH = false, bool CUT = false>
struct SequenceTiles {
    static constexpr int AT_ONCE = 4;                                /* 64 sequences at once: their bounds are one trip to memory */
    SequencesArg a;
    int height;
    int lo[AT_ONCE], hi[AT_ONCE], klo[AT_ONCE], khi[AT_ONCE];        /* this lane's sequences of the last looked at: rows, keys */
    int upto[AT_ONCE], total, most, key_most;    /* tiles of all sequences up to each; of all so far; the largest values in front of those */
    int each;                                    /* of the cut */

    /* first[g] and the next one, each as the largest value up to its place, limited to 0 .. limit */
    static __device__ __forceinline__ void range(int from, int to, int limit, int &most, int &lo, int &hi) {
        const int x = max(wave_max_upto(max(from, 0)), most), y = max(x, to);
        most = __builtin_amdgcn_readlane(y, 63);
        lo = min(x, limit);
        hi = min(y, limit);
    }
    __device__ __forceinline__ int tiles(int i) const { return ((hi[i] - lo[i]) * a.per_row + height - 1) / height; }
    /* the first 64: each to the lane that is the number of those with more keys, or as many and in front */
    __device__ __forceinline__ void by_length() {
        const int lane = threadIdx.x & 63, m = khi[0] - klo[0];
        int to = lane < a.n ? 0 : lane;
        for (int j = 0; j < a.n; j++) {
            const int other = __builtin_amdgcn_readlane(m, j);
            if (lane < a.n) to += other > m || (other == m && j < lane);
        }
        lo[0] = __builtin_amdgcn_ds_permute(4 * to, lo[0]);
        hi[0] = __builtin_amdgcn_ds_permute(4 * to, hi[0]);
        klo[0] = __builtin_amdgcn_ds_permute(4 * to, klo[0]);
        khi[0] = __builtin_amdgcn_ds_permute(4 * to, khi[0]);
    }
    __device__ __forceinline__ void look(int base) {
        const int lane = threadIdx.x & 63;
        int from[AT_ONCE], to[AT_ONCE], kfrom[AT_ONCE], kto[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) {
            const int g = min(base + 64 * i + lane, a.n), next = min(g + 1, a.n);        /* behind the last one: no rows */
            from[i] = g; to[i] = next; kfrom[i] = kto[i] = 0;
            if (base + 64 * i < a.n) {
                if (a.first_row) { from[i] = a.first_row[g]; to[i] = a.first_row[next]; }
                if (a.first_key) { kfrom[i] = a.first_key[g]; kto[i] = a.first_key[next]; }
            }
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) {
            lo[i] = hi[i] = klo[i] = khi[i] = 0;
            upto[i] = total;
            if (base + 64 * i < a.n) {
                range(from[i], to[i], a.rows, most, lo[i], hi[i]);
                klo[i] = lo[i]; khi[i] = hi[i];
                if (a.first_key) range(kfrom[i], kto[i], a.keys, key_most, klo[i], khi[i]);
                if (BY_LENGTH && i == 0 && a.n > 1 && a.n <= 64) by_length();
                upto[i] += wave_sum_upto(tiles(i));
                total = __builtin_amdgcn_readlane(upto[i], 63);
            }
        }
    }
    /* all tiles */
    __device__ __forceinline__ int count(const SequencesArg &arg, int columns) {
        a = arg; height = columns;
        most = key_most = total = 0;
        for (int base = 0; base < a.n; base += 64 * AT_ONCE) look(base);
        return total;
    }
    /* Cuts the tiles of count(), for each of `heads` heads, into not more than most_entries entries for all heads; there are fewer tiles than that
     * for them. */
    __device__ __forceinline__ int cut(int heads, int most_entries) {
        int work = 0;
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++)
            if (64 * i < a.n) work += __builtin_amdgcn_readlane(wave_sum_upto(tiles(i) * blocks(khi[i] - klo[i])), 63);
        each = part_blocks(work * heads, total * heads, most_entries, [&](int blocks_each) {
            each = blocks_each;
            int entries = 0;
#pragma unroll
            for (int i = 0; i < AT_ONCE; i++)
                if (64 * i < a.n) entries += __builtin_amdgcn_readlane(wave_sum_upto(tiles(i) * parts(khi[i] - klo[i])), 63);
            return entries * heads;
        });
        total = 0;
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) {
            upto[i] = total;
            if (64 * i < a.n) {
                upto[i] += wave_sum_upto(tiles(i) * parts(khi[i] - klo[i]));
                total = __builtin_amdgcn_readlane(upto[i], 63);
            }
        }
        return total;
    }
    static __device__ __forceinline__ int blocks(int keys) { return (keys + 63) / 64; }
    __device__ __forceinline__ int parts(int keys) const { return max(1, (blocks(keys) + each - 1) / each); }
    /* tile t of them, t < count(), or entry t < cut() */
    __device__ __forceinline__ SequenceTile tile(int t) {
        int base = 0;
        if (a.n > 64 * AT_ONCE) {
            most = key_most = total = 0;
            for (; base < a.n; base += 64 * AT_ONCE) {
                look(base);
                if (t < total) break;
            }
        }
        SequenceTile s = {0, 0, 0, 0, 0, 0, 0, 1};
        bool found = false;
#pragma unroll
        for (int i = 0; i < AT_ONCE; i++) {
            const unsigned long long past = __ballot(upto[i] > t);
            if (past && !found) {
                found = true;
                const int at = __ffsll(past) - 1;
                s.g = base + 64 * i + at;
                s.row0 = __builtin_amdgcn_readlane(lo[i], at);
                s.n = __builtin_amdgcn_readlane(hi[i], at) - s.row0;
                s.key0 = __builtin_amdgcn_readlane(klo[i], at);
                s.m = __builtin_amdgcn_readlane(khi[i], at) - s.key0;
                const int mine = (s.n * a.per_row + height - 1) / height;
                if constexpr (CUT) {
                    s.parts = parts(s.m);
                    const int entry = t - (__builtin_amdgcn_readlane(upto[i], at) - mine * s.parts), tile = entry / s.parts;
                    s.part = entry - tile * s.parts;
                    s.c0 = tile * height;
                } else {
                    s.c0 = (t - (__builtin_amdgcn_readlane(upto[i], at) - mine)) * height;
                }
            }
        }
        return s;
    }
};

/* the most tiles that there can be */
static inline long sequence_tiles_at_most(const SequencesArg &a, int height) {
    const long some = a.n < a.rows ? a.n : a.rows;
    return ((long)a.rows * a.per_row + some * (height - 1)) / height;
}

#endif
