/*
 * Rows of several sequences one behind the other: rows [first[g], first[g + 1]) of `rows` are sequence g, first: device int [n + 1], and
 * its keys are [first_key[g], first_key[g + 1]) of `keys` (first_key NULL: its own rows).
 *
 * Every row has `per_row` columns (the query heads that share a key-value head, or one), numbered row by row inside a sequence. The
 * kernels walk one list of tiles of `height` columns: those of sequence 0, of sequence 1, ... No tile straddles sequences. The host
 * knows an upper bound of their number; a workgroup finds the true number and its own tile, 64 sequences at a time, one to a lane.
 *
 * Whatever the arrays hold, every tile lies inside [0, rows) and [0, keys): a value counts as the largest up to its place, limited to
 * 0 .. rows (keys). Rows outside [first[0], first[n]) are in no tile. first NULL: row g is sequence g.
 */
#ifndef IRIS_SEQUENCES_H
#define IRIS_SEQUENCES_H

struct SequencesArg { const int *first_row, *first_key; int n, rows, keys, per_row; };       /* the kernels' argument */

/* the tile's columns are c0 .. c0 + height - 1 of the sequence's n * per_row; column c is row row0 + c / per_row */
struct SequenceTile { int row0, n, c0, key0, m, g; };

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

struct SequenceTiles {
    SequencesArg a;
    int height;
    int lo, hi, upto, tiles, most;               /* this lane's sequence of the last 64 looked at: its rows, its tiles with all before it */
    int key_most;                                /* the largest value of first_key before those 64 */

    /* first[base + lane] and the next one, each as the largest value up to its place, limited to 0 .. limit */
    static __device__ __forceinline__ void range(const int *first, int n, int g, int limit, int &most, int &lo, int &hi) {
        lo = max(wave_max_upto(g < n ? max(first[g], 0) : 0), most);
        hi = max(lo, g < n ? first[g + 1] : 0);
        most = __builtin_amdgcn_readlane(hi, 63);
        lo = min(lo, limit);
        hi = min(hi, limit);
    }
    __device__ __forceinline__ void look(int base) {
        const int g = base + (threadIdx.x & 63);
        if (a.first_row) {
            range(a.first_row, a.n, g, a.rows, most, lo, hi);
        } else {
            lo = min(g, min(a.rows, a.n));
            hi = min(g + 1, min(a.rows, a.n));
        }
        upto = tiles + wave_sum_upto(((hi - lo) * a.per_row + height - 1) / height);
        tiles = __builtin_amdgcn_readlane(upto, 63);
    }
    __device__ __forceinline__ int count(const SequencesArg &arg, int columns) {
        a = arg; height = columns; tiles = 0; most = 0;
        for (int base = 0; base < a.n; base += 64) look(base);
        return tiles;
    }
    /* tile t of them, t < count() */
    __device__ __forceinline__ SequenceTile tile(int t) {
        int base = 0;
        if (a.n > 64) {
            tiles = 0; most = 0;
            for (; base < a.n; base += 64) {
                look(base);
                if (t < tiles) break;
            }
        }
        const unsigned long long past = __ballot(upto > t);
        const int at = past ? __ffsll(past) - 1 : 0;
        SequenceTile s;
        s.g = base + at;
        s.row0 = __builtin_amdgcn_readlane(lo, at);
        s.n = __builtin_amdgcn_readlane(hi, at) - s.row0;
        s.c0 = (t - (__builtin_amdgcn_readlane(upto, at) - (s.n * a.per_row + height - 1) / height)) * height;
        s.key0 = s.row0; s.m = s.n;
        if (a.first_key) {
            int klo = 0, khi = 0;
            key_most = 0;
            for (int b = 0; b <= base; b += 64) range(a.first_key, a.n, b + (threadIdx.x & 63), a.keys, key_most, klo, khi);
            s.key0 = __builtin_amdgcn_readlane(klo, at);
            s.m = __builtin_amdgcn_readlane(khi, at) - s.key0;
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
