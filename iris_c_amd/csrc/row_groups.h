/*
 * Rows of a matrix in groups: rows [first[g], first[g + 1]) of `rows` are group g, first: device int [groups + 1].
 *
 * The kernels that multiply every group by weights of its own walk one list of row tiles: the tiles of group 0, those of group 1, ...
 * A tile never straddles groups. The host knows an upper bound of their number (row_tiles_at_most); a workgroup finds the true
 * number and its own tile from `first` (a few hundred bytes, in the L2 behind the first workgroup), 64 groups at a time: each
 * lane counts the tiles of one group, a prefix sum over the wave places them. All waves of a workgroup do the same and agree.
 *
 * Whatever `first` holds, every tile lies inside [0, rows) and no row is in two: a value counts as the largest up to its place,
 * limited to 0 .. rows. Rows outside [first[0], first[groups]) are in no tile.
 */
#ifndef IRIS_ROW_GROUPS_H
#define IRIS_ROW_GROUPS_H

struct RowGroupsArg { const int *first_row; int groups; };    /* the kernels' argument */

struct RowTile { int m0, end, group; };          /* rows [m0, min(m0 + height, end)) */

template <int HEIGHT>
struct RowGroups {
    const int *first;
    int groups, rows;
    int lo, hi, upto, tiles;                     /* this lane's group of the last 64 looked at: its rows, and its tiles with all before it */
    int most;                                    /* the largest value of `first` before those 64 */

    __device__ __forceinline__ void look(int base, int before) {
        const int lane = threadIdx.x & 63, g = base + lane;
        lo = g < groups ? first[g] : 0;
        hi = g < groups ? first[g + 1] : 0;
        const int span = min(groups - base, 64);               /* the same for all lanes */
        lo = max(lo, most);
        for (int d = 1; d < span; d <<= 1) {
            const int v = __shfl_up(lo, d, 64);
            if (lane >= d) lo = max(lo, v);
        }
        hi = max(lo, hi);
        lo = min(max(lo, 0), rows);
        hi = min(max(hi, 0), rows);
        upto = g < groups ? (hi - lo + HEIGHT - 1) / HEIGHT : 0;
        for (int d = 1; d < span; d <<= 1) {
            const int v = __shfl_up(upto, d, 64);
            if (lane >= d) upto += v;
        }
        upto += before;
        tiles = __builtin_amdgcn_readlane(upto, span - 1);
        most = max(most, __builtin_amdgcn_readlane(hi, span - 1));
    }

    /* all row tiles */
    __device__ __forceinline__ int count(const int *first_row, int n, int all_rows) {
        first = first_row; groups = n; rows = all_rows; tiles = 0; most = 0;
        for (int base = 0; base < groups; base += 64) look(base, tiles);
        return tiles;
    }
    /* tile t of them, t < count() */
    __device__ __forceinline__ RowTile tile(int t) {
        int base = 0;
        if (groups > 64) {
            tiles = 0; most = 0;
            for (; base < groups; base += 64) {
                look(base, tiles);
                if (t < tiles) break;
            }
        }
        const unsigned long long past = __ballot(upto > t);
        const int at = past ? __ffsll(past) - 1 : 0;
        const int l = __builtin_amdgcn_readlane(lo, at), h = __builtin_amdgcn_readlane(hi, at), u = __builtin_amdgcn_readlane(upto, at);
        const int last = (h - l + HEIGHT - 1) / HEIGHT;        /* tiles of the group */
        return {l + (t - (u - last)) * HEIGHT, h, base + at};
    }
};

/* the rows that are in a group, [*from, *to): what the whole wave finds */
__device__ __forceinline__ void row_groups_span(const int *first, int groups, int rows, int *from, int *to) {
    int most = first[0];
    const int lo = min(max(most, 0), rows);
    for (int i = threadIdx.x & 63; i <= groups; i += 64) most = max(most, first[i]);
    for (int d = 32; d > 0; d >>= 1) most = max(most, __shfl_xor(most, d, 64));
    *from = lo;
    *to = min(max(most, 0), rows);
}

/* the most tiles that `rows` rows in `groups` groups can have */
static inline long row_tiles_at_most(int rows, int groups, int height) {
    const long some = groups < rows ? groups : rows;
    return (rows + some * (height - 1)) / height;
}

/* about how many they have: where groups are long, those of rows without groups and half a tile more for each further group (none, if
 * groups end with their tiles); where they are short, one a group */
static inline long row_tiles_about(int rows, int groups, int height) {
    const long some = groups < rows ? groups : rows, filled = (rows + height - 1L) / height + (some - 1) / 2;
    return filled > some ? filled : some;
}

/* a launch has fewer than 2^32 threads: whether `wgs` workgroups, rounded up to as many for every XCD, can be one */
static inline bool launch_fits(long wgs, int threads) { return (wgs + 7) / 8 * 8 <= ((1L << 32) - 1) / threads; }

#endif
