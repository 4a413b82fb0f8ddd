/* The search for the blocks of keys to a part (part_blocks of sequences.h) on random tiles: host code. For each call: every number that is tried lies strictly
 * between those in front of it, few are tried, the result makes no more entries than there are places, and one a 32nd less makes more
 * (or is below the least). Prints the calls and those that fail. */
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <random>
#include <vector>

#include "sequences.h"

int main() {
    std::mt19937_64 rng(5);
    auto upto = [&](double lo, double hi) { return (long)std::exp(std::uniform_real_distribution<double>(std::log(lo), std::log(hi))(rng)); };
    long calls = 0, failed = 0, searched = 0;
    for (int turn = 0; turn < 200000; turn++) {
        const int heads = (int)upto(1, 30), n = (int)upto(1, 257), most = 512, equal = (int)(rng() % 3);
        std::vector<long> tiles(n), blocks(n);
        long total = 0, work = 0;
        const long length = upto(1, 300000);
        for (int g = 0; g < n; g++) {
            tiles[g] = rng() % 5 ? 1 : (long)upto(1, 40);
            if ((total + tiles[g]) * heads > most / 8 * 7) tiles[g] = 0;      /* calls with more are not cut */
            blocks[g] = equal == 0 ? length : equal == 1 ? (rng() % 9 ? 0 : length) : upto(1, (double)length + 1) - 1;
            total += tiles[g];
            work += tiles[g] * blocks[g];
        }
        if (!total || work * heads >= 1L << 30) continue;
        calls++;
        int lowest = 0, highest = 1 << 30, tried = 0;
        bool ok = true;
        auto entries = [&](int each) {
            long e = 0;
            for (int g = 0; g < n; g++) e += tiles[g] * std::max(1L, (blocks[g] + each - 1) / each);
            return (int)std::min(e * heads, 1L << 30);
        };
        const int each = part_blocks((int)(work * heads), (int)(total * heads), most, [&](int x) {
            ok = ok && x > lowest && x < highest && ++tried < 32;
            const int e = entries(x);
            (e <= most ? highest : lowest) = x;
            return e;
        });
        searched += tried > 0;
        const int below = each - 1 - each / 32;
        ok = ok && each >= 4 && entries(each) <= most && (below < 4 || entries(below) > most);
        if (!ok) {
            failed++;
            printf("failed: %d sequences, %d heads, %ld tiles, %ld blocks: %d to a part, %d entries, %d tried\n", n, heads, total, work, each, entries(each), tried);
        }
    }
    printf("%ld calls, %ld searched, %ld failed\n", calls, searched, failed);
    return failed != 0;
}
