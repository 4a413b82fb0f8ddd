/* Every address that k_grouped_rows reads words from (half_words.h), for matrices of a few rows at all alignments: host code, nothing is read.
 * Prints the calls whose reads leave their matrix, and the number of reads. */
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdio>

#include "half_words.h"

static long reads = 0, outside = 0;

static void look(const char *what, uintptr_t from, uintptr_t to, uintptr_t lo, uintptr_t hi, int K, int U, int at) {
    reads++;
    if (from >= lo && to <= hi) return;
    outside++;
    printf("outside: %s, start %% 4 = %d, K %d, step of %d, step %d: %ld bytes in front, %ld behind\n", what, (int)(lo & 3), K, 32 * U, at,
           std::max(0L, (long)(lo - from)), std::max(0L, (long)(to - hi)));
}

int main() {
    for (int U = 2; U <= 4; U += 2)
        for (int K = 1; K <= 700; K++)
            for (int xo = 0; xo <= 2; xo += 2)
                for (int wo = 0; wo <= 2; wo += 2) {
                    const uint16_t *x = (const uint16_t *)(uintptr_t)(1u << 20 | xo), *W = (const uint16_t *)(uintptr_t)(1u << 24 | wo);
                    if (!(K & 1) && !xo && !wo) continue;      /* rows that all start at 4 bytes: nothing is shifted */
                    const HalfSteps inside = half_steps(x, W, K, 32 * U);
                    for (const uint16_t *matrix : {x, W})
                        for (int rows = 1; rows <= 3; rows++)
                            for (int r = 0; r < rows; r++)
                                for (int at = inside.first; at < inside.upto; at++)
                                    for (int lg = 0; lg < 4; lg++) {
                                        const uint16_t *row = matrix + (size_t)r * K;
                                        const uintptr_t lo = (uintptr_t)matrix, hi = (uintptr_t)(matrix + (size_t)rows * K);
                                        for (int u = 0; u < U; u++) {
                                            const uintptr_t p = (uintptr_t)run_start(row + at * 32 * U + 8 * (U * lg + u), half(row));
                                            look("a run", p, p + 16, lo, hi, K, U, at);
                                        }
                                        const uintptr_t p = (uintptr_t)run_last(row + at * 32 * U + 8 * U * (lg + 1), half(row));
                                        look("the end of a run", p, p + 4, lo, hi, K, U, at);
                                    }
                }
    printf("%ld reads, %ld outside\n", reads, outside);
    return outside != 0;
}
