/*
 * Rows of 2-byte values read in whole 4 bytes, wherever they start.
 *
 * A run of values that starts in the middle of 4 bytes is read from those 4 bytes on, up to the 4 bytes in which it ends. The other
 * halves of these two words belong to the values around the run: to the row in front or behind, or, where a matrix itself starts
 * or ends in the middle of 4 bytes, to whatever lies beside it in memory, which is not read. Host code can call everything here.
 */
#ifndef IRIS_HALF_WORDS_H
#define IRIS_HALF_WORDS_H

#include <stdint.h>

/* 1 where p is in the middle of 4 bytes */
__host__ __device__ __forceinline__ int half(const uint16_t *p) { return (int)((uintptr_t)p >> 1 & 1); }
/* where the first 4 bytes of a run from p start, and where those that hold the value in front of `end` do, of a run that starts at `half` */
__host__ __device__ __forceinline__ const uint16_t *run_start(const uint16_t *p, int half) { return p - half; }
__host__ __device__ __forceinline__ const uint16_t *run_last(const uint16_t *end, int half) { return end - 2 + half; }

/* The whole steps of `step` columns, [first, upto), whose words lie inside the matrices x and W (any number of rows of K columns).
 * Of a matrix that starts at 4 bytes all do: a row of it that does not has a row in front of it and an odd K, so no whole step ends with it. One that starts in the
 * middle of 4 bytes has nothing in front of its first step, and, where K is a multiple of `step`, nothing behind its last one. */
struct HalfSteps { int first, upto; };
__host__ __device__ __forceinline__ HalfSteps half_steps(const uint16_t *x, const uint16_t *W, int K, int step) {
    const int inside = half(x) | half(W);
    return {inside, (K - inside) / step};
}

#endif
