/*
 * The key-value cache in pages, as kernels see it. Pages of K and of V are [pages][kv_heads][page_size] rows of head_dim values: bf16, or
 * e4m3 codes with a scale byte s a row, 2^(s - 127) (255: not a number), in arrays of their own [pages][kv_heads][page_size].
 * Position p of sequence g is place p % page_size of page table[g * ld + p / page_size]; a page number outside 0 .. pages - 1 stands for
 * a page that is not there. page_size is a power of two.
 */
#ifndef IRIS_PAGED_CACHE_H
#define IRIS_PAGED_CACHE_H

#include <stdint.h>

struct PagedArg {
    const int *table, *lengths;
    int ld, pages, shift, kv_heads, head_dim;
};

/* tokens of sequence g: not negative, and no more than its pages hold */
__device__ __forceinline__ int paged_length(const PagedArg &c, int g) {
    const long most = (long)c.ld << c.shift;
    const int n = max(c.lengths[g], 0);
    return n < most ? n : (int)most;
}

/* the row of (position, head) in the pages, or -1 where there is no such page */
__device__ __forceinline__ long paged_row(const PagedArg &c, int g, int pos, int kvh) {
    const int page = c.table[(size_t)g * c.ld + (pos >> c.shift)];
    if ((unsigned)page >= (unsigned)c.pages) return -1;
    return (((long)page * c.kv_heads + kvh) << c.shift) + (pos & ((1 << c.shift) - 1));
}

/* the scale byte of a row whose largest magnitude has these bf16 bits (sign off), the smallest power of two that it is at most 448 times of,
 * and what the row's values are multiplied by */
__device__ __forceinline__ unsigned scale_byte(unsigned top, float *factor) {
    const int exponent = (int)(top >> 7), e = max(exponent - 135 + ((top & 0x7f) > 0x60), -127);
    *factor = e == -127 ? __uint_as_float(0x7f000000u) : __uint_as_float((unsigned)(127 - e) << 23);
    return exponent == 255 ? 255 : (unsigned)(e + 127);
}

__device__ __forceinline__ float paged_scale(unsigned s) {
    return __uint_as_float(s == 255 ? 0x7fc00000u : s ? s << 23 : 0x00400000u);
}

#endif
