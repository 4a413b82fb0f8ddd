/*
 * Attention whose keys were cut into parts, joined. A part's place in a workspace holds, for each of COLUMNS columns of HD dims, its
 * unnormalised sums [COLUMNS][HD], the maximum of its scores in units of log2 [COLUMNS], and its denominator [COLUMNS]:
 *
 *     out = sum_i 2^(top_i - top) sums_i / sum_i 2^(top_i - top) den_i,   top = max_i top_i
 *
 * A workgroup of THREADS threads joins `cols` columns of `parts` parts. 32 lanes take 4 dims each of a column and every so many-th part, eight at a
 * time so that their loads are under way together; the LDS joins what several groups of 32 have. Parts are added in an order that their number
 * alone determines. Columns without keys give zeros.
 */
#ifndef IRIS_JOIN_PARTS_H
#define IRIS_JOIN_PARTS_H

#include <stdint.h>

constexpr int part_floats(int columns, int hd) { return columns * (hd + 2); }

/* place(i): part i; column(n): the number of the n-th column in a place; out(n): where it goes, 8-byte aligned */
template <int THREADS, int COLUMNS, int HD, class Place, class Column, class Out>
__device__ __forceinline__ void join_parts(int cols, int parts, Place place, Column column, Out out) {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    static_assert(HD == 128, "32 lanes of 4 dims");
    __shared__ f32x4 sums[THREADS];
    __shared__ float tops[THREADS / 32], dens[THREADS / 32];
    constexpr int UNITS = THREADS / 32;
    int places = 1;                                                  /* columns at a time */
    while (places < cols && places < UNITS) places *= 2;
    const int groups = UNITS / places, unit = threadIdx.x >> 5, group = unit / places, at = threadIdx.x & 31;
    for (int n = unit & (places - 1), turn = 0; turn < cols; turn += places, n += places) {
        const int c = column(n);
        float top = -INFINITY, den = 0.0f;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        if (n < cols) {
            for (int i0 = group; i0 < parts; i0 += 8 * groups) {
                float t[8], d[8];
                f32x4 o[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int i = i0 + j * groups;
                    const float *pp = place(min(i, parts - 1));
                    t[j] = i < parts ? pp[COLUMNS * HD + c] : -INFINITY;
                    d[j] = pp[COLUMNS * (HD + 1) + c];
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
                    if (i0 + j * groups >= parts) break;
                    const float f = __builtin_amdgcn_exp2f(t[j] - base);
                    sum += o[j] * f;
                    den += d[j] * f;
                }
                top = now;
            }
        }
        if (groups > 1) {
            __syncthreads();                                         /* the columns before these have been read */
            sums[threadIdx.x] = sum;
            if (at == 0) { tops[unit] = top; dens[unit] = den; }
            __syncthreads();
        }
        if (group == 0 && n < cols) {
            float now = top;
            for (int j = 1; j < groups; j++) now = fmaxf(now, tops[unit + j * places]);
            const float base = now == -INFINITY ? 0.0f : now, alpha = __builtin_amdgcn_exp2f(top - base);
            sum *= alpha;
            den *= alpha;
            for (int j = 1; j < groups; j++) {
                const float f = __builtin_amdgcn_exp2f(tops[unit + j * places] - base);
                sum += sums[threadIdx.x + 32 * places * j] * f;
                den += dens[unit + j * places] * f;
            }
            const float inv = den == 0.0f ? 0.0f : 1.0f / den;
            const f32x2 lo = {sum[0] * inv, sum[1] * inv}, hi = {sum[2] * inv, sum[3] * inv};
            *reinterpret_cast<uint2 *>(out(n) + 4 * at) = make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf16x2)),
                                                                     __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf16x2)));
        }
    }
}

#endif
