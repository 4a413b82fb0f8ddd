/*
 * Attention over packed sequences and over the paged cache for every head_dim, stride and alignment: the kernel behind the matrix-core
 * ones (fa_sequences_gfx950.hip, fa_paged_gfx950.hip), which take head_dim 128 on aligned rows.
 *
 *     out[c] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q_c . k_j - max),   j over the keys of the column's sequence, causal:
 *     j <= row + (keys - rows)
 *
 * A column is one query row of one head; those of the heads that share a key-value head lie side by side. One wave takes QB columns of a
 * sequence and walks its keys 64 at a time with a running maximum and sum, all in f32: first a key to a lane (its row dotted with every
 * column's query), then an output dim to a lane. A key that a column does not see is passed over and not multiplied by zero, whatever
 * its row holds. head_dim beyond 512 walks the keys once for each 512 output dims. Bound by the uncoalesced reads of K: 512 causal rows
 * of 64 dims, 32 heads on 8, take 317 us, and one token of each of 48 texts of 1024 721 us; the matrix-core kernels on 128 dims 15 and 39.
 */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iris_kernels_hip.h"
#include "paged_cache.h"
#include "sequences.h"

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

namespace {

constexpr int QB = 8, KT = 64, DIMS = 512, SLOTS = DIMS / 64;

__device__ __forceinline__ float value(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float value(uint8_t v) { return __builtin_amdgcn_cvt_f32_fp8(v, 0); }
__device__ __forceinline__ uint16_t to_bf16(float f) {
    const f32x2 p = {f, 0.0f};
    return (uint16_t)__builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}
__device__ __forceinline__ float wave_max(float v) {
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

/* where the rows of keys are: offset(j) of key j of the sequence in K and in V, or -1; scale bytes where there are any */
struct RowKeys {
    typedef uint16_t T;
    const uint16_t *k, *v;
    size_t ld;
    int key0, col;
    __device__ long offset(int j) const { return (long)((size_t)(key0 + j) * ld) + col; }
    __device__ float scale(const uint8_t *, long) const { return 1.0f; }
    const uint8_t *ks, *vs;
};
template <typename V> struct PageKeys {
    typedef V T;
    const V *k, *v;
    const uint8_t *ks, *vs;
    PagedArg c;
    int g, kvh;
    __device__ long offset(int j) const {
        const long row = paged_row(c, g, j, kvh);
        return row < 0 ? -1 : row * c.head_dim;
    }
    __device__ float scale(const uint8_t *s, long offset) const { return s ? paged_scale(s[offset / c.head_dim]) : 1.0f; }
};

/* nq columns whose queries are q + qat[c]; limit(c): the keys that column c sees are [0, limit(c)); outputs to out + oat[c] */
template <class Keys, class Q, class Out, class Limit>
__device__ __forceinline__ void walk(const Keys &keys, int nq, int m, int hd, float scale, const uint16_t *q, Q qat, uint16_t *out, Out oat, Limit limit) {
    __shared__ float ps[QB][KT];
    const int lane = threadIdx.x;
    for (int oc = 0; oc < hd; oc += DIMS) {
        float acc[QB][SLOTS], top[QB], sum[QB];
#pragma unroll
        for (int c = 0; c < QB; c++) {
            top[c] = -INFINITY; sum[c] = 0.0f;
#pragma unroll
            for (int t = 0; t < SLOTS; t++) acc[c][t] = 0.0f;
        }
        int end = 0;
        for (int c = 0; c < nq; c++) end = max(end, min(m, limit(c)));
        for (int k0 = 0; k0 < end; k0 += KT) {
            const int j = k0 + lane, nk = min(KT, end - k0);
            const long at = j < end ? keys.offset(j) : -1;
            float dot[QB];
#pragma unroll
            for (int c = 0; c < QB; c++) dot[c] = 0.0f;
            if (at >= 0) {
                for (int d = 0; d < hd; d++) {
                    const float kd = value(keys.k[at + d]);
#pragma unroll
                    for (int c = 0; c < QB; c++) dot[c] = fmaf(value(q[qat(min(c, nq - 1)) + d]), kd, dot[c]);
                }
            }
            const float ks = (at >= 0 ? keys.scale(keys.ks, at) : 1.0f) * scale, vs = at >= 0 ? keys.scale(keys.vs, at) : 1.0f;
            float alpha[QB];
            __syncthreads();
#pragma unroll
            for (int c = 0; c < QB; c++) {
                const bool sees = at >= 0 && c < nq && j < limit(min(c, nq - 1));
                const float s = sees ? dot[c] * ks : -INFINITY;
                const float high = fmaxf(top[c], wave_max(s)), base = high == -INFINITY ? 0.0f : high;
                alpha[c] = expf(top[c] - base);
                const float p = sees ? expf(s - base) : 0.0f;
                sum[c] = sum[c] * alpha[c] + wave_sum(p);
                top[c] = high;
                ps[c][lane] = sees ? p * vs : -1.0f;            /* -1: not seen (p * vs is never negative) */
            }
            __syncthreads();
            /* a whole tile's rows one after the other: lane t of the wave knows where row t is */
            for (int t = 0; t < SLOTS; t++) {
                const int d = oc + lane + 64 * t;
                if (oc + 64 * t >= hd) break;
#pragma unroll
                for (int c = 0; c < QB; c++) acc[c][t] *= alpha[c];
                for (int i = 0; i < nk; i++) {
                    const long row = __shfl(at, i, 64);
                    if (row < 0) continue;
                    const float vd = d < hd ? value(keys.v[row + d]) : 0.0f;
#pragma unroll
                    for (int c = 0; c < QB; c++) {
                        const float p = ps[c][i];
                        acc[c][t] = p < 0.0f ? acc[c][t] : fmaf(p, vd, acc[c][t]);
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < QB; c++) {
            if (c >= nq) break;
            const float inv = sum[c] == 0.0f ? 0.0f : 1.0f / sum[c];      /* no key: a row of zeros */
#pragma unroll
            for (int t = 0; t < SLOTS; t++) {
                const int d = oc + lane + 64 * t;
                if (d < hd) out[oat(c) + d] = to_bf16(acc[c][t] * inv);
            }
        }
    }
}

__global__ void __launch_bounds__(64)
k_sequences_any(uint16_t *out, int ldo, const uint16_t *q, int ldq, const uint16_t *k, const uint16_t *v, int ldkv, SequencesArg seqs,
                int kv_heads, int hd, float scale, int causal) {
    SequenceTiles<> tiles;
    const int count = tiles.count(seqs, QB), t = blockIdx.x / kv_heads, kvh = blockIdx.x % kv_heads, group = seqs.per_row;
    if (t >= count) return;
    const SequenceTile s = tiles.tile(t);
    const int nq = min(QB, s.n * group - s.c0);
    const RowKeys keys = {k, v, (size_t)ldkv, s.key0, kvh * hd, nullptr, nullptr};
    auto place = [&](int c, int ld) { return (size_t)(s.row0 + (s.c0 + c) / group) * ld + (size_t)(kvh * group + (s.c0 + c) % group) * hd; };
    walk(keys, nq, s.m, hd, scale, q, [&](int c) { return place(c, ldq); }, out, [&](int c) { return place(c, ldo); },
         [&](int c) { return causal ? (s.c0 + c) / group + 1 + s.m - s.n : s.m; });
}

template <typename T>
__global__ void __launch_bounds__(64)
k_paged_any(uint16_t *out, int ldo, const uint16_t *q, int ldq, const T *k, const T *v, const uint8_t *ks, const uint8_t *vs, PagedArg cache,
            int group, float scale) {
    const int blocks = (group + QB - 1) / QB, c0 = blockIdx.x % blocks * QB, kvh = blockIdx.x / blocks % cache.kv_heads;
    const int g = blockIdx.x / blocks / cache.kv_heads, nq = min(QB, group - c0), hd = cache.head_dim, m = paged_length(cache, g);
    const PageKeys<T> keys = {k, v, ks, vs, cache, g, kvh};
    auto place = [&](int c, int ld) { return (size_t)g * ld + (size_t)(kvh * group + c0 + c) * hd; };
    walk(keys, nq, m, hd, scale, q, [&](int c) { return place(c, ldq); }, out, [&](int c) { return place(c, ldo); }, [&](int) { return m; });
}

bool fits(long wgs) { return wgs <= ((1L << 32) - 1) / 64; }

}  // namespace

extern "C" int iris_hip_sequences_any(void *stream, uint16_t *out, int ldo, const uint16_t *q, int ldq, const uint16_t *k, const uint16_t *v,
                                      int ldkv, const int *first_row, const int *first_key, int n, int rows, int keys, int heads,
                                      int kv_heads, int head_dim, float scale, int causal) {
    const SequencesArg a = {first_row, first_key, n, rows, keys, heads / kv_heads};
    const long wgs = sequence_tiles_at_most(a, QB) * kv_heads;
    if (!wgs) return 0;
    if (!fits(wgs)) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(k_sequences_any, dim3((unsigned)wgs), dim3(64), 0, (hipStream_t)stream, out, ldo, q, ldq, k, v, ldkv, a, kv_heads,
                       head_dim, scale, causal);
    return (int)hipGetLastError();
}

extern "C" int iris_hip_paged_any(void *stream, uint16_t *out, int ldo, const uint16_t *q, int ldq, const void *k, const void *v,
                                  const uint8_t *ks, const uint8_t *vs, int pages, int page_shift, const int *table, int table_ld,
                                  const int *lengths, int n, int heads, int kv_heads, int head_dim, float scale) {
    const PagedArg c = {table, lengths, table_ld, pages, page_shift, kv_heads, head_dim};
    const int group = heads / kv_heads;
    const long wgs = (long)n * kv_heads * ((group + QB - 1) / QB);
    if (!fits(wgs)) return (int)hipErrorInvalidValue;
    if (ks)
        hipLaunchKernelGGL(k_paged_any<uint8_t>, dim3((unsigned)wgs), dim3(64), 0, (hipStream_t)stream, out, ldo, q, ldq, (const uint8_t *)k,
                           (const uint8_t *)v, ks, vs, c, group, scale);
    else
        hipLaunchKernelGGL(k_paged_any<uint16_t>, dim3((unsigned)wgs), dim3(64), 0, (hipStream_t)stream, out, ldo, q, ldq, (const uint16_t *)k,
                           (const uint16_t *)v, nullptr, nullptr, c, group, scale);
    return (int)hipGetLastError();
}
