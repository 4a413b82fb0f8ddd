/*
 * Attention over packed sequences and over the paged cache for every head_dim, stride and alignment: the kernel behind the matrix-core
 * ones (fa_sequences_gfx950.hip, fa_paged_gfx950.hip), which take head_dim 128 on aligned rows.
 *
 *     out[c] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q_c . k_j - max),   j over the keys of the column's sequence, causal:
 *     j <= row + (keys - rows)
 *
 * A column is one query row of one head; those of the heads that share a key-value head lie side by side. A workgroup takes QB columns of a
 * sequence; each of its waves walks every fourth 64 of its keys with a running maximum and sum, all in f32: first a key to a lane (its row dotted
 * with every column's query), then an output dim to a lane; at the end the waves' sums are joined. A key that a column does not see is passed over
 * and not multiplied by zero, whatever its row holds. head_dim beyond 512 walks the keys once for each 512 output dims.
 *
 * Bound by the latency of reads, of which each wave has few under way: 512 causal rows, 32 heads on 8, of 64 dims take 120 us, of 256 273; one
 * token of each of 48 texts of 1024 143 and 227 (with one wave to a column 204, 695, 450 and 2620). The matrix-core kernels on 128 dims: 14 and 38.
 */
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "iris_kernels_hip.h"
#include "paged_cache.h"
#include "sequences.h"

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

namespace {

constexpr int QB = 8, KT = 64, MOST_DIMS = 512, VEC = 8, WAVES = 4, THREADS = 64 * WAVES;

__device__ __forceinline__ float value(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float value(uint8_t v) { return __builtin_amdgcn_cvt_f32_fp8(v, 0); }
/* eight values from a place that is aligned to their size */
__device__ __forceinline__ void eight(const uint16_t *p, float (&v)[VEC]) {
    const u32x4 w = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
    for (int i = 0; i < VEC / 2; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void eight(const uint8_t *p, float (&v)[VEC]) {
    const u32x2 w = *reinterpret_cast<const u32x2 *>(p);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
        v[4 * i] = lo[0]; v[4 * i + 1] = lo[1]; v[4 * i + 2] = hi[0]; v[4 * i + 3] = hi[1];
    }
}
__device__ __forceinline__ uint16_t to_bf16(float f) {
    const f32x2 p = {f, 0.0f};
    return (uint16_t)__builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}
/* over all lanes, for all of them: in the vector registers (shifts inside rows of 16, then the rows' last lanes to those behind them) */
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp(float other, float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(other), __float_as_uint(v), CTRL, ROWS, 0xf, false));
}
template <class F> __device__ __forceinline__ float over_wave(float v, float none, F f) {
    v = f(v, dpp<0x111, 0xf>(none, v));
    v = f(v, dpp<0x112, 0xf>(none, v));
    v = f(v, dpp<0x114, 0xf>(none, v));
    v = f(v, dpp<0x118, 0xf>(none, v));
    v = f(v, dpp<0x142, 0xa>(none, v));
    v = f(v, dpp<0x143, 0xc>(none, v));
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}
__device__ __forceinline__ float wave_max(float v) { return over_wave(v, -INFINITY, [](float x, float y) { return fmaxf(x, y); }); }
__device__ __forceinline__ float wave_sum(float v) { return over_wave(v, 0.0f, [](float x, float y) { return x + y; }); }
/* what this wave has written to the LDS can be read by all of its lanes */
__device__ __forceinline__ void wave_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

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

/* nq columns whose queries are q + qat[c]; limit(c): the keys that column c sees are [0, limit(c)); outputs to out + oat[c]. wide: head_dim is a
 * multiple of 8 and rows of keys are aligned to 8 values */
template <int SLOTS, class Keys, class Q, class Out, class Limit>
__device__ __forceinline__ void walk(const Keys &keys, int nq, int m, int hd, float scale, bool wide, const uint16_t *q, Q qat, uint16_t *out, Out oat, Limit limit) {
    __shared__ __align__(16) float all_ps[WAVES][QB][KT], buf[WAVES][QB][64], tops[WAVES][QB], sums[WAVES][QB];
    extern __shared__ __align__(16) float qs[];                      /* [QB][head_dim], the first DIMS dims */
    constexpr int DIMS = 64 * SLOTS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), staged = min(hd, DIMS);
    auto &ps = all_ps[wave];
    for (int c = 0; c < QB; c++)
        for (int d = threadIdx.x; d < staged; d += THREADS) qs[c * staged + d] = value(q[qat(min(c, nq - 1)) + d]);
    __syncthreads();
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
        for (int tile = wave, tiles = (end + KT - 1) / KT; tile < tiles; tile += WAVES) {
            const int k0 = tile * KT, j = k0 + lane, nk = min(KT, end - k0);
            const long at = j < end ? keys.offset(j) : -1;
            float dot[QB];
#pragma unroll
            for (int c = 0; c < QB; c++) dot[c] = 0.0f;
            if (at >= 0) {
                int d = 0;
                if (wide)
#pragma unroll 4
                    for (; d < staged; d += VEC) {
                        float kd[VEC];
                        eight(keys.k + at + d, kd);
#pragma unroll
                        for (int c = 0; c < QB; c++)
#pragma unroll
                            for (int i = 0; i < VEC; i++) dot[c] = fmaf(qs[c * staged + d + i], kd[i], dot[c]);
                    }
                for (; d < hd; d++) {
                    const float kd = value(keys.k[at + d]);
#pragma unroll
                    for (int c = 0; c < QB; c++) dot[c] = fmaf(d < staged ? qs[c * staged + d] : value(q[qat(min(c, nq - 1)) + d]), kd, dot[c]);
                }
            }
            const float ks = (at >= 0 ? keys.scale(keys.ks, at) : 1.0f) * scale, vs = at >= 0 ? keys.scale(keys.vs, at) : 1.0f;
            float alpha[QB];
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
            wave_lds();
            /* the rows of V, eight under way together: lane t of the wave knows where row t is; one that is not there is read as another, and not seen */
            const unsigned long long any = __ballot(at >= 0);
            const long some = any ? __shfl(at, __ffsll(any) - 1, 64) : 0;
#pragma unroll
            for (int t = 0; t < SLOTS; t++) {
                const int d = oc + lane + 64 * t, dim = min(d, hd - 1);
                if (!any || oc + 64 * t >= hd) continue;
#pragma unroll
                for (int c = 0; c < QB; c++) acc[c][t] *= alpha[c];
                for (int i0 = 0; i0 < nk; i0 += VEC) {
                    typename Keys::T raw[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        const long row = __shfl(at, i0 + i, 64);
                        raw[i] = keys.v[(row < 0 ? some : row) + dim];
                    }
#pragma unroll
                    for (int c = 0; c < QB; c++)
#pragma unroll
                        for (int i = 0; i < VEC; i += 4) {
                            const f32x4 p = *reinterpret_cast<const f32x4 *>(&ps[c][i0 + i]);
#pragma unroll
                            for (int j = 0; j < 4; j++) acc[c][t] = p[j] < 0.0f ? acc[c][t] : fmaf(p[j], value(raw[i + j]), acc[c][t]);
                        }
                }
            }
        }
        /* the waves' sums joined, 64 dims at a time, every fourth column by a wave */
        __syncthreads();
        if (lane == 0)
#pragma unroll
            for (int c = 0; c < QB; c++) { tops[wave][c] = top[c]; sums[wave][c] = sum[c]; }
#pragma unroll
        for (int t = 0; t < SLOTS; t++) {
            if (oc + 64 * t >= hd) continue;
            __syncthreads();
#pragma unroll
            for (int c = 0; c < QB; c++) buf[wave][c][lane] = acc[c][t];
            __syncthreads();
            const int d = oc + lane + 64 * t;
            for (int c = wave; c < nq; c += WAVES) {
                float high = -INFINITY, den = 0.0f, o = 0.0f;
                for (int w = 0; w < WAVES; w++) high = fmaxf(high, tops[w][c]);
                const float base = high == -INFINITY ? 0.0f : high;
                for (int w = 0; w < WAVES; w++) {
                    const float f = expf(tops[w][c] - base);
                    o += f * buf[w][c][lane];
                    den += f * sums[w][c];
                }
                const float inv = den == 0.0f ? 0.0f : 1.0f / den;            /* no key: a row of zeros */
                if (d < hd) out[oat(c) + d] = to_bf16(o * inv);
            }
        }
    }
}

template <int SLOTS>
__global__ void __launch_bounds__(THREADS)
k_sequences_any(uint16_t *out, int ldo, const uint16_t *q, int ldq, const uint16_t *k, const uint16_t *v, int ldkv, SequencesArg seqs,
                int kv_heads, int hd, float scale, int wide, int causal) {
    SequenceTiles<> tiles;
    const int count = tiles.count(seqs, QB), t = blockIdx.x / kv_heads, kvh = blockIdx.x % kv_heads, group = seqs.per_row;
    if (t >= count) return;
    const SequenceTile s = tiles.tile(t);
    const int nq = min(QB, s.n * group - s.c0);
    const RowKeys keys = {k, v, (size_t)ldkv, s.key0, kvh * hd, nullptr, nullptr};
    auto place = [&](int c, int ld) { return (size_t)(s.row0 + (s.c0 + c) / group) * ld + (size_t)(kvh * group + (s.c0 + c) % group) * hd; };
    walk<SLOTS>(keys, nq, s.m, hd, scale, wide, q, [&](int c) { return place(c, ldq); }, out, [&](int c) { return place(c, ldo); },
         [&](int c) { return causal ? (s.c0 + c) / group + 1 + s.m - s.n : s.m; });
}

template <typename T, int SLOTS>
__global__ void __launch_bounds__(THREADS)
k_paged_any(uint16_t *out, int ldo, const uint16_t *q, int ldq, const T *k, const T *v, const uint8_t *ks, const uint8_t *vs, PagedArg cache,
            int group, float scale, int wide) {
    const int blocks = (group + QB - 1) / QB, c0 = blockIdx.x % blocks * QB, kvh = blockIdx.x / blocks % cache.kv_heads;
    const int g = blockIdx.x / blocks / cache.kv_heads, nq = min(QB, group - c0), hd = cache.head_dim, m = paged_length(cache, g);
    const PageKeys<T> keys = {k, v, ks, vs, cache, g, kvh};
    auto place = [&](int c, int ld) { return (size_t)g * ld + (size_t)(kvh * group + c0 + c) * hd; };
    walk<SLOTS>(keys, nq, m, hd, scale, wide, q, [&](int c) { return place(c, ldq); }, out, [&](int c) { return place(c, ldo); }, [&](int) { return m; });
}

bool aligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
size_t staged_bytes(int head_dim) { return (size_t)QB * (head_dim < MOST_DIMS ? head_dim : MOST_DIMS) * sizeof(float); }
/* f with the output dims of a lane: as many as the head has, at most 8 */
template <class F> void with_slots(int head_dim, F f) {
    if (head_dim <= 64) f(std::integral_constant<int, 1>{});
    else if (head_dim <= 128) f(std::integral_constant<int, 2>{});
    else if (head_dim <= 256) f(std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, MOST_DIMS / 64>{});
}
bool fits(long wgs) { return wgs <= ((1L << 32) - 1) / THREADS; }

}  // namespace

extern "C" int iris_hip_sequences_any(void *stream, uint16_t *out, int ldo, const uint16_t *q, int ldq, const uint16_t *k, const uint16_t *v,
                                      int ldkv, const int *first_row, const int *first_key, int n, int rows, int keys, int heads,
                                      int kv_heads, int head_dim, float scale, int causal) {
    const SequencesArg a = {first_row, first_key, n, rows, keys, heads / kv_heads};
    const long wgs = sequence_tiles_at_most(a, QB) * kv_heads;
    if (!wgs) return 0;
    if (!fits(wgs)) return (int)hipErrorInvalidValue;
    with_slots(head_dim, [&](auto slots) {
        hipLaunchKernelGGL(k_sequences_any<decltype(slots)::value>, dim3((unsigned)wgs), dim3(THREADS), staged_bytes(head_dim), (hipStream_t)stream, out, ldo, q, ldq,
                           k, v, ldkv, a, kv_heads, head_dim, scale, head_dim % VEC == 0 && ldkv % VEC == 0 && aligned(k, 2 * VEC), causal);
    });
    return (int)hipGetLastError();
}

extern "C" int iris_hip_paged_any(void *stream, uint16_t *out, int ldo, const uint16_t *q, int ldq, const void *k, const void *v,
                                  const uint8_t *ks, const uint8_t *vs, int pages, int page_shift, const int *table, int table_ld,
                                  const int *lengths, int n, int heads, int kv_heads, int head_dim, float scale) {
    const PagedArg c = {table, lengths, table_ld, pages, page_shift, kv_heads, head_dim};
    const int group = heads / kv_heads;
    const long wgs = (long)n * kv_heads * ((group + QB - 1) / QB);
    if (!fits(wgs)) return (int)hipErrorInvalidValue;
    with_slots(head_dim, [&](auto slots) {
        constexpr int SLOTS = decltype(slots)::value;
        if (ks)
            hipLaunchKernelGGL((k_paged_any<uint8_t, SLOTS>), dim3((unsigned)wgs), dim3(THREADS), staged_bytes(head_dim), (hipStream_t)stream, out, ldo, q, ldq,
                               (const uint8_t *)k, (const uint8_t *)v, ks, vs, c, group, scale, head_dim % VEC == 0 && aligned(k, VEC));
        else
            hipLaunchKernelGGL((k_paged_any<uint16_t, SLOTS>), dim3((unsigned)wgs), dim3(THREADS), staged_bytes(head_dim), (hipStream_t)stream, out, ldo, q, ldq,
                               (const uint16_t *)k, (const uint16_t *)v, nullptr, nullptr, c, group, scale, head_dim % VEC == 0 && aligned(k, 2 * VEC));
    });
    return (int)hipGetLastError();
}
