/*
 * Rows of K and V into the pages of a cache (paged_cache.h) and back, as bf16 or as e4m3 codes with a scale for each row of a head.
 *
 * Quantising a row x of head_dim values: 2^e is the smallest power of two with max |x| <= 448 * 2^e (448 is the largest e4m3 value), at
 * least 2^-127; the codes are x / 2^e rounded to the nearest code, ties to the even one. Dividing by a power of two is exact, so that
 * one rounding is the only one, at most half a step, 2^-4 of the value (2^-10 of 2^e below 2^-6 of it), and no value saturates. From
 * the bits of the largest magnitude, sign off: e = exponent - 8, one more where its fraction is above .75. A row with an infinity or a
 * NaN in it becomes NaN as a whole (scale byte 255, all codes 0x7f).
 *
 * The rows of a call are the last ones of their sequences: row i of n is position length - n + i. A workgroup takes ROWS rows of one
 * sequence, of K or of V. Bound by memory: each value is read and written once. 95547 rows of 8 heads x 128 read back from 8 bits (587 MB)
 * take 125 us, 4.7 TB/s, two thirds of it written (a copy reaches 4.9); 2692 rows written in 8 bits 6.2 us and read back 7.0 (16 MB each);
 * 48 rows 3 us, a launch and four dependent reads (bounds, length, page, row).
 */
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "iris_kernels_hip.h"
#include "paged_cache.h"
#include "sequences.h"

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

namespace {

constexpr int ROWS = 16, THREADS = 256, UNROLL = 4;                  /* rows of a workgroup; four times as many in a large call, a quarter in a small one */

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const f32x2 p = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}

/* position of row `row` of the sequence, or -1 where the cache has no place for it */
__device__ __forceinline__ int position(const PagedArg &c, const SequenceTile &s, int row) {
    const int pos = max(c.lengths[s.g], 0) - s.n + row;
    return pos >= 0 && pos < ((long)c.ld << c.shift) ? pos : -1;
}

struct Pair { void *k, *v; };
struct ConstPair { const void *k, *v; };

/* head_dim HEAD, rows 16-byte aligned. A unit is 8 values of bf16, 16 of 8 bits (16 bytes of the pages), of consecutive lanes; a thread has
 * the loads of UNROLL units under way together. The places of the rows are looked up once, a row to a thread. magic: 2^32 / kv_heads rounded
 * up, which divides numbers of rows of heads up to ROWS * kv_heads exactly while kv_heads < 8192; 0 for one head. */
template <int HEAD, bool FP8, bool WRITE, int ROWS>
__global__ void __launch_bounds__(THREADS)
k_cache_rows(Pair pages, Pair scales, ConstPair rows, Pair out, int ld, PagedArg cache, SequencesArg seqs, uint32_t magic) {
    constexpr int VALUES = FP8 ? 16 : 8, LANES = HEAD / VALUES, WORDS = FP8 ? 2 : 1;      /* 16-byte words of bf16 to a unit */
    __shared__ long places[ROWS];
    SequenceTiles<> tiles;
    const int count = tiles.count(seqs, ROWS), t = blockIdx.x >> 1;
    if (t >= count) return;
    const bool second = blockIdx.x & 1;
    const SequenceTile s = tiles.tile(t);
    const int n = min(ROWS, s.n - s.c0), units = n * cache.kv_heads * LANES;
    if (threadIdx.x < n) {
        const int pos = position(cache, s, s.c0 + threadIdx.x);
        places[threadIdx.x] = pos < 0 ? -1 : paged_row(cache, s.g, pos, 0);
    }
    __syncthreads();
    uint8_t *bytes = (uint8_t *)(second ? scales.v : scales.k);
    u32x4 *in_pages = (u32x4 *)(second ? pages.v : pages.k);         /* of LANES words to a row */
    const uint16_t *from = (const uint16_t *)(second ? rows.v : rows.k);
    uint16_t *to = (uint16_t *)(second ? out.v : out.k);
    for (int u0 = threadIdx.x; u0 < units; u0 += THREADS * UNROLL) {
        long place[UNROLL];
        size_t at[UNROLL];
        u32x4 x[UNROLL][WORDS], code[UNROLL];                        /* of a vector type: arrays of structs go into the LDS, by an address that is
                                                                      * read from the host's memory: 1690 rows 15 us, with these 4 */
        unsigned byte[UNROLL];
#pragma unroll
        for (int j = 0; j < UNROLL; j++) {
            const int u = min(u0 + j * THREADS, units - 1), lane = u % LANES, row = magic ? (int)__umulhi((unsigned)(u / LANES), magic) : u / LANES;
            const int head = u / LANES - row * cache.kv_heads;
            const long first = u0 + j * THREADS < units ? places[row] : -1;
            place[j] = first < 0 ? -1 : first + ((long)head << cache.shift);       /* the same for the LANES lanes of a row */
            at[j] = (size_t)(s.row0 + s.c0 + row) * ld + (size_t)head * HEAD + VALUES * lane;
            const long safe = max(place[j], 0L) * LANES + lane;
            if (WRITE) {
#pragma unroll
                for (int i = 0; i < WORDS; i++) x[j][i] = *reinterpret_cast<const u32x4 *>(from + at[j] + 8 * i);
            } else if (place[j] >= 0) {
                code[j] = in_pages[safe];
                if (FP8) byte[j] = bytes[place[j]];
            }
        }
#pragma unroll
        for (int j = 0; j < UNROLL; j++) {
            const int lane = (u0 + j * THREADS) % LANES;
            if constexpr (WRITE && FP8) {
                const unsigned w[8] = {x[j][0][0], x[j][0][1], x[j][0][2], x[j][0][3], x[j][WORDS - 1][0], x[j][WORDS - 1][1], x[j][WORDS - 1][2], x[j][WORDS - 1][3]};
                unsigned top = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) top = max(top, max(w[i] & 0x7fff, (w[i] >> 16) & 0x7fff));
#pragma unroll
                for (int d = 1; d < LANES; d <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, d, 64));
                float factor;
                byte[j] = scale_byte(top, &factor);
                int c[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float lo = __uint_as_float(w[i] << 16) * factor, hi = __uint_as_float(w[i] & 0xffff0000u) * factor;
                    c[i / 2] = i % 2 ? __builtin_amdgcn_cvt_pk_fp8_f32(lo, hi, c[i / 2], true) : __builtin_amdgcn_cvt_pk_fp8_f32(lo, hi, c[i / 2], false);
                }
                code[j] = byte[j] == 255 ? u32x4{0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f} : u32x4{(unsigned)c[0], (unsigned)c[1], (unsigned)c[2], (unsigned)c[3]};
            }
            if (place[j] < 0) continue;
            if constexpr (WRITE) {
                in_pages[place[j] * LANES + lane] = FP8 ? code[j] : x[j][0];
                if (FP8 && lane == 0) bytes[place[j]] = (uint8_t)byte[j];
            } else if constexpr (FP8) {
                const float scale = paged_scale(byte[j]);
                const u32x4 c = code[j];
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const f32x2 f = i % 2 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i / 2], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i / 2], false);
                    w[i] = pack_bf16(f[0] * scale, f[1] * scale);
                }
                *reinterpret_cast<u32x4 *>(to + at[j]) = u32x4{w[0], w[1], w[2], w[3]};
                *reinterpret_cast<u32x4 *>(to + at[j] + 8) = u32x4{w[4], w[5], w[6], w[7]};
            } else {
                *reinterpret_cast<u32x4 *>(to + at[j]) = code[j];
            }
        }
    }
}

/* any head_dim, stride and alignment: a wave to a row of a head */
template <bool FP8, bool WRITE>
__global__ void __launch_bounds__(THREADS)
k_cache_rows_any(Pair pages, Pair scales, ConstPair rows, Pair out, int ld, PagedArg cache, SequencesArg seqs) {
    SequenceTiles<> tiles;
    const int count = tiles.count(seqs, ROWS), t = blockIdx.x >> 1, hd = cache.head_dim;
    if (t >= count) return;
    const bool second = blockIdx.x & 1;
    const SequenceTile s = tiles.tile(t);
    const int units = min(ROWS, s.n - s.c0) * cache.kv_heads, lane = threadIdx.x & 63;
    uint8_t *codes = (uint8_t *)(second ? pages.v : pages.k), *bytes = (uint8_t *)(second ? scales.v : scales.k);
    uint16_t *plain = (uint16_t *)(second ? pages.v : pages.k);
    const uint16_t *from = (const uint16_t *)(second ? rows.v : rows.k);
    uint16_t *to = (uint16_t *)(second ? out.v : out.k);
    for (int u = threadIdx.x >> 6; u < units; u += THREADS / 64) {
        const int head = u % cache.kv_heads, row = s.c0 + u / cache.kv_heads;
        const int pos = position(cache, s, row);
        const long place = pos < 0 ? -1 : paged_row(cache, s.g, pos, head);
        if (place < 0) continue;
        const size_t at = (size_t)(s.row0 + row) * ld + (size_t)head * hd, in_pages = (size_t)place * hd;
        if constexpr (!FP8) {
            for (int d = lane; d < hd; d += 64)
                if (WRITE) plain[in_pages + d] = from[at + d];
                else to[at + d] = plain[in_pages + d];
        } else if constexpr (WRITE) {
            unsigned top = 0;
            for (int d = lane; d < hd; d += 64) top = max(top, (unsigned)(from[at + d] & 0x7fff));
            for (int d = 1; d < 64; d <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, d, 64));
            float factor;
            const unsigned byte = scale_byte(top, &factor);
            for (int d = lane; d < hd; d += 64) {
                const int c = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float((uint32_t)from[at + d] << 16) * factor, 0.0f, 0, false);
                codes[in_pages + d] = byte == 255 ? (uint8_t)0x7f : (uint8_t)c;
            }
            if (lane == 0) bytes[place] = (uint8_t)byte;
        } else {
            const float scale = paged_scale(bytes[place]);
            for (int d = lane; d < hd; d += 64)
                to[at + d] = (uint16_t)pack_bf16(__builtin_amdgcn_cvt_f32_fp8(codes[in_pages + d], 0) * scale, 0.0f);
        }
    }
}

bool aligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

template <bool FP8, bool WRITE>
int launch(hipStream_t stream, Pair pages, Pair scales, ConstPair rows, Pair out, int ld, const PagedArg &c, const SequencesArg &seqs) {
    const bool wide = ld % 8 == 0 && aligned(WRITE ? rows.k : out.k, 16) && aligned(WRITE ? rows.v : out.v, 16) && aligned(pages.k, 16) &&
                      aligned(pages.v, 16) && (c.head_dim == 128 || c.head_dim == 64 || c.head_dim == 256) && c.kv_heads < 8192;
    const long bytes = (long)c.kv_heads * c.head_dim * (FP8 ? 1 : 2);                     /* of a row in the pages */
    /* many rows of few bytes, of which 16 are little work for what finding them takes: 100000 of one head in 8 bits written in 25 us, with 64 to a workgroup
     * 15; of 8 heads 118 and 128, and read back 132 and 153 */
    const bool large = wide && bytes <= 256 && seqs.rows >= 1 << 14 && seqs.rows / 32 >= seqs.n;
    /* 4 to a workgroup: few rows, of which 16 would leave most CUs without any (300 rows of 24 heads in 8 bits written 8.0 us, with 4 5.0; but 3219 of 8
     * heads 5.7 and 7.7), single ones, and rows of many bytes (30000 of 24 heads in 8 bits 112 and 105, read back 145 and 128; 100000 of 8 in bf16 156 and
     * 140; but in 8 bits 118 and 148) */
    const bool small = wide && !large && (sequence_tiles_at_most(seqs, ROWS) <= 128 || seqs.rows / 4 <= seqs.n || bytes >= 2048);
    const long wgs = 2 * sequence_tiles_at_most(seqs, large ? 4 * ROWS : small ? ROWS / 4 : ROWS);
    if (!wgs) return 0;
    if (wgs > ((1L << 32) - 1) / THREADS) return (int)hipErrorInvalidValue;
    const dim3 grid((unsigned)wgs), block(THREADS);
    const uint32_t magic = c.kv_heads > 1 ? (uint32_t)(((1ull << 32) + c.kv_heads - 1) / c.kv_heads) : 0;
    auto rows_of = [&](auto head) {
        constexpr int HEAD = decltype(head)::value;
        if (large) hipLaunchKernelGGL((k_cache_rows<HEAD, FP8, WRITE, 4 * ROWS>), grid, block, 0, stream, pages, scales, rows, out, ld, c, seqs, magic);
        else if (small) hipLaunchKernelGGL((k_cache_rows<HEAD, FP8, WRITE, ROWS / 4>), grid, block, 0, stream, pages, scales, rows, out, ld, c, seqs, magic);
        else hipLaunchKernelGGL((k_cache_rows<HEAD, FP8, WRITE, ROWS>), grid, block, 0, stream, pages, scales, rows, out, ld, c, seqs, magic);
    };
    if (wide && c.head_dim == 128) rows_of(std::integral_constant<int, 128>{});
    else if (wide && c.head_dim == 64) rows_of(std::integral_constant<int, 64>{});
    else if (wide) rows_of(std::integral_constant<int, 256>{});
    else hipLaunchKernelGGL((k_cache_rows_any<FP8, WRITE>), grid, block, 0, stream, pages, scales, rows, out, ld, c, seqs);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" int iris_hip_cache_write(void *stream, void *k_pages, void *v_pages, uint8_t *k_scales, uint8_t *v_scales, int pages, int page_shift,
                                    const int *table, int table_ld, const int *lengths, const uint16_t *k, const uint16_t *v, int ld,
                                    const int *first_row, int n, int rows, int kv_heads, int head_dim) {
    const PagedArg c = {table, lengths, table_ld, pages, page_shift, kv_heads, head_dim};
    const SequencesArg s = {first_row, nullptr, n, rows, 0, 1};
    const Pair scales = {k_scales, v_scales}, none = {nullptr, nullptr};
    return k_scales ? launch<true, true>((hipStream_t)stream, {k_pages, v_pages}, scales, {k, v}, none, ld, c, s)
                    : launch<false, true>((hipStream_t)stream, {k_pages, v_pages}, scales, {k, v}, none, ld, c, s);
}

extern "C" int iris_hip_cache_read(void *stream, uint16_t *k, uint16_t *v, int ld, const void *k_pages, const void *v_pages,
                                   const uint8_t *k_scales, const uint8_t *v_scales, int pages, int page_shift, const int *table, int table_ld,
                                   const int *lengths, const int *first_row, int n, int rows, int kv_heads, int head_dim) {
    const PagedArg c = {table, lengths, table_ld, pages, page_shift, kv_heads, head_dim};
    const SequencesArg s = {first_row, nullptr, n, rows, 0, 1};
    const Pair at = {const_cast<void *>(k_pages), const_cast<void *>(v_pages)}, scales = {const_cast<uint8_t *>(k_scales), const_cast<uint8_t *>(v_scales)};
    return k_scales ? launch<true, false>((hipStream_t)stream, at, scales, {nullptr, nullptr}, {k, v}, ld, c, s)
                    : launch<false, false>((hipStream_t)stream, at, scales, {nullptr, nullptr}, {k, v}, ld, c, s);
}
