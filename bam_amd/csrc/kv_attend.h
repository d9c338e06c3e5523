// The key-value cache in the pages of an array: attention of the newest tokens over what the cache holds.
#ifndef __BAM_KV_ATTEND_H__
#define __BAM_KV_ATTEND_H__
#include "kv_cache.h"

struct kv_att {
    const uint16_t* q;
    int64_t q_row, q_head;
    uint32_t aligned, q_heads, group;   /* group: heads of queries to a head of keys */
    float scale;                        /* times log2(e) */
    uint32_t window, sinks;             /* window 0: none */
    uint16_t* out;                      /* [rows][q_heads][dim] */
    float* lse;                         /* [rows][q_heads] or NULL */
    uint32_t tiles, splits, steps;      /* tiles of rows of a sequence, splits of its tokens, steps of 32 tokens to a split */
    float* part;                        /* [item][rows of a tile][split][dim] sums, then their maxima and denominators [item][row][split] each */
    float *part_m, *part_l;
    uint8_t* left;                      /* [item][split] pages were missing */
    uint32_t chunk;                     /* blocks whose pages a wave asks for at a time when it holds them */
    uint32_t items, tile_rows, max_new;
};
/* (bam_kv8.hip) */
struct kv_plan;
void kv8_rows(const bam_kv_t* kv, const kv_seqs& s, const kv_rows& io, bool write, hipStream_t st);
void kv8_attend(const bam_kv_t* kv, const kv_seqs& s, const kv_att& a, const kv_plan& p, hipStream_t st);
struct kv_plan { uint32_t nt, waves, rows, tiles, splits, steps; uint64_t items, left_at, m_at, l_at, part_at, bytes; };

namespace {

template <int F16> __device__ __forceinline__ f32x4 mma(const u32x4 a, const u32x4 b, const f32x4 c)
{
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
/* the halves of the wave, or the rows of sixteen lanes of each half, exchanged between two registers that hold the same: then one of them has a lane's own, the other
 * its partner's.  (The results go through scalars: a bit cast of a vector's element takes its first one, whichever is named.) */
__device__ __forceinline__ void swap_halves(float& a, float& b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
    const uint32_t x = r[0], y = r[1];
    a = __builtin_bit_cast(float, x);
    b = __builtin_bit_cast(float, y);
}
__device__ __forceinline__ void swap_rows(float& a, float& b)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
    const uint32_t x = r[0], y = r[1];
    a = __builtin_bit_cast(float, x);
    b = __builtin_bit_cast(float, y);
}
__device__ __forceinline__ float max_of_four(float a)
{
    float b = a;
    swap_halves(a, b);
    a = b = fmaxf(a, b);
    swap_rows(a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float sum_of_four(float a)
{
    float b = a;
    swap_halves(a, b);
    a = b = a + b;
    swap_rows(a, b);
    return a + b;
}
/*
 * Weights go to the product with the values in 16 bits: exp2(score - maximum + WEIGHT_SHIFT).  A float16 has full precision from 2^-14 on and nothing below 2^-25, and a
 * quarter of a million tokens of 2^-25 of the largest weigh 2^-7 of it: they are scaled up by a power of two that the type has room for (2^16), and the sums with them.  In
 * tiles, weights are up to 2^TILE_SLACK before the maximum is followed.  What falls below 2^-25 now is 2^-39 (2^-36 in tiles) of the largest.  A bfloat16 has a float's range.
 */
template <int F16> constexpr float WEIGHT_SHIFT = F16 ? 14.0f : 0.0f;
template <int F16> constexpr float TILE_SLACK = F16 ? 4.0f : 8.0f;
template <int F16> constexpr float TILE_SHIFT = F16 ? 11.0f : 0.0f;
/* whether one of the two 16-bit numbers is an infinity or NaN */
template <int F16> __device__ __forceinline__ bool odd16(const uint32_t x)
{
    constexpr uint32_t e = F16 ? 0x7c00u : 0x7f80u;
    return (x & e) == e || ((x >> 16) & e) == e;
}
/*
 * The pieces of a step, each at an address of the lane's own, loaded past the vector L1 like all payload and marked as not to be kept (bam_wave.h, ld_payload_nt): the
 * keys of the two tiles of 16 tokens, and the values.  With their wait in one statement: the compiler does not count what an asm statement leaves in flight.  (Ordinary
 * loads behind an acquire for each chunk overlap the scores with the wait for the values, and lost 3 to 30 % to what an acquire invalidates.)
 * SECOND: from a token's keys to the second tile's, 128 bytes, or 64 where a block has eight tokens.
 */
template <int SECOND> __device__ __forceinline__ void load_step(const uint8_t* const (&k)[2], const uint8_t* const (&v)[4], u32x4 (&k0)[2], u32x4 (&k1)[2], u32x4 (&x)[4])
{
    if constexpr (SECOND == 64)
        asm volatile("global_load_dwordx4 %0, %8, off sc1 nt\n\t"
                     "global_load_dwordx4 %1, %9, off sc1 nt\n\t"
                     "global_load_dwordx4 %2, %8, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %3, %9, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %4, %10, off sc1 nt\n\t"
                     "global_load_dwordx4 %5, %11, off sc1 nt\n\t"
                     "global_load_dwordx4 %6, %12, off sc1 nt\n\t"
                     "global_load_dwordx4 %7, %13, off sc1 nt\n\t"
                     "s_waitcnt vmcnt(0)"
                     : "=&v"(k0[0]), "=&v"(k0[1]), "=&v"(k1[0]), "=&v"(k1[1]), "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
                     : "v"(k[0]), "v"(k[1]), "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]) : "memory");
    if constexpr (SECOND == 128)
        asm volatile("global_load_dwordx4 %0, %8, off sc1 nt\n\t"
                     "global_load_dwordx4 %1, %9, off sc1 nt\n\t"
                     "global_load_dwordx4 %2, %8, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %3, %9, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %4, %10, off sc1 nt\n\t"
                     "global_load_dwordx4 %5, %11, off sc1 nt\n\t"
                     "global_load_dwordx4 %6, %12, off sc1 nt\n\t"
                     "global_load_dwordx4 %7, %13, off sc1 nt\n\t"
                     "s_waitcnt vmcnt(0)"
                     : "=&v"(k0[0]), "=&v"(k0[1]), "=&v"(k1[0]), "=&v"(k1[1]), "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
                     : "v"(k[0]), "v"(k[1]), "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]) : "memory");
}
template <int SECOND> __device__ __forceinline__ void load_step(const uint8_t* const (&k)[4], const uint8_t* const (&v)[8], u32x4 (&k0)[4], u32x4 (&k1)[4], u32x4 (&x)[8])
{
    if constexpr (SECOND == 64)
        asm volatile("global_load_dwordx4 %0, %16, off sc1 nt\n\t"
                     "global_load_dwordx4 %1, %17, off sc1 nt\n\t"
                     "global_load_dwordx4 %2, %18, off sc1 nt\n\t"
                     "global_load_dwordx4 %3, %19, off sc1 nt\n\t"
                     "global_load_dwordx4 %4, %16, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %5, %17, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %6, %18, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %7, %19, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %8, %20, off sc1 nt\n\t"
                     "global_load_dwordx4 %9, %21, off sc1 nt\n\t"
                     "global_load_dwordx4 %10, %22, off sc1 nt\n\t"
                     "global_load_dwordx4 %11, %23, off sc1 nt\n\t"
                     "global_load_dwordx4 %12, %24, off sc1 nt\n\t"
                     "global_load_dwordx4 %13, %25, off sc1 nt\n\t"
                     "global_load_dwordx4 %14, %26, off sc1 nt\n\t"
                     "global_load_dwordx4 %15, %27, off sc1 nt\n\t"
                     "s_waitcnt vmcnt(0)"
                     : "=&v"(k0[0]), "=&v"(k0[1]), "=&v"(k0[2]), "=&v"(k0[3]), "=&v"(k1[0]), "=&v"(k1[1]), "=&v"(k1[2]), "=&v"(k1[3]), "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
                     : "v"(k[0]), "v"(k[1]), "v"(k[2]), "v"(k[3]), "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[4]), "v"(v[5]), "v"(v[6]), "v"(v[7]) : "memory");
    if constexpr (SECOND == 128)
        asm volatile("global_load_dwordx4 %0, %16, off sc1 nt\n\t"
                     "global_load_dwordx4 %1, %17, off sc1 nt\n\t"
                     "global_load_dwordx4 %2, %18, off sc1 nt\n\t"
                     "global_load_dwordx4 %3, %19, off sc1 nt\n\t"
                     "global_load_dwordx4 %4, %16, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %5, %17, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %6, %18, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %7, %19, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %8, %20, off sc1 nt\n\t"
                     "global_load_dwordx4 %9, %21, off sc1 nt\n\t"
                     "global_load_dwordx4 %10, %22, off sc1 nt\n\t"
                     "global_load_dwordx4 %11, %23, off sc1 nt\n\t"
                     "global_load_dwordx4 %12, %24, off sc1 nt\n\t"
                     "global_load_dwordx4 %13, %25, off sc1 nt\n\t"
                     "global_load_dwordx4 %14, %26, off sc1 nt\n\t"
                     "global_load_dwordx4 %15, %27, off sc1 nt\n\t"
                     "s_waitcnt vmcnt(0)"
                     : "=&v"(k0[0]), "=&v"(k0[1]), "=&v"(k0[2]), "=&v"(k0[3]), "=&v"(k1[0]), "=&v"(k1[1]), "=&v"(k1[2]), "=&v"(k1[3]), "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
                     : "v"(k[0]), "v"(k[1]), "v"(k[2]), "v"(k[3]), "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[4]), "v"(v[5]), "v"(v[6]), "v"(v[7]) : "memory");
}
template <int SECOND> __device__ __forceinline__ void load_keys(const uint8_t* const (&k)[8], u32x4 (&k0)[8], u32x4 (&k1)[8])
{
    if constexpr (SECOND == 64)
        asm volatile("global_load_dwordx4 %0, %16, off sc1 nt\n\t"
                     "global_load_dwordx4 %1, %17, off sc1 nt\n\t"
                     "global_load_dwordx4 %2, %18, off sc1 nt\n\t"
                     "global_load_dwordx4 %3, %19, off sc1 nt\n\t"
                     "global_load_dwordx4 %4, %20, off sc1 nt\n\t"
                     "global_load_dwordx4 %5, %21, off sc1 nt\n\t"
                     "global_load_dwordx4 %6, %22, off sc1 nt\n\t"
                     "global_load_dwordx4 %7, %23, off sc1 nt\n\t"
                     "global_load_dwordx4 %8, %16, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %9, %17, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %10, %18, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %11, %19, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %12, %20, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %13, %21, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %14, %22, off offset:64 sc1 nt\n\t"
                     "global_load_dwordx4 %15, %23, off offset:64 sc1 nt\n\t"
                     "s_waitcnt vmcnt(0)"
                     : "=&v"(k0[0]), "=&v"(k0[1]), "=&v"(k0[2]), "=&v"(k0[3]), "=&v"(k0[4]), "=&v"(k0[5]), "=&v"(k0[6]), "=&v"(k0[7]), "=&v"(k1[0]), "=&v"(k1[1]), "=&v"(k1[2]), "=&v"(k1[3]), "=&v"(k1[4]), "=&v"(k1[5]), "=&v"(k1[6]), "=&v"(k1[7])
                     : "v"(k[0]), "v"(k[1]), "v"(k[2]), "v"(k[3]), "v"(k[4]), "v"(k[5]), "v"(k[6]), "v"(k[7]) : "memory");
    if constexpr (SECOND == 128)
        asm volatile("global_load_dwordx4 %0, %16, off sc1 nt\n\t"
                     "global_load_dwordx4 %1, %17, off sc1 nt\n\t"
                     "global_load_dwordx4 %2, %18, off sc1 nt\n\t"
                     "global_load_dwordx4 %3, %19, off sc1 nt\n\t"
                     "global_load_dwordx4 %4, %20, off sc1 nt\n\t"
                     "global_load_dwordx4 %5, %21, off sc1 nt\n\t"
                     "global_load_dwordx4 %6, %22, off sc1 nt\n\t"
                     "global_load_dwordx4 %7, %23, off sc1 nt\n\t"
                     "global_load_dwordx4 %8, %16, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %9, %17, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %10, %18, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %11, %19, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %12, %20, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %13, %21, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %14, %22, off offset:128 sc1 nt\n\t"
                     "global_load_dwordx4 %15, %23, off offset:128 sc1 nt\n\t"
                     "s_waitcnt vmcnt(0)"
                     : "=&v"(k0[0]), "=&v"(k0[1]), "=&v"(k0[2]), "=&v"(k0[3]), "=&v"(k0[4]), "=&v"(k0[5]), "=&v"(k0[6]), "=&v"(k0[7]), "=&v"(k1[0]), "=&v"(k1[1]), "=&v"(k1[2]), "=&v"(k1[3]), "=&v"(k1[4]), "=&v"(k1[5]), "=&v"(k1[6]), "=&v"(k1[7])
                     : "v"(k[0]), "v"(k[1]), "v"(k[2]), "v"(k[3]), "v"(k[4]), "v"(k[5]), "v"(k[6]), "v"(k[7]) : "memory");
}
__device__ __forceinline__ void load_pieces(const uint8_t* const (&v)[8], u32x4* x)
{
    u32x4 y[8];
    asm volatile("global_load_dwordx4 %0, %8, off sc1 nt\n\t"
                     "global_load_dwordx4 %1, %9, off sc1 nt\n\t"
                     "global_load_dwordx4 %2, %10, off sc1 nt\n\t"
                     "global_load_dwordx4 %3, %11, off sc1 nt\n\t"
                     "global_load_dwordx4 %4, %12, off sc1 nt\n\t"
                     "global_load_dwordx4 %5, %13, off sc1 nt\n\t"
                     "global_load_dwordx4 %6, %14, off sc1 nt\n\t"
                     "global_load_dwordx4 %7, %15, off sc1 nt\n\t"
                     "s_waitcnt vmcnt(0)"
                     : "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3]), "=&v"(y[4]), "=&v"(y[5]), "=&v"(y[6]), "=&v"(y[7])
                     : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[4]), "v"(v[5]), "v"(v[6]), "v"(v[7]) : "memory");
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = y[i];
}

/* of the eight tokens from t on, those up to `last` that are not before `low`, or are before `sinks` */
__device__ __forceinline__ uint32_t seen_of_eight(const int32_t t, const int32_t last, const int32_t low, const int32_t sinks)
{
    auto below = [t](const int32_t end) { const int32_t n = end - t; return (1u << (n < 0 ? 0 : n > 8 ? 8 : n)) - 1u; };
    return below(last + 1) & (~below(low) | below(sinks));
}
/* the first token that a row at `pos` sees through the window */
__device__ __forceinline__ int32_t low_of(const kv_att& a, const int32_t pos) { return a.window && pos >= (int32_t)a.window ? pos - (int32_t)a.window + 1 : 0; }
/* eight 16-bit numbers, those whose bit is not set as zero */
__device__ __forceinline__ u32x4 only(u32x4 x, const uint32_t bits)
{
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] &= ((bits >> (2 * e)) & 1u) * 0xffffu | ((bits >> (2 * e + 1)) & 1u) * 0xffff0000u;
    return x;
}

/* whether one of the four e4m3 numbers is NaN */
__device__ __forceinline__ bool odd8(const uint32_t x) { return (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }
/* half a piece of keys in 8 bits: eight numbers of a token as an operand in 16 */
template <int F16> __device__ __forceinline__ u32x4 keys_of(const uint32_t lo, const uint32_t hi, const float by)
{
    return u32x4{from8<F16, false>(lo, by), from8<F16, true>(lo, by), from8<F16, false>(hi, by), from8<F16, true>(hi, by)};
}
/* a piece of values in 8 bits: numbers 2x and 2x + 1 of eight tokens, each with its own power of two, as two operands in 16 */
template <int F16> __device__ __forceinline__ void values_of(const u32x4 x, const float (&by)[8], u32x4& a, u32x4& b)
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = x[i], y = from8<F16, false>(w, by[2 * i]), z = from8<F16, true>(w, by[2 * i + 1]);
        a[i] = __builtin_amdgcn_perm(z, y, 0x05040100u);         /* the low halves, and the high ones: an instruction each, four with masks */
        b[i] = __builtin_amdgcn_perm(z, y, 0x07060302u);
    }
}

/* which tokens a tile of rows sees, and the order in which they are gone through: steps of 32 tokens, first those that stay visible in front of the window */
struct kv_span {
    int32_t first_pos, last_pos;        /* positions of the tile's rows */
    uint32_t len;                       /* tokens to look at: up to the last row's */
    uint32_t low, front, base, n_steps; /* first token of the window; steps in front of it; first token of the step it begins in; steps */
};
__device__ __forceinline__ kv_span span_of(const kv_att& a, const uint32_t most, const int32_t p0 /* position of the sequence's first new row */, const uint32_t r0, const uint32_t r1)
{
    kv_span s;
    s.first_pos = p0 + (int32_t)(r0 / a.group);
    s.last_pos = p0 + (int32_t)((r1 - 1) / a.group);
    s.len = s.last_pos < 0 ? 0u : (uint32_t)s.last_pos + 1u;
    if (s.len > most) s.len = most;             /* what lies past the table is not visible */
    s.low = a.window && s.first_pos + 1 > (int64_t)a.window ? (uint32_t)(s.first_pos + 1) - a.window : 0u;
    const uint32_t sinks = a.sinks < s.low ? a.sinks : s.low;
    s.front = (sinks + 31u) / 32u;
    s.base = s.low & ~31u;
    if (s.front * 32u >= s.base) { s.front = 0; s.base = 0; }
    s.n_steps = s.front + (s.len > s.base ? (s.len - s.base + 31u) / 32u : 0u);
    return s;
}

/*
 * One wave's share of a split: steps [v0, v1) for NT tiles of 16 rows.  Lane l: row l % 16, tokens 8 (l / 16) .. + 7 of each step.
 * The largest score and the denominator (of this lane's tokens) and the sums of every row are carried over the steps in 32 bits; exp(score - max) is
 * rounded to 16 bits for the product with the values, which the matrix unit takes in 16 bits; the denominator is the sum of what was not rounded.
 *
 * HELD false: pages are read without a reference, a chunk of 32 blocks at a time: one look at their descriptors, the reads (past the L1: a slot may have
 * been refilled since this compute unit last read it), and a second look that has to find the same.  False if a page was missing or has gone.
 * HELD true: the pages of a.chunk blocks at a time are asked for, and held together if they can be had without waiting while one is held; else each is brought in and given
 * back, and they are asked for again.  If others have pushed some of them out by then, the pages of each step are loaded one by one, those of a step that came are loaded and given
 * back before the next is waited for: no wave waits for a slot while it keeps another, however many calls share the page cache.  `gone` is set, and the rest left, where a wait was given up.
 *   Bound by the reads of keys and values, each once and marked as not to be kept (without the mark 10 % slower): a step's 16 KiB are on their way at once, the matrix unit is idle most of the
 * time, and what is left of a tile of 16 rows by a group of four heads costs nothing.  128 sequences of up to 8192 tokens, 3.2 GB: 511 us, 6.3 TB/s (a copy
 * reaches 4.9 on this card, a plain reader 7.2); 64 of up to 4099: 142 us, 5.6 TB/s, the longest sequence's workgroups last; one of 262121: 165 us, 6.5 TB/s with the join.  More waves to
 * a SIMD (three, four) were 9 % slower.
 */
template <int DP, int F16, int E8, int NT, bool HELD>
__device__ __forceinline__ bool kv_steps(const kv_geom& g, const kv_seqs& s, const kv_att& a, const kv_span& sp, const uint32_t seq, const uint32_t head, const uint32_t v0, const uint32_t v1,
                                         const u32x4 (&q)[NT][DP / 32], const int32_t (&pos)[NT], f32x4 (&o)[NT][DP / 16], float (&m)[NT], float (&l)[NT], bool& gone, uint32_t& n_access, uint32_t& n_hit)
{
    using namespace bam;
    const uint32_t lane = bam::lane(), row = lane & 15u, grp = lane >> 4;
    const uint32_t T = g.tokens, D = g.dim;
    /* 8 bits: half the bytes to a step of 32 tokens, so two steps at a time, or as little as before would be on its way */
    constexpr int HALVES = E8 && DP <= 128 ? 2 : 1, KP = E8 ? DP / 64 : DP / 32, VP = E8 ? DP / 32 : DP / 16;      /* pieces of a token's keys, and of eight tokens' values, to a lane */
    for (uint32_t v = v0; v < v1;) {
        /* a run of neighbouring steps within one chunk of blocks */
        const bool front = v < sp.front;
        const uint32_t t_first = front ? v * 32u : sp.base + (v - sp.front) * 32u;
        const uint32_t run = (front && sp.front < v1 ? sp.front : v1) - v;
        const uint32_t b_first = t_first >> g.tokens_log, n_chunk = HELD ? a.chunk : 32u;
        uint32_t t_end = (b_first + n_chunk) << g.tokens_log;
        if (t_first + run * 32u < t_end) t_end = t_first + run * 32u;
        const uint32_t t_seen = t_end < sp.len ? t_end : sp.len;                  /* tokens from here on are not looked at */
        /* lanes 0..31: the pages of keys, 32..63: of values */
        const uint32_t blk = b_first + (lane & 31u);
        uint64_t page = 0;
        const bool in_run = (lane & 31u) < n_chunk && (blk << g.tokens_log) < t_end, asked = in_run && (blk << g.tokens_log) < t_seen;
        const bool need = asked && page_of_block(g, s, seq, blk, head, page);
        if (lane >= 32) page += 1;
        /* blocks the table does not have, or that lie past its end (the last step may go on behind it): their tokens are not visible */
        const uint32_t holes = (uint32_t)ballot((asked && !need) || (in_run && blk >= s.width));
        uint32_t slot = 0;
        [[maybe_unused]] const uint64_t powers_at = need ? page - g.first_page : 0u;      /* where a lane's page has its powers of two (a block that is not there: the first, which it does not use) */
        uint64_t seen = 0;
        if constexpr (!HELD) {
            if (need) seen = __hip_atomic_load((const uint64_t*)(g.pages + page), __ATOMIC_RELAXED, BAM_AGENT);
            if (ballot(need && ((uint32_t)seen >> (CNT_SHIFT + 1)) != V_NB)) return false;
            slot = need ? (uint32_t)(seen >> 32) & BAM_SLOT_MASK : 0u;
            n_access += need ? 1u : 0u;
            n_hit += need ? 1u : 0u;
        }
        [[maybe_unused]] range_view<uint64_t> view;
        bool all = true;                                                          /* the chunk's pages are held (or read without a reference) */
        if constexpr (HELD) {
            view.load(g.r);
            bool left = need;
            while (ballot(left)) {
                const bool in = view.template acquire_some<true>(page, left, slot);
                if (!ballot(in)) { gone = true; break; }
                all = !ballot(need && !in);                                       /* at the first go */
                if (all) break;
                if (in) bam_release_refs(g.pages + page, 1, false);
                left = left && !in;
            }
            n_access += view.n_access;                                            /* a page of the chunk is one access, however often it is asked for */
            n_hit += view.n_hit;
            if (!all && !gone) {
                const bool in = view.template acquire_some<true>(page, need, slot);
                all = !ballot(need && !in);
                if (in && !all) bam_release_refs(g.pages + page, 1, false);
            }
            view.n_access = view.n_hit = 0;
            if (gone) return true;
            if (!all) slot = 0;
        }
        const uint32_t n_blocks = T < 32 ? 32u >> g.tokens_log : 1u, step_blocks = (1u << n_blocks) - 1u;        /* of a step */
        for (uint32_t t_step = t_first; t_step < t_end; t_step += 32u * HALVES) {
            u32x4 k0[HALVES * KP], k1[HALVES * KP], vv[HALVES * VP];
            /* what lies past a row's end is not loaded: its place takes the row's beginning, zero among the keys, of no row among the values */
            const uint8_t *k_at[HALVES * KP], *v_at[HALVES * VP];
            [[maybe_unused]] float k_by[HALVES][2];
            [[maybe_unused]] uint64_t v_by[HALVES];
            /* this lane's tokens as a row of K (8 (row / 4) + row % 4, and 4 further on) and as its part of V (8 grp .. + 7) lie in one block each */
            uint32_t kbs[HALVES], vbs[HALVES], vts[HALVES];
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                /* where the run ends with one step the other is a second look at it, which counts for nothing */
                const uint32_t t0 = t_step + 32u * h < t_end ? t_step + 32u * h : t_step;
                const uint32_t kt = T < 16 ? t0 + 8u * (row >> 2) : t0 + 16u * (row >> 3), vt = t0 + 8u * grp;
                const uint32_t kb = (kt >> g.tokens_log) - b_first, vb = (vt >> g.tokens_log) - b_first;
                kbs[h] = kb; vbs[h] = vb; vts[h] = vt;
                const uint8_t* kp = g.base + ((uint64_t)bam::shfl(slot, kb) << g.page_log) + ((kt & (T - 1u)) + (T < 16 ? row & 3u : row & 7u)) * 16u;
                if constexpr (E8) {
                    const uint8_t* vp = g.base + ((uint64_t)bam::shfl(slot, 32u + vb) << g.page_log) + ((vt & (T - 1u)) >> 3) * (D / 2u) * 16u;
#pragma unroll
                    for (uint32_t j = 0; j < KP; j++) k_at[h * KP + j] = kp + ((4u * j + grp) * 16u < D ? (4u * j + grp) * T * 16u : 0u);
#pragma unroll
                    for (uint32_t i = 0; i < VP; i++) v_at[h * VP + i] = vp + (32u * i + 2u * row < D ? (16u * i + row) * 16u : 0u);
                    /* the powers of two of the tokens of the lane's rows of K (places row and row + 8 of sixteen), and of its part of V */
                    const uint8_t* const kw = g.scales + (uint64_t)bam::shfl(powers_at, kb) * T + (kt & (T - 1u)) + ((row & 4u) << 1 | (row & 3u));
                    k_by[h][0] = scale_of(kw[0]);
                    k_by[h][1] = scale_of(kw[4]);
                    v_by[h] = *(const uint64_t*)(g.scales + (uint64_t)bam::shfl(powers_at, 32u + vb) * T + (vt & (T - 1u)));
                } else {
                    const uint8_t* vp = g.base + ((uint64_t)bam::shfl(slot, 32u + vb) << g.page_log) + (((vt & (T - 1u)) >> 3) * D + row) * 16u;
#pragma unroll
                    for (uint32_t j = 0; j < KP; j++) k_at[j] = kp + ((4u * j + grp) * 8u < D ? (4u * j + grp) * T * 16u : 0u);
#pragma unroll
                    for (uint32_t i = 0; i < VP; i++) v_at[i] = 16u * i < D ? vp + i * 256u : vp;
                }
            }
            /* keys (part 0) or values (part 32) of a step, page by page: `load` for the lanes whose block came, which is `mine` for this lane */
            auto by_page = [&](const uint32_t t0, const uint32_t part, const uint32_t mine, auto&& load) {
                bool left = need && (lane & 32u) == part && (lane & 31u) - ((t0 >> g.tokens_log) - b_first) < n_blocks;
                while (ballot(left)) {
                    uint32_t at = 0;
                    const bool in = view.template acquire_some<true>(page, left, at);
                    const uint32_t came = (uint32_t)(ballot(in) >> part);
                    if (!came) { gone = true; break; }
                    const uint64_t by = (uint64_t)bam::shfl(at, part + mine) << g.page_log;
                    if ((came >> mine) & 1u) load(by);
                    if (in) bam_release_refs(g.pages + page, 1, false);          /* waits for what was loaded */
                    left = left && !in;
                }
                view.n_access = view.n_hit = 0;
            };
            if (HELD && !all) {
#pragma unroll
                for (int j = 0; j < HALVES * KP; j++) k0[j] = k1[j] = u32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < HALVES * VP; i++) vv[i] = u32x4{0, 0, 0, 0};
#pragma unroll
                for (int h = 0; h < HALVES; h++) {
                    if (h && t_step + 32u * h >= t_end) break;
                    by_page(t_step + 32u * h, 0, kbs[h], [&](const uint64_t by) {
#pragma unroll
                        for (int j = h * KP; j < (h + 1) * KP; j++) { k0[j] = ld_payload((const u32x4*)(k_at[j] + by)); k1[j] = ld_payload((const u32x4*)(k_at[j] + by + (T < 16 ? 64 : 128))); }
                    });
                    if (gone) return true;
                }
            } else if constexpr (DP <= 128 || E8) {
                if (!E8 && T < 16) load_step<64>(k_at, v_at, k0, k1, vv); else load_step<128>(k_at, v_at, k0, k1, vv);
            } else {
                if (T < 16) load_keys<64>(k_at, k0, k1); else load_keys<128>(k_at, k0, k1);
            }
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
            const uint32_t t0 = t_step + 32u * h, vb = vbs[h], vt = vts[h];
            if (h && t0 >= t_end) break;
            if (D < DP) {
#pragma unroll
                for (uint32_t j = 0; j < KP; j++) { const bool in = (4u * j + grp) * (E8 ? 16u : 8u) < D; k0[h * KP + j] = in ? k0[h * KP + j] : u32x4{0, 0, 0, 0}; k1[h * KP + j] = in ? k1[h * KP + j] : u32x4{0, 0, 0, 0}; }
            }
            const bool whole = !((holes >> ((t0 >> g.tokens_log) - b_first)) & step_blocks) && (int64_t)t0 + 31 <= sp.first_pos && (!a.window || (int64_t)sp.last_pos - t0 < a.window || t0 + 32u <= a.sinks);
            f32x4 s0[NT], s1[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                s0[n] = s1[n] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < DP / 32; j++) {
                    if constexpr (E8) {
                        const u32x4 x = k0[h * KP + j / 2], y = k1[h * KP + j / 2];
                        s0[n] = mma<F16>(j & 1 ? keys_of<F16>(x[2], x[3], k_by[h][0]) : keys_of<F16>(x[0], x[1], k_by[h][0]), q[n][j], s0[n]);
                        s1[n] = mma<F16>(j & 1 ? keys_of<F16>(y[2], y[3], k_by[h][1]) : keys_of<F16>(y[0], y[1], k_by[h][1]), q[n][j], s1[n]);
                    } else { s0[n] = mma<F16>(k0[j], q[n][j], s0[n]); s1[n] = mma<F16>(k1[j], q[n][j], s1[n]); }
                }
            }
            if (HELD && !all) {
                by_page(t0, 32, vb, [&](const uint64_t by) {
#pragma unroll
                    for (int i = h * VP; i < (h + 1) * VP; i++) vv[i] = ld_payload((const u32x4*)(v_at[i] + by));
                });
                if (gone) return true;
            } else if constexpr (DP > 128 && !E8) {         /* wide heads: the values behind the scores, for which they would not leave registers */
#pragma unroll
                for (int part = 0; part < 2; part++) {
                    const uint8_t* at[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) at[i] = v_at[8 * part + i];
                    load_pieces(at, vv + 8 * part);
                }
            }
            const bool hole = (holes >> vb) & 1u;
            bool slow = false;
            if (!whole) {
                /* values of tokens that no row sees may be anything: none of it may meet the zeros of P */
                const uint32_t any = hole ? 0u : seen_of_eight((int32_t)vt, sp.last_pos, low_of(a, sp.first_pos), (int32_t)a.sinks);
#pragma unroll
                for (int i = h * VP; i < (h + 1) * VP; i++) vv[i] = only(vv[i], any);      /* (in 8 bits: the numbers of a token are 16 bits here too) */
                if constexpr (E8) {                      /* and powers of two that may be anything are 2^0 */
#pragma unroll
                    for (int e = 0; e < 8; e++) v_by[h] = (any >> e) & 1u ? v_by[h] : (v_by[h] & ~(0xffull << (8 * e))) | 127ull << (8 * e);
                }
                if (sp.first_pos != sp.last_pos) {
                    bool odd = false;
#pragma unroll
                    for (int i = h * VP; i < (h + 1) * VP; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) odd |= E8 ? odd8(vv[i][e]) : odd16<F16>(vv[i][e]);
                    slow = ballot(odd) != 0;
                    if (!HELD && slow) return false;             /* row by row, in the launch that holds its pages: the sums of this one stay where they are */
                }
            }
            /* the values as operands: in 8 bits with each token's power of two */
            u32x4 w[DP / 16];
            if constexpr (E8) {
                float by[8];
#pragma unroll
                for (int e = 0; e < 8; e++) by[e] = scale_of((uint32_t)(v_by[h] >> (8 * e)) & 0xffu);
#pragma unroll
                for (int i = 0; i < VP; i++) values_of<F16>(vv[h * VP + i], by, w[2 * i], w[2 * i + 1]);
            } else {
#pragma unroll
                for (int i = 0; i < DP / 16; i++) w[i] = vv[i];
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 4; e++) { x[e] = s0[n][e] * a.scale; x[4 + e] = s1[n][e] * a.scale; }
                uint32_t sees = 0xffu;
                if (!whole) {
                    sees = hole ? 0u : seen_of_eight((int32_t)vt, pos[n], low_of(a, pos[n]), (int32_t)a.sinks);
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++) x[e] = (sees >> e) & 1u ? x[e] : -INFINITY;
                }
                float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                top = fmaxf(max_of_four(top), m[n]);
                const float use = top == -INFINITY ? 0.0f : top;
                if (ballot(top != m[n])) {
                    const float by = __builtin_amdgcn_exp2f(m[n] - use);
                    l[n] *= by;
#pragma unroll
                    for (int i = 0; i < DP / 16; i++) o[n][i] *= by;
                    m[n] = top;
                }
                float sum = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) { x[e] = __builtin_amdgcn_exp2f(x[e] - use + WEIGHT_SHIFT<F16>); sum += x[e]; }
                l[n] += sum;
                u32x4 p;
#pragma unroll
                for (int e = 0; e < 4; e++) p[e] = to16<F16>(x[2 * e], x[2 * e + 1]);
                if (!HELD || !slow) {
#pragma unroll
                    for (int i = 0; i < DP / 16; i++) o[n][i] = mma<F16>(w[i], p, o[n][i]);
                } else {
                    /* an infinity or NaN among the values of tokens that some rows see and others do not: row by row, what the row does not see as zero */
                    for (uint32_t c = 0; c < 16; c++) {
                        const uint32_t sc = bam::shfl(sees, (lane & 48u) + c);
#pragma unroll
                        for (int i = 0; i < DP / 16; i++) {
                            const f32x4 with = mma<F16>(only(w[i], sc), p, o[n][i]);
                            if (row == c) o[n][i] = with;
                        }
                    }
                }
            }
            }
        }
        fence_meta();                                            /* what was read is here */
        if constexpr (!HELD) {
            uint64_t now = seen;
            if (need) now = __hip_atomic_load((const uint64_t*)(g.pages + page), __ATOMIC_RELAXED, BAM_AGENT);
            if (ballot(need && ((seen ^ now) & 0xFFFFFFFFC0000000ull) != 0)) return false;
        } else if (need && all) bam_release_refs(g.pages + page, 1, false);
        v += (t_end - t_first) / 32u;
    }
    return true;
}

/*
 * kv_steps without references for pages of 8 bits and 32 tokens and more, where a step lies in one block: the next step's pieces are on their way while one is worked on.  128 sequences of up to
 * 8192 tokens, 64 heads on 8 of 128 numbers: 270 us, 6.0 TB/s, for 277; 24 of up to 9000, 32 heads, 80 for 87.  Loads are of the compiler's
 * making here (buffer loads of a page, past the vector L1 and not to be kept, like the others), which waits for those of the step that it needs; what lies past a row's end among
 * the keys is past the end of the buffer, and zero.
 */
template <int DP, int F16, int NT>
__device__ __forceinline__ bool kv_steps_ahead(const kv_geom& g, const kv_seqs& s, const kv_att& a, const kv_span& sp, const uint32_t seq, const uint32_t head, const uint32_t v0, const uint32_t v1,
                                               const u32x4 (&q)[NT][DP / 32], const int32_t (&pos)[NT], f32x4 (&o)[NT][DP / 16], float (&m)[NT], float (&l)[NT], uint32_t& n_access, uint32_t& n_hit)
{
    using namespace bam;
    constexpr int KP = DP / 64, VP = DP / 32;
    const uint32_t lane = bam::lane(), row = lane & 15u, grp = lane >> 4, T = g.tokens, D = g.dim;
    struct step_t { u32x4 k0[KP], k1[KP], v[VP]; uint32_t by0, by1; uint64_t by; };
    const uint32_t k_lane = (grp * T + 16u * (row >> 3) + (row & 7u)) * 16u, k_token = 16u * (row >> 3) + ((row & 4u) << 1 | (row & 3u));
    uint32_t v_lane[VP];
#pragma unroll
    for (uint32_t i = 0; i < VP; i++) v_lane[i] = grp * (D / 2u) * 16u + (32u * i + 2u * row < D ? (16u * i + row) * 16u : 0u);
    for (uint32_t v = v0; v < v1;) {
        const bool front = v < sp.front;
        const uint32_t t_first = front ? v * 32u : sp.base + (v - sp.front) * 32u;
        const uint32_t run = (front && sp.front < v1 ? sp.front : v1) - v, b_first = t_first >> g.tokens_log;
        uint32_t t_end = (b_first + 32u) << g.tokens_log;
        if (t_first + run * 32u < t_end) t_end = t_first + run * 32u;
        const uint32_t t_seen = t_end < sp.len ? t_end : sp.len;
        const uint32_t blk = b_first + (lane & 31u);
        uint64_t page = 0, seen = 0;
        const bool in_run = (blk << g.tokens_log) < t_end, asked = in_run && (blk << g.tokens_log) < t_seen;
        const bool need = asked && page_of_block(g, s, seq, blk, head, page);
        if (lane >= 32) page += 1;
        const uint32_t holes = (uint32_t)ballot((asked && !need) || (in_run && blk >= s.width));
        if (need) seen = __hip_atomic_load((const uint64_t*)(g.pages + page), __ATOMIC_RELAXED, BAM_AGENT);
        if (ballot(need && ((uint32_t)seen >> (CNT_SHIFT + 1)) != V_NB)) return false;
        const uint32_t slot = need ? (uint32_t)(seen >> 32) & BAM_SLOT_MASK : 0u;
        const uint64_t powers_at = need ? page - g.first_page : 0u;
        n_access += need ? 1u : 0u;
        n_hit += need ? 1u : 0u;
        auto load = [&](step_t& x, const uint32_t t0) {
            const uint32_t b = (t0 >> g.tokens_log) - b_first, in = t0 & (T - 1u);
            const __amdgpu_buffer_rsrc_t k_at = __builtin_amdgcn_make_buffer_rsrc(g.base + ((uint64_t)bcast(slot, b) << g.page_log), 0, (int)(D * T), 0x00027000);
            const __amdgpu_buffer_rsrc_t v_at = __builtin_amdgcn_make_buffer_rsrc(g.base + ((uint64_t)bcast(slot, 32u + b) << g.page_log), 0, (int)(D * T), 0x00027000);
            const __amdgpu_buffer_rsrc_t by = __builtin_amdgcn_make_buffer_rsrc(g.scales + bcast(powers_at, b) * T, 0, (int)(2u * T), 0x00027000);
#pragma unroll
            for (uint32_t j = 0; j < KP; j++) {
                x.k0[j] = __builtin_amdgcn_raw_buffer_load_b128(k_at, k_lane, (4u * j * T + in) * 16u, 18);
                x.k1[j] = __builtin_amdgcn_raw_buffer_load_b128(k_at, k_lane + 128u, (4u * j * T + in) * 16u, 18);
            }
#pragma unroll
            for (uint32_t i = 0; i < VP; i++) x.v[i] = __builtin_amdgcn_raw_buffer_load_b128(v_at, v_lane[i], (in >> 3) * (D / 2u) * 16u, 18);
            x.by0 = __builtin_amdgcn_raw_buffer_load_b8(by, k_token, in, 0);
            x.by1 = __builtin_amdgcn_raw_buffer_load_b8(by, k_token + 4u, in, 0);
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            const u32x2 y = __builtin_amdgcn_raw_buffer_load_b64(by, 8u * grp, T + in, 0);
            x.by = (uint64_t)y[1] << 32 | y[0];
        };
        /* false: an infinity or NaN among values that some rows see and others do not */
        auto work = [&](step_t& x, const uint32_t t0) {
            const uint32_t b = (t0 >> g.tokens_log) - b_first;
            const int32_t vt = (int32_t)(t0 + 8u * grp);
            const bool hole = (holes >> b) & 1u;
            const bool whole = !hole && (int64_t)t0 + 31 <= sp.first_pos && (!a.window || (int64_t)sp.last_pos - t0 < a.window || t0 + 32u <= a.sinks);
            const float by0 = scale_of(x.by0), by1 = scale_of(x.by1);
            f32x4 s0[NT], s1[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) s0[n] = s1[n] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < DP / 32; j++) {
                const u32x4 y0 = x.k0[j / 2], y1 = x.k1[j / 2];
                const u32x4 k0 = j & 1 ? keys_of<F16>(y0[2], y0[3], by0) : keys_of<F16>(y0[0], y0[1], by0), k1 = j & 1 ? keys_of<F16>(y1[2], y1[3], by1) : keys_of<F16>(y1[0], y1[1], by1);
#pragma unroll
                for (int n = 0; n < NT; n++) { s0[n] = mma<F16>(k0, q[n][j], s0[n]); s1[n] = mma<F16>(k1, q[n][j], s1[n]); }
            }
            if (!whole) {
                const uint32_t any = hole ? 0u : seen_of_eight(vt, sp.last_pos, low_of(a, sp.first_pos), (int32_t)a.sinks);
#pragma unroll
                for (int i = 0; i < VP; i++) x.v[i] = only(x.v[i], any);
#pragma unroll
                for (int e = 0; e < 8; e++) x.by = (any >> e) & 1u ? x.by : (x.by & ~(0xffull << (8 * e))) | 127ull << (8 * e);
                if (sp.first_pos != sp.last_pos) {
                    bool odd = false;
#pragma unroll
                    for (int i = 0; i < VP; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) odd |= odd8(x.v[i][e]);
                    if (ballot(odd)) return false;
                }
            }
            u32x4 p[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 4; e++) { y[e] = s0[n][e] * a.scale; y[4 + e] = s1[n][e] * a.scale; }
                if (!whole) {
                    const uint32_t sees = hole ? 0u : seen_of_eight(vt, pos[n], low_of(a, pos[n]), (int32_t)a.sinks);
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++) y[e] = (sees >> e) & 1u ? y[e] : -INFINITY;
                }
                float top = fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
                top = fmaxf(max_of_four(top), m[n]);
                const float use = top == -INFINITY ? 0.0f : top;
                if (ballot(top != m[n])) {
                    const float less = __builtin_amdgcn_exp2f(m[n] - use);
                    l[n] *= less;
#pragma unroll
                    for (int i = 0; i < DP / 16; i++) o[n][i] *= less;
                    m[n] = top;
                }
                float sum = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) { y[e] = __builtin_amdgcn_exp2f(y[e] - use + WEIGHT_SHIFT<F16>); sum += y[e]; }
                l[n] += sum;
#pragma unroll
                for (int e = 0; e < 4; e++) p[n][e] = to16<F16>(y[2 * e], y[2 * e + 1]);
            }
            float by[8];
#pragma unroll
            for (int e = 0; e < 8; e++) by[e] = scale_of((uint32_t)(x.by >> (8 * e)) & 0xffu);
#pragma unroll
            for (int i = 0; i < VP; i++) {
                u32x4 w0, w1;
                values_of<F16>(x.v[i], by, w0, w1);
#pragma unroll
                for (int n = 0; n < NT; n++) { o[n][2 * i] = mma<F16>(w0, p[n], o[n][2 * i]); o[n][2 * i + 1] = mma<F16>(w1, p[n], o[n][2 * i + 1]); }
            }
            return true;
        };
        step_t x, y;
        load(x, t_first);
        uint32_t t = t_first;
        for (; t + 64u < t_end; t += 64u) {
            load(y, t + 32u);
            if (!work(x, t)) return false;
            load(x, t + 64u);
            if (!work(y, t + 32u)) return false;
        }
        const bool two = t + 32u < t_end;
        if (two) load(y, t + 32u);
        if (!work(x, t)) return false;
        if (two && !work(y, t + 32u)) return false;
        fence_meta();                            /* what was read is here */
        uint64_t now = seen;
        if (need) now = __hip_atomic_load((const uint64_t*)(g.pages + page), __ATOMIC_RELAXED, BAM_AGENT);
        if (ballot(need && ((seen ^ now) & 0xFFFFFFFFC0000000ull) != 0)) return false;
        v += (t_end - t_first) / 32u;
    }
    return true;
}

/* rows of an item: a head of keys, a tile of the rows (new token, head of queries) of a sequence */
struct kv_item { uint32_t seq, head, tile, r0, r1; int32_t pos0, start; };      /* pos0: position of row `start` */
__device__ __forceinline__ bool item_of(const kv_geom& g, const kv_seqs& s, const kv_att& a, const uint32_t item, kv_item& it)
{
    const uint32_t tile_rows = a.tile_rows;
    it.head = item % g.heads;
    it.tile = item / g.heads % a.tiles;
    it.seq = item / g.heads / a.tiles;
    it.start = s.starts ? s.starts[it.seq] : (int32_t)it.seq;
    const int32_t end = s.starts ? s.starts[it.seq + 1] : (int32_t)it.seq + 1;
    if (it.start < 0) it.start = 0;
    /* positions count from the end that `starts` says, rows end where the rows do */
    const int32_t last = end < (int32_t)s.rows ? end : (int32_t)s.rows;
    if (last <= it.start) return false;
    int32_t len = s.lens[it.seq];
    if (len < 0) len = 0;
    it.pos0 = len - (end - it.start);
    const uint32_t all = ((uint32_t)(last - it.start) < a.max_new ? (uint32_t)(last - it.start) : a.max_new) * a.group;
    if (it.tile * (uint64_t)tile_rows >= all) return false;
    it.r0 = it.tile * tile_rows;
    it.r1 = it.r0 + tile_rows < all ? it.r0 + tile_rows : all;
    return true;
}

/*
 * The steps of a split.  In 16 bits as many as were announced for each, and the last takes what is beyond that.  In 8 bits a sequence's own steps are shared out: of sequences of different lengths, or with
 * a table much wider than they are, the splits behind the shorter ones' ends would have nothing.  One token each of 8 sequences of 8000 to 16000 tokens 51 and 46 us.
 */
template <int E8> __device__ __forceinline__ void steps_of(const kv_att& a, const kv_span& sp, const uint32_t split, uint32_t& v0, uint32_t& v1)
{
    const uint32_t each = E8 ? ((sp.n_steps + a.splits - 1u) / a.splits + 3u) & ~3u : a.steps;
    v0 = split * each;
    v1 = v0 + each;
    if (v1 > sp.n_steps || split + 1 == a.splits) v1 = sp.n_steps;
    if (v0 > v1) v0 = v1;
}

/* a workgroup's split of an item, of its rows from s0 on: its four waves a quarter of the steps each, joined over LDS; the sums to their rows where there is one split, else to a.part */
template <int DP, int F16, int E8, int NT, bool HELD>
__device__ __forceinline__ bool kv_split(const kv_geom& g, const kv_seqs& s, const kv_att& a, const uint32_t item, const kv_item& it, const uint32_t s0, const uint32_t split, float* lds, bool& gone)
{
    using namespace bam;
    constexpr uint32_t R = 16 * NT;
    const uint32_t lane = bam::lane(), wave = first(threadIdx.x / 64u), row = lane & 15u, grp = lane >> 4, D = g.dim;
    const uint32_t s1 = s0 + R < it.r1 ? s0 + R : it.r1;
    kv_span sp = span_of(a, s.width << g.tokens_log, it.pos0, it.r0, it.r1);                     /* the item's splits, */
    sp.first_pos = it.pos0 + (int32_t)(s0 / a.group);                           /* as these rows see them */
    sp.last_pos = it.pos0 + (int32_t)((s1 - 1) / a.group);
    uint32_t v0, v1;
    steps_of<E8>(a, sp, split, v0, v1);
    const uint32_t each = (v1 - v0 + 3u) / 4u;
    uint32_t w0 = v0 + wave * each, w1 = w0 + each;
    if (w0 > v1) w0 = v1;
    if (w1 > v1) w1 = v1;
    u32x4 q[NT][DP / 32];
    int32_t pos[NT];
    f32x4 o[NT][DP / 16];
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const uint32_t r = s0 + n * 16u + row;
        const bool has = r < s1;
        const uint32_t tok = has ? r / a.group : 0u, h = it.head * a.group + (has ? r % a.group : 0u);
        pos[n] = has ? it.pos0 + (int32_t)tok : -1;
        const uint16_t* const from = a.q + (int64_t)(it.start + (int32_t)tok) * a.q_row + (int64_t)h * a.q_head;
#pragma unroll
        for (int j = 0; j < DP / 32; j++) {
            q[n][j] = u32x4{0, 0, 0, 0};
            /* the eight numbers of the lane's operand of keys: in 8 bits, two products share a piece of sixteen */
            const uint32_t c = E8 ? (4u * (j / 2) + grp) * 16u + (j & 1) * 8u : (4u * j + grp) * 8u;
            if (has && c < D) q[n][j] = a.aligned ? load_piece<true>(from + c) : load_piece<false>(from + c);
        }
        m[n] = -INFINITY;
        l[n] = 0;
#pragma unroll
        for (int i = 0; i < DP / 16; i++) o[n][i] = f32x4{0, 0, 0, 0};
    }
    uint32_t n_access = 0, n_hit = 0;
    bool ok;
    if (E8 && !HELD && DP <= 128 && g.tokens >= 32) {
        if constexpr (E8 && !HELD && DP <= 128) ok = kv_steps_ahead<DP, F16, NT>(g, s, a, sp, it.seq, it.head, w0, w1, q, pos, o, m, l, n_access, n_hit);
    } else ok = kv_steps<DP, F16, E8, NT, HELD>(g, s, a, sp, it.seq, it.head, w0, w1, q, pos, o, m, l, gone, n_access, n_hit);
    /* [4][R] maxima, [4][R] denominators, [R][DP] sums */
    float *const ms = lds, *const ls = lds + 4 * R, *const os = lds + 8 * R;
    uint32_t* const flag = (uint32_t*)(lds + 8 * R + R * DP);
#pragma unroll
    for (int n = 0; n < NT; n++) {
        l[n] = sum_of_four(l[n]);
        if (grp == 0) { ms[wave * R + n * 16u + row] = m[n]; ls[wave * R + n * 16u + row] = l[n]; }
    }
    if (threadIdx.x == 0) *flag = 0;
    __syncthreads();
    if ((!ok || gone) && lane == 0) __hip_atomic_fetch_or(flag, (ok ? 0u : 1u) | (gone ? 2u : 0u), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    float by[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const uint32_t r = n * 16u + row;
        const float top = fmaxf(fmaxf(ms[r], ms[R + r]), fmaxf(ms[2 * R + r], ms[3 * R + r]));
        by[n] = __builtin_amdgcn_exp2f(m[n] - (top == -INFINITY ? 0.0f : top) - WEIGHT_SHIFT<F16>);          /* and out of the sums again */
    }
    /* a quarter of the columns each, by turns: the order in which a column's four parts are added does not depend on who comes first */
    constexpr int QUARTER = DP / 64;
#pragma unroll 1
    for (uint32_t turn = 0; turn < 4; turn++) {
        const uint32_t part = (wave + turn) & 3u;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < DP / 16; i++) {
                if ((uint32_t)(i / QUARTER) != part) continue;
                f32x4* const at = (f32x4*)(os + (n * 16u + row) * DP + i * 16 + grp * 4);
                const f32x4 x = o[n][i] * by[n];
                *at = turn ? *at + x : x;
            }
        __syncthreads();
    }
    const uint32_t bad = *flag;
    gone = (bad & 2u) != 0;
    if (!HELD && (bad & 1u)) return false;              /* nothing of it counts: who does it again counts */
    count_accesses(g, n_access, n_hit);
    const uint32_t n_rows = s1 - s0;
    for (uint32_t x = threadIdx.x; x < n_rows * (DP / 8u); x += 256u) {
        const uint32_t r = x / (DP / 8u), c = x % (DP / 8u) * 8u;
        if (c >= D) continue;
        const float top = fmaxf(fmaxf(ms[r], ms[R + r]), fmaxf(ms[2 * R + r], ms[3 * R + r])), use = top == -INFINITY ? 0.0f : top;
        float den = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) den += ls[w * R + r] * __builtin_amdgcn_exp2f(ms[w * R + r] - use - WEIGHT_SHIFT<F16>);
        if (gone) den = __builtin_nanf("");
        f32x4 lo, hi;
        if constexpr (E8) {                              /* rows 16 i + 2 r and 16 i + 2 r + 1 of O^T are row r of two products */
            const f32x4 x = *(const f32x4*)(os + r * DP + c / 32u * 32u + c % 32u / 2u), y = *(const f32x4*)(os + r * DP + c / 32u * 32u + 16u + c % 32u / 2u);
            lo = f32x4{x[0], y[0], x[1], y[1]};
            hi = f32x4{x[2], y[2], x[3], y[3]};
        } else { lo = *(const f32x4*)(os + r * DP + c); hi = *(const f32x4*)(os + r * DP + c + 4); }
        if (a.splits > 1) {
            const uint64_t at = ((uint64_t)item * a.tile_rows + (s0 - it.r0) + r) * a.splits + split;
            *(f32x4*)(a.part + at * D + c) = lo;
            *(f32x4*)(a.part + at * D + c + 4) = hi;
            if (c == 0) { a.part_m[at] = top; a.part_l[at] = den; }
        } else {
            /* a row that sees no token is zero */
            const float inv = top == -INFINITY && !gone ? 0.0f : 1.0f / den;
            const uint32_t rr = s0 + r, tok = (uint32_t)it.start + rr / a.group, h = it.head * a.group + rr % a.group;
            const u32x4 y = {to16<F16>(lo[0] * inv, lo[1] * inv), to16<F16>(lo[2] * inv, lo[3] * inv), to16<F16>(hi[0] * inv, hi[1] * inv), to16<F16>(hi[2] * inv, hi[3] * inv)};
            *(u32x4*)(a.out + ((uint64_t)tok * a.q_heads + h) * D + c) = y;
            if (a.lse && c == 0) a.lse[(uint64_t)tok * a.q_heads + h] = (top + __builtin_amdgcn_logf(den)) * 0.6931471805599453f;
        }
    }
    return true;
}
template <int DP, int NT> constexpr uint32_t split_lds() { return (8 * 16 * NT + 16 * NT * DP + 4) * 4; }

template <int DP, int F16, int E8, int NT>
__global__ __launch_bounds__(256) void k_kv_attend(const kv_geom g, const kv_seqs s, const kv_att a)
{
    extern __shared__ float lds[];
    const uint32_t item = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    kv_item it;
    bool gone = false, ok = true;
    if (item_of(g, s, a, item, it)) ok = kv_split<DP, F16, E8, NT, false>(g, s, a, item, it, it.r0, split, lds, gone);
    if (threadIdx.x == 0) a.left[blockIdx.x] = ok ? 0 : 1;
}

// ---- many rows: tiles of rows against tiles of tokens in LDS ----
/* 16 bytes a lane from memory to LDS, from base + at to lds + 16 x lane, past the vector L1 as all payload is (ld_payload); counted by the wave's memory counter, and by nobody else: wait for all of them before a barrier.
 * (m0 is one of the compiler's reserved registers: it keeps nothing there, and warns of a clobber list that names it.) */
__device__ __forceinline__ void to_lds(const uint8_t* base, const uint32_t at, const uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 sc1" :: "s"(lds), "v"(at), "s"(base) : "memory");
}
template <int F16> __device__ __forceinline__ f32x16 mma32(const u32x4 a, const u32x4 b, const f32x16 c)
{
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int DP> constexpr uint32_t tile_tokens() { return DP > 128 ? 32 : 64; }
template <int DP> constexpr uint32_t tile_lds() { return 2 * 2 * tile_tokens<DP>() * DP * 2; }

/*
 * NW waves of 32 rows each, all against the same tokens, KT at a time, which the waves bring into LDS together while they work on the tile before (two
 * buffers, one barrier to a tile).  Pages lie in LDS as they lie in the cache, piece by piece.  Lane l: row l % 32 of its wave, and of each 16 tokens
 * those 8 (l / 32) .. + 7.  Pages are read without a reference, in chunks of 64 blocks, as in kv_steps (past the L1; an
 * acquire behind each first look instead, which invalidates more than that, cost a tenth, and a quarter where there are 18 tiles to a workgroup).
 *   Bound by the matrix unit and by what its two waves to a SIMD cannot hide: 32 products of 32 cycles and some 200 other instructions, 32 of them exponentials of 16
 * cycles, to a tile and wave.  A document of 16384 tokens, 32 heads on 8 of 128 numbers: 2.12 ms, 1040 TFLOP/s of what is visible (a large product of the library's: 1218).  Rows of 32 to a
 * wave read a tile's 32 KiB of LDS in as many cycles as its products take; eight waves to a workgroup, one to a compute unit, were a tenth slower than two of four.
 */
template <int DP, int F16, int E8, int NW, bool EXACT>
__global__ __launch_bounds__(64 * NW, DP > 128 ? 1 : 2) void k_kv_attend_tiles(const kv_geom g, const kv_seqs s, const kv_att a)
{
    using namespace bam;
    extern __shared__ float lds[];
    constexpr uint32_t KT = tile_tokens<DP>(), HALF = KT * DP * 2, PIECES = KT * DP / 8;      /* bytes and pieces of a tile's keys, and of its values */
    constexpr uint32_t UNITS = KT / 8 / NW;      /* of eight tokens, that a wave brings in: their keys, then their values, as they lie in their pages */
    static_assert(UNITS >= 1, "a unit to a wave");
    const uint32_t lane = bam::lane(), wave = first(threadIdx.x / 64u), row = lane & 31u, half = lane >> 5, D = EXACT ? DP : g.dim, T = g.tokens;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    /* the tiles with the most tokens to look at first */
    const uint32_t per_seq = a.tiles * g.heads, work = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const uint32_t item = work / per_seq * per_seq + (a.tiles - 1u - work % per_seq / g.heads) * g.heads + work % g.heads;
    kv_item it;
    if (!item_of(g, s, a, item, it)) { if (threadIdx.x == 0) a.left[(uint64_t)item * a.splits + split] = 0; return; }
    const kv_span sp = span_of(a, s.width << g.tokens_log, it.pos0, it.r0, it.r1);
    uint32_t v0, v1;
    steps_of<E8>(a, sp, split, v0, v1);
    if (!EXACT) {                                /* what no piece is loaded for is zero */
        for (uint32_t x = threadIdx.x; x < tile_lds<DP>() / 16u; x += 64u * NW) ((u32x4*)lds)[x] = u32x4{0, 0, 0, 0};
        __syncthreads();
    }
    /* this lane's row, and the positions of the wave's rows */
    const uint32_t w0 = it.r0 + wave * 32u, w1 = w0 + 32u < it.r1 ? w0 + 32u : it.r1;
    const bool idle = w0 >= it.r1;
    const uint32_t r = w0 + row;
    const bool has = r < it.r1;
    const uint32_t tok = has ? r / a.group : 0u, head = it.head * a.group + (has ? r % a.group : 0u);
    const int32_t p0 = it.pos0, pos = has ? p0 + (int32_t)tok : -1;
    const int32_t first_pos = idle ? -1 : p0 + (int32_t)(w0 / a.group), last_pos = idle ? -1 : p0 + (int32_t)((w1 - 1) / a.group);
    const int32_t first_of_all = sp.first_pos, last_of_all = sp.last_pos;
    /* a negative scale goes into the sign of the queries: the largest score is then the largest product */
    const float c = fmaxf(fabsf(a.scale), 1e-30f);
    const uint32_t flip = a.scale < 0 ? 0x80008000u : 0u;
    u32x4 q[DP / 16];
    {
        const uint16_t* const from = a.q + (int64_t)(it.start + (int32_t)tok) * a.q_row + (int64_t)head * a.q_head;
#pragma unroll
        for (uint32_t j = 0; j < DP / 16; j++) {
            q[j] = u32x4{0, 0, 0, 0};
            if (has && (2u * j + half) * 8u < D) q[j] = (a.aligned ? load_piece<true>(from + (2u * j + half) * 8u) : load_piece<false>(from + (2u * j + half) * 8u)) ^ flip;
        }
    }
    f32x16 o[DP / 32];
#pragma unroll
    for (uint32_t i = 0; i < DP / 32; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[i][e] = 0;
    float m = -INFINITY, l = 0, l1 = 0;
    bool ok = true;
    uint32_t n_access = 0;

    /*
     * The chunk that tiles are loaded from, a block to a lane, and the blocks of the one after it.  What is loaded here has arrived before the next tile is asked for: the
     * compiler waits for its own loads by waiting for all that are on their way.
     */
    uint32_t b_first = 0, t_next = 0, t_end = 0, k_slot = 0, v_slot = 0, v = v0, nb_first = 0, nt_first = 0, nt_end = 0;
    uint64_t holes = 0, page = 0, k_seen = 0, v_seen = 0;
    int32_t nblock = -1;
    bool need = false, nasked = false, there = false;      /* there: nblock and the like are those of a chunk to come */
    auto next_blocks = [&]() {
        there = v < v1;
        if (!there) return;
        const bool front = v < sp.front;
        nt_first = front ? v * 32u : sp.base + (v - sp.front) * 32u;
        const uint32_t run = (front && sp.front < v1 ? sp.front : v1) - v;
        nb_first = nt_first >> g.tokens_log;
        nt_end = (nb_first + 64u) << g.tokens_log;
        if (nt_first + run * 32u < nt_end) nt_end = nt_first + run * 32u;
        const uint32_t blk = nb_first + lane;
        nasked = (blk << g.tokens_log) < (nt_end < sp.len ? nt_end : sp.len);
        nblock = -1;
        if (nasked && blk < s.width) nblock = s.table[(int64_t)it.seq * s.stride + blk];
        asm volatile("" : "+v"(nblock));
        v += (nt_end - nt_first) / 32u;
    };
    auto look = [&](uint64_t& k, uint64_t& v_) {
        k = v_ = (uint64_t)VALID;
        if (need) {
            k = __hip_atomic_load((const uint64_t*)(g.pages + page), __ATOMIC_RELAXED, BAM_AGENT);
            v_ = __hip_atomic_load((const uint64_t*)(g.pages + page + 1), __ATOMIC_RELAXED, BAM_AGENT);
        }
        asm volatile("" : "+v"(k), "+v"(v_));
    };
    auto look_again = [&]() {
        uint64_t k, v_;
        look(k, v_);
        if (ballot(need && (((k_seen ^ k) | (v_seen ^ v_)) & 0xFFFFFFFFC0000000ull) != 0)) ok = false;
    };
    auto enter_next = [&]() {
        b_first = nb_first; t_next = nt_first; t_end = nt_end;
        need = nblock >= 0 && (uint64_t)nblock < g.n_blocks;
        page = g.first_page + ((uint64_t)(uint32_t)nblock * g.heads + it.head) * 2u;
        holes = ballot(nasked && !need);
        look(k_seen, v_seen);
        if (ballot(((uint32_t)k_seen >> (CNT_SHIFT + 1)) != V_NB || ((uint32_t)v_seen >> (CNT_SHIFT + 1)) != V_NB)) ok = false;
        k_slot = (uint32_t)(k_seen >> 32) & BAM_SLOT_MASK;
        v_slot = (uint32_t)(v_seen >> 32) & BAM_SLOT_MASK;
        n_access += 2u * popc(ballot(need));
        next_blocks();
    };
    /* the tile from t_next on into a buffer */
    uint32_t at_first = 0, at_end = 0, at_block = 0;          /* of the tile that is on its way */
    uint64_t at_holes = 0;
    const uint32_t k_lane0 = (lane & 7u) * 16u + (lane >> 3) * T * 16u, k_lane1 = (lane & 7u) * 16u + (lane >> 3 ^ 1u) * T * 16u;
    /*
     * 8 bits: a set of tokens (two units of one block, or one) at a time, a piece of keys and one of values to a lane and load.  They go to where a part of the 16-bit numbers that they
     * stand for will lie, and are taken from there, and the numbers put there, when the tile before is done with (put_tile): each wave in its own units, so nobody else is waited for, and no registers
     * are held meanwhile (held, they made the queries spill: 500 new tokens after 32500, 610 us, and 310 so, where a 16-bit cache
     * takes 290).  What of a place depends on the lane does not depend on the load; the rest, and the powers
     * of two of the values where a load is of one group of eight tokens, are scalars.
     */
    constexpr uint32_t ST = UNITS > 1 ? 16 : 8, SETS = UNITS * 8 / ST, CPL = 64 / ST, GROUPS = ST / 8, KL = (DP / 16 + CPL - 1) / CPL, GL = (DP / 2 + 63) / 64;      /* CPL: pieces of a token's keys to a load; loads to a set's keys, to a group of eight tokens' values */
    constexpr bool ONE = DP > 64, FULL = EXACT && DP % 64 == 0;      /* ONE: a load is of one group; FULL: all of its lanes have something */
    constexpr uint32_t VL = ONE ? GROUPS * GL : 1;
    [[maybe_unused]] uint32_t k_by[E8 ? SETS : 1];
    [[maybe_unused]] uint64_t v_by[E8 ? SETS * GROUPS : 1];
    auto load_tile = [&](const uint32_t buf) {
        if constexpr (E8) {
            const uint32_t to = lds0 + buf * 2u * HALF + wave * UNITS * DP * 16u;
            uint32_t l_ = lane;                  /* (worked out anew for each tile, not kept) */
            asm volatile("" : "+v"(l_));
            const uint32_t k_place = l_ % ST, k_piece = l_ / ST, v_group = ONE ? 0u : l_ / 32u, v_pair = ONE ? l_ : l_ % 32u;
            const uint32_t k_off = (k_piece * T + k_place) * 16u, v_off = (v_group * (D / 2u) + v_pair) * 16u;
#pragma unroll
            for (uint32_t x = 0; x < SETS; x++) {
                const uint32_t t = t_next + wave * UNITS * 8u + x * ST, b = ((t >> g.tokens_log) - b_first) & 63u, in = t & (T - 1u), unit = to + x * GROUPS * DP * 16u;
                const uint8_t* const k_at = g.base + ((uint64_t)bcast(k_slot, b) << g.page_log) + in * 16u;
                const uint8_t* const v_at = g.base + ((uint64_t)bcast(v_slot, b) << g.page_log) + (in >> 3) * (D / 2u) * 16u;
                const uint64_t by = (uint64_t)(uintptr_t)g.scales + bcast(need ? page - g.first_page : (uint64_t)0, b) * T;
#pragma unroll
                for (uint32_t i = 0; i < KL; i++) if (FULL || (i * CPL + k_piece) * 16u < D) to_lds(k_at, k_off + i * CPL * T * 16u, unit + i * 1024u);
#pragma unroll
                for (uint32_t i = 0; i < VL; i++) {
                    if constexpr (ONE) {
                        if (FULL || ((i % GL) * 64u + v_pair) * 2u < D) to_lds(v_at, v_off + (i / GL * (D / 2u) + (i % GL) * 64u) * 16u, unit + HALF + i / GL * DP * 16u + (i % GL) * 1024u);
                    } else {
#pragma unroll
                        for (uint32_t n = 0; n < 2; n++) if (v_group == n && (FULL || v_pair * 2u < D)) to_lds(v_at, v_off, unit + HALF + n * (DP * 16u - 512u));
                    }
                }
                k_by[x] = ((const uint8_t*)by)[place_in(g, in + k_place)];
                if constexpr (ONE) {
#pragma unroll
                    for (uint32_t n = 0; n < GROUPS; n++) v_by[x * GROUPS + n] = *(const __attribute__((address_space(4))) uint64_t*)(by + T + in + n * 8u);
                } else v_by[x * GROUPS] = *(const uint64_t*)(by + T + in + v_group * 8u);
            }
        } else {
            const uint32_t to = lds0 + buf * 2u * HALF;
#pragma unroll
            for (uint32_t x = 0; x < UNITS; x++) {
                const uint32_t u = wave * UNITS + x, t = t_next + 8u * u, b = ((t >> g.tokens_log) - b_first) & 63u, in = t & (T - 1u);
                const uint8_t* const k_at = g.base + ((uint64_t)bcast(k_slot, b) << g.page_log) + in * 16u;
                const uint8_t* const v_at = g.base + ((uint64_t)bcast(v_slot, b) << g.page_log) + (in >> 3) * D * 16u;
#pragma unroll
                for (uint32_t i = 0; i < DP / 64; i++) {
                    /* odd units with neighbouring pieces exchanged: read by sixteen lanes from two units, they lie in different banks */
                    const uint32_t odd = UNITS % 2 ? u & 1u : x & 1u;
                    if (EXACT || (8u * i + (lane >> 3 ^ odd)) * 8u < D) to_lds(k_at, (odd ? k_lane1 : k_lane0) + i * 128u * T, to + u * DP * 16u + i * 1024u);
                    if (EXACT || 64u * i + lane < D) to_lds(v_at, (64u * i + lane) * 16u, to + HALF + u * DP * 16u + i * 1024u);
                }
            }
        }
        at_first = t_next; at_end = t_end < sp.len ? t_end : sp.len; at_holes = holes; at_block = b_first;          /* (the last step may go on behind the table's end) */
        t_next += KT;
    };
    [[maybe_unused]] auto put_tile = [&](const uint32_t buf) {
        uint8_t* const to = (uint8_t*)lds + buf * 2u * HALF + wave * UNITS * DP * 16u;
        fence_meta();                            /* the wave's loads are in LDS */
        uint32_t l_ = lane;
        asm volatile("" : "+v"(l_));
        const uint32_t k_place = l_ % ST, k_piece = l_ / ST, v_group = ONE ? 0u : l_ / 32u, v_pair = ONE ? l_ : l_ % 32u;
#pragma unroll
        for (uint32_t x = 0; x < SETS; x++) {
            uint8_t* const unit = to + x * GROUPS * DP * 16u;
            /* (what nothing was loaded for is not used) */
            u32x4 k_raw[KL], v_raw[VL];
#pragma unroll
            for (uint32_t i = 0; i < KL; i++) k_raw[i] = *(const u32x4*)(unit + i * 1024u + l_ * 16u);
#pragma unroll
            for (uint32_t i = 0; i < VL; i++) v_raw[i] = *(const u32x4*)(unit + HALF + (ONE ? i / GL * DP * 16u + (i % GL) * 1024u + l_ * 16u : v_group * DP * 16u + v_pair * 16u));
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      /* all lanes have theirs before one writes */
            const uint32_t odd = (wave * UNITS + (k_place >> 3)) & 1u;
            const float by = scale_of(k_by[x]);
            uint8_t* const k_to = unit + (k_place >> 3) * DP * 16u + (k_place & 7u) * 16u + k_piece * 256u;
            uint8_t* const v_to = unit + HALF + v_group * DP * 16u + v_pair * 32u;
#pragma unroll
            for (uint32_t i = 0; i < KL; i++)
                if (FULL || (i * CPL + k_piece) * 16u < D) {
                    *(u32x4*)(k_to + i * CPL * 256u + odd * 128u) = keys_of<F16>(k_raw[i][0], k_raw[i][1], by);
                    *(u32x4*)(k_to + i * CPL * 256u + (odd ^ 1u) * 128u) = keys_of<F16>(k_raw[i][2], k_raw[i][3], by);
                }
#pragma unroll
            for (uint32_t i = 0; i < VL; i++) {
                float each[8];
#pragma unroll
                for (int e = 0; e < 8; e++) each[e] = scale_of((uint32_t)(v_by[x * GROUPS + (ONE ? i / GL : 0)] >> (8 * e)) & 0xffu);
                u32x4 a0, a1;
                values_of<F16>(v_raw[i], each, a0, a1);
                /* neighbouring numbers exchanged in every other sixteen: sixteen lanes that write every other piece meet all banks */
                uint8_t* const at = v_to + (i / GL * DP + i % GL * 128u) * 16u;
                if (FULL || ((i % GL) * 64u + v_pair) * 2u < D) {
                    *(u32x4*)(at + (v_pair >> 3 & 1u) * 16u) = a0;
                    *(u32x4*)(at + ((v_pair >> 3 & 1u) ^ 1u) * 16u) = a1;
                }
            }
        }
    };
    next_blocks();
    bool more = there;
    if (more) { enter_next(); load_tile(0); if constexpr (E8) put_tile(0); }
    /* the lane's row of K among the places of 32 tokens: the one that puts the scores of tokens 8 half .. + 7 of each 16 into its accumulators */
    const uint32_t k_row = T < 16 ? (row & 0x13u) | ((row & 4u) << 1) | ((row & 8u) >> 1) : row;
    const uint32_t k_read = (k_row >> 3) * DP * 16u + (k_row & 7u) * 16u + (half ^ (k_row >> 3 & 1u)) * 128u;
    const uint32_t v_row = E8 ? row ^ (row >> 4) : row;
    for (uint32_t buf = 0; more; buf ^= 1u) {
        fence_meta();                            /* this wave's part of the tile is in LDS, */
        __syncthreads();                         /* and everybody's; and everybody has done with the buffer that is loaded next */
        const uint32_t t0 = at_first, t_lim = at_end, t_block = at_block;
        const uint64_t t_holes = at_holes;
        more = true;
        if (t_next >= t_end) {
            more = there;
            if (more) { look_again(); enter_next(); }
        }
        if (more) load_tile(buf ^ 1u);
        const uint8_t* const keys = (const uint8_t*)lds + buf * 2u * HALF;
        const uint8_t* const values = keys + HALF;
        /* whether all rows from `from` to `to` see all of the tile */
        auto all_seen = [&](const int32_t from, const int32_t to) {
            return !t_holes && (int32_t)(t0 + KT) - 1 <= from && t0 + KT <= t_lim && (!a.window || to - (int32_t)t0 < (int32_t)a.window || t0 + KT <= a.sinks);
        };
        if (!all_seen(first_of_all, last_of_all)) {
            /* values of tokens that a row does not see meet zeros of P.  That leaves them out unless there is an infinity or NaN among them: then
             * the split is left to the launch that takes the rows one by one there (kv_steps).  Each wave looks at a part of the values. */
            bool odd = false;
#pragma unroll
            for (uint32_t n = 0; n < PIECES / (64u * NW); n++) {
                const u32x4 z = *(const u32x4*)(values + (n * 64u * NW + threadIdx.x) * 16u);
                odd |= odd16<F16>(z[0]) || odd16<F16>(z[1]) || odd16<F16>(z[2]) || odd16<F16>(z[3]);
            }
            if (ballot(odd)) ok = false;
        }
        do {
        if (idle || (int32_t)t0 > last_pos) break;
        /*
         * The operands from LDS are read eight ahead of the products that take them, and the order is held (sched_barrier): left to itself the compiler reads each right before
         * its product and waits for it, a hundred cycles for every 32 of the matrix unit.
         */
        constexpr uint32_t NK = DP / 16 * (KT / 32), NV = DP / 32 * (KT / 16);
        auto key_piece = [&](const uint32_t n) { return *(const u32x4*)(keys + (n / (KT / 32)) * 256u + (n % (KT / 32)) * (DP * 64u) + k_read); };
        auto value_piece = [&](const uint32_t n) { return *(const u32x4*)(values + ((2u * (n / (DP / 32)) + half) * DP + 32u * (n % (DP / 32)) + v_row) * 16u); };
        f32x16 x[KT / 32];
#pragma unroll
        for (uint32_t mt = 0; mt < KT / 32; mt++)
#pragma unroll
            for (int e = 0; e < 16; e++) x[mt][e] = 0;
        u32x4 f[8];
#pragma unroll
        for (uint32_t n = 0; n < 8; n++) f[n] = key_piece(n);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t n = 0; n < NK; n += 4) {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) x[(n + e) % (KT / 32)] = mma32<F16>(f[(n + e) % 8], q[(n + e) / (KT / 32)], x[(n + e) % (KT / 32)]);
            /* behind the last keys, the first values */
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) f[(n + e) % 8] = n + 8 < NK ? key_piece(n + 8 + e) : value_piece(n + 8 + e - NK);
            __builtin_amdgcn_sched_barrier(0);
        }
        const bool whole = all_seen(first_pos, last_pos);
        if (!whole) {
            uint32_t sees = 0;                   /* of each 16 tokens, which of its eight the row sees */
            const int32_t lim = (int32_t)t_lim - 1;
#pragma unroll
            for (uint32_t k = 0; k < KT / 16; k++) {
                const uint32_t tt = t0 + k * 16u + half * 8u;
                if ((t_holes >> (((tt >> g.tokens_log) - t_block) & 63u)) & 1u) continue;
                sees |= seen_of_eight((int32_t)tt, pos < lim ? pos : lim, low_of(a, pos), (int32_t)a.sinks) << (8u * k);
            }
#pragma unroll
            for (uint32_t mt = 0; mt < KT / 32; mt++)
#pragma unroll
                for (uint32_t e = 0; e < 16; e++) x[mt][e] = (sees >> (16u * mt + e)) & 1u ? x[mt][e] : -INFINITY;
        }
        float top = x[0][0];
#pragma unroll
        for (uint32_t mt = 0; mt < KT / 32; mt++)
#pragma unroll
            for (int e = 0; e < 16; e++) top = __builtin_elementwise_maximum(top, x[mt][e]);      /* three operands to an instruction, and no quieting of each */
        {
            float other = top;
            swap_halves(top, other);
            top = fmaxf(top, other);
        }
        /* the sums are moved to a larger maximum only where its weight would be above 2^TILE_SLACK: up to there weights lose nothing */
        if (ballot((top - m) * c > TILE_SLACK<F16> || (m == -INFINITY && top != -INFINITY))) {
            const float larger = fmaxf(top, m);
            const float by = larger == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - larger) * c);
            l *= by;
            l1 *= by;
#pragma unroll
            for (uint32_t i = 0; i < DP / 32; i++) o[i] *= by;
            m = larger;
        }
        const float mc = m == -INFINITY ? 0.0f : __builtin_fmaf(-m, c, TILE_SHIFT<F16>);
        u32x4 p[KT / 16];
#pragma unroll
        for (uint32_t k = 0; k < KT / 16; k++) {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const float y0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[k >> 1][(k & 1u) * 8u + 2u * e], c, mc)), y1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[k >> 1][(k & 1u) * 8u + 2u * e + 1u], c, mc));
                l += y0;
                l1 += y1;
                p[k][e] = to16<F16>(y0, y1);
            }
            /* the weights of the next sixteen tokens are worked out while the matrix unit has these */
#pragma unroll
            for (uint32_t i = 0; i < DP / 32; i++) {
                const uint32_t n = k * (DP / 32) + i;
                o[i] = mma32<F16>(f[(n + NK) % 8], p[k], o[i]);
                if (n + 8 < NV) f[(n + NK) % 8] = value_piece(n + 8);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        } while (false);
        if constexpr (E8) if (more) put_tile(buf ^ 1u);
    }
    fence_meta();
    look_again();
    if (__syncthreads_or(!ok)) { if (threadIdx.x == 0) a.left[(uint64_t)item * a.splits + split] = 1; return; }
    if (threadIdx.x == 0) a.left[(uint64_t)item * a.splits + split] = 0;
    if (wave == 0) count_accesses(g, lane == 0 ? n_access : 0u, lane == 0 ? n_access : 0u);
    {
        l += l1;
        float other = l;
        swap_halves(l, other);
        l += other;
    }
    if (!has) return;
    const float at_one = m == -INFINITY ? -INFINITY : -__builtin_fmaf(-m, c, TILE_SHIFT<F16>);      /* the score whose weight in the sums is one */
    /* lane: numbers 8i + 4 half .. + 3 of its row */
    if (a.splits > 1) {
        const uint64_t at = ((uint64_t)item * a.tile_rows + (r - it.r0)) * a.splits + split;
#pragma unroll
        for (uint32_t i = 0; i < DP / 8; i++) {
            const uint32_t d = 8u * i + 4u * half;
            if (d < D) *(f32x4*)(a.part + at * D + d) = f32x4{o[i / 4][i % 4 * 4], o[i / 4][i % 4 * 4 + 1], o[i / 4][i % 4 * 4 + 2], o[i / 4][i % 4 * 4 + 3]};
        }
        if (half == 0) { a.part_m[at] = at_one; a.part_l[at] = l; }
        return;
    }
    const float inv = m == -INFINITY ? 0.0f : 1.0f / l;
    uint16_t* const to = a.out + ((uint64_t)(it.start + (int32_t)tok) * a.q_heads + head) * D;
#pragma unroll
    for (uint32_t i = 0; i < DP / 8; i++) {
        const uint32_t d = 8u * i + 4u * half;
        if (d < D) {
            uint2 y;
            y.x = to16<F16>(o[i / 4][i % 4 * 4] * inv, o[i / 4][i % 4 * 4 + 1] * inv);
            y.y = to16<F16>(o[i / 4][i % 4 * 4 + 2] * inv, o[i / 4][i % 4 * 4 + 3] * inv);
            *(uint2*)(to + d) = y;
        }
    }
    if (a.lse && half == 0) a.lse[(uint64_t)(it.start + (int32_t)tok) * a.q_heads + head] = (at_one + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

/*
 * Both launches in one, where there are no more workgroups than compute units: the miss path beside the other wants all registers of a SIMD, which one workgroup to a compute
 * unit has.  One token over 200, heads of 64: 7.4 and 4.5 us of two launches, 7.6 of this one (10.2 a pass for 12.6); over 8000, of 128: 18.5 a pass for 20.0; 7 sequences of 3000
 * 22.2 for 23.9; 60000 and more: the same.  Heads of 256 would spill (5 % slower over 60000), and keep two launches.
 */
template <int DP, int F16, int E8, int NT>
__global__ __launch_bounds__(256) void k_kv_attend_once(const kv_geom g, const kv_seqs s, const kv_att a)
{
    extern __shared__ float lds[];
    const uint32_t item = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    kv_item it;
    bool gone = false;
    if (!item_of(g, s, a, item, it)) return;
    if (kv_split<DP, F16, E8, NT, false>(g, s, a, item, it, it.r0, split, lds, gone)) return;
    __syncthreads();
    gone = false;
    kv_split<DP, F16, E8, NT, true>(g, s, a, item, it, it.r0, split, lds, gone);
}

/* what the first launch left, with its pages held; ends at once where that is nothing */
template <int DP, int F16, int E8, int NT>
__global__ __launch_bounds__(256) void k_kv_rest(const kv_geom g, const kv_seqs s, const kv_att a)
{
    extern __shared__ float lds[];
    const uint32_t each = (a.items + gridDim.x - 1) / gridDim.x, first = blockIdx.x * each, last = first + each < a.items ? first + each : a.items;
    bool mine = false;
    for (uint64_t k = (uint64_t)first * a.splits + threadIdx.x; k < (uint64_t)last * a.splits; k += 256u) mine |= a.left[k] != 0;
    if (!__syncthreads_or(mine)) return;
    for (uint64_t x = (uint64_t)first * a.splits; x < (uint64_t)last * a.splits; x++) {
        kv_item it;
        if (!a.left[x] || !item_of(g, s, a, (uint32_t)(x / a.splits), it)) continue;
        for (uint32_t s0 = it.r0; s0 < it.r1; s0 += 16u * NT) {
            bool gone = false;
            kv_split<DP, F16, E8, NT, true>(g, s, a, (uint32_t)(x / a.splits), it, s0, (uint32_t)(x % a.splits), lds, gone);
            __syncthreads();
        }
    }
}

/*
 * The splits of a row joined: out = sum over splits of exp(m_s - m) O_s / sum of exp(m_s - m) l_s.  LPR lanes to a row, four numbers to a lane; WIDE: the four waves of a
 * workgroup share the splits of a row, else they have rows of their own.  32 splits of 32 rows: 4.6 us, 4 splits of 16 000 rows 7.5 (by the workgroups that look after
 * missing pages, an item each: 42 and 85 with 128 and 8 splits).
 */
template <int LPR, int F16, bool WIDE>
__global__ __launch_bounds__(256) void k_kv_join(const kv_geom g, const kv_seqs s, const kv_att a)
{
    __shared__ f32x4 sums[WIDE ? 256 : 1];
    __shared__ float tops[WIDE ? 256 : 1], dens[WIDE ? 256 : 1];
    constexpr uint32_t RPW = 64 / LPR;
    const uint32_t lane = bam::lane(), wave = threadIdx.x / 64u, c = lane % LPR * 4u, D = g.dim;
    const uint64_t x = (uint64_t)(WIDE ? blockIdx.x : blockIdx.x * 4u + wave) * RPW + lane / LPR;
    const uint32_t item = (uint32_t)(x / a.tile_rows), r = (uint32_t)(x % a.tile_rows);
    kv_item it;
    const bool has = item < a.items && item_of(g, s, a, item, it) && it.r0 + r < it.r1 && c < D;
    float top = -INFINITY, den = 0;
    f32x4 sum{0, 0, 0, 0};
    if (has) {
        const uint64_t at = ((uint64_t)item * a.tile_rows + r) * a.splits;
        auto take = [&](const float m, const float l, const f32x4 o) {
            const float larger = fmaxf(top, m), use = larger == -INFINITY ? 0.0f : larger;
            const float mine = __builtin_amdgcn_exp2f(top - use), by = __builtin_amdgcn_exp2f(m - use);
            den = den * mine + l * by;
            sum = sum * mine + o * by;
            top = larger;
        };
        const uint32_t step = WIDE ? 4u : 1u;
        uint32_t k = WIDE ? wave : 0u;
        for (; k + 3u * step < a.splits; k += 4u * step) {
            float m[4], l[4];
            f32x4 o[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) { m[i] = a.part_m[at + k + i * step]; l[i] = a.part_l[at + k + i * step]; o[i] = *(const f32x4*)(a.part + (at + k + i * step) * D + c); }
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) take(m[i], l[i], o[i]);
        }
        for (; k < a.splits; k += step) take(a.part_m[at + k], a.part_l[at + k], *(const f32x4*)(a.part + (at + k) * D + c));
        if constexpr (WIDE) { sums[threadIdx.x] = sum; tops[threadIdx.x] = top; dens[threadIdx.x] = den; }
    }
    if constexpr (WIDE) {
        __syncthreads();
        if (wave) return;
        if (has) {
            auto take = [&](const float m, const float l, const f32x4 o) {
                const float larger = fmaxf(top, m), use = larger == -INFINITY ? 0.0f : larger;
                const float mine = __builtin_amdgcn_exp2f(top - use), by = __builtin_amdgcn_exp2f(m - use);
                den = den * mine + l * by;
                sum = sum * mine + o * by;
                top = larger;
            };
#pragma unroll
            for (uint32_t w = 1; w < 4; w++) take(tops[w * 64u + lane], dens[w * 64u + lane], sums[w * 64u + lane]);
        }
    }
    if (!has) return;
    const float inv = top == -INFINITY && den == 0 ? 0.0f : 1.0f / den;
    const uint32_t rr = it.r0 + r, tok = (uint32_t)it.start + rr / a.group, h = it.head * a.group + rr % a.group;
    uint2 y;
    y.x = to16<F16>(sum[0] * inv, sum[1] * inv);
    y.y = to16<F16>(sum[2] * inv, sum[3] * inv);
    *(uint2*)(a.out + ((uint64_t)tok * a.q_heads + h) * D + c) = y;
    if (a.lse && c == 0) a.lse[(uint64_t)tok * a.q_heads + h] = (top + __builtin_amdgcn_logf(den)) * 0.6931471805599453f;
}
// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

/* a kernel and not a memset: the stream may be captured */
__global__ void k_kv_all_left(uint8_t* left, const uint64_t n)
{
    const uint64_t i = blockIdx.x * 256ull + threadIdx.x;
    if (i < n) left[i] = 1;
}

template <int DP, int F16, int E8>
void launch_tiles(const bam_kv_t* kv, const kv_seqs& s, const kv_att& a, const kv_plan& p, const dim3 grid, hipStream_t st)
{
    constexpr uint32_t lds = tile_lds<DP>();
    static_assert(lds <= 65536, "more LDS than a launch has without asking for it");
    const bool exact = kv->g.dim == DP;
    if (p.waves == 2 && exact) hipLaunchKernelGGL((k_kv_attend_tiles<DP, F16, E8, 2, true>), grid, dim3(128), lds, st, kv->g, s, a);
    else if (p.waves == 2) hipLaunchKernelGGL((k_kv_attend_tiles<DP, F16, E8, 2, false>), grid, dim3(128), lds, st, kv->g, s, a);
    else if (exact) hipLaunchKernelGGL((k_kv_attend_tiles<DP, F16, E8, 4, true>), grid, dim3(256), lds, st, kv->g, s, a);
    else hipLaunchKernelGGL((k_kv_attend_tiles<DP, F16, E8, 4, false>), grid, dim3(256), lds, st, kv->g, s, a);
}

template <int DP, int F16, int E8, int NT>
void launch_attend(const bam_kv_t* kv, const kv_seqs& s, kv_att a, const kv_plan& p, hipStream_t st)
{
    constexpr uint32_t lds = split_lds<DP, NT>();
    static_assert(lds <= 65536, "more LDS than a launch has without asking for it");
    /* what all waves that may hold pages ask for at a time stays under half the cache, or they push each other's pages out */
    const uint32_t least = kv->g.tokens < 32 ? 32 / kv->g.tokens : 1;
    const uint64_t half = kv->cache_pages / 2, all = p.items * p.splits;
    const bool once = DP <= 128 && kv->unheld && !p.waves && all <= 256 && all * 8 * least <= half;
    uint64_t groups = once ? all : p.items < 512 ? p.items : 512;
    if (groups * 8 * least > half) groups = half / (8 * least);
    uint64_t chunk = half / (groups * 8) / least * least;
    a.chunk = (uint32_t)(chunk > 32 ? 32 : chunk);
    a.tile_rows = p.rows;
    const dim3 grid((uint32_t)all);
    if (once) {
        if constexpr (DP <= 128) hipLaunchKernelGGL((k_kv_attend_once<DP, F16, E8, NT>), grid, dim3(256), lds, st, kv->g, s, a);
    } else {
        if (!kv->unheld) hipLaunchKernelGGL(k_kv_all_left, dim3((uint32_t)((all + 255) / 256)), dim3(256), 0, st, a.left, all);
        else if (!p.waves) hipLaunchKernelGGL((k_kv_attend<DP, F16, E8, NT>), grid, dim3(256), lds, st, kv->g, s, a);
        else if constexpr (NT == 2) {
            /* heads of up to 96 numbers in 8 bits: without the products of a third as many zeros (4 prompts of 8000 tokens, heads of 96, window 1024: 617 and 558 us) */
            if constexpr (E8 && DP == 128) {
                if (kv->g.dim <= 96) launch_tiles<96, F16, E8>(kv, s, a, p, grid, st);
                else launch_tiles<DP, F16, E8>(kv, s, a, p, grid, st);
            } else launch_tiles<DP, F16, E8>(kv, s, a, p, grid, st);
        }
        hipLaunchKernelGGL((k_kv_rest<DP, F16, E8, NT>), dim3((uint32_t)groups), dim3(256), lds, st, kv->g, s, a);
    }
    if (p.splits == 1) return;
    constexpr int LPR = DP / 4;
    const uint64_t rows = p.items * p.rows, rpw = 64 / LPR;
    if (p.splits >= 16) hipLaunchKernelGGL((k_kv_join<LPR, F16, true>), dim3((uint32_t)((rows + rpw - 1) / rpw)), dim3(256), 0, st, kv->g, s, a);
    else hipLaunchKernelGGL((k_kv_join<LPR, F16, false>), dim3((uint32_t)((rows + 4 * rpw - 1) / (4 * rpw))), dim3(256), 0, st, kv->g, s, a);
}
template <int DP, int F16, int E8>
void launch_attend(const bam_kv_t* kv, const kv_seqs& s, const kv_att& a, const kv_plan& p, hipStream_t st)
{
    if (p.nt == 1) launch_attend<DP, F16, E8, 1>(kv, s, a, p, st);
    else launch_attend<DP, F16, E8, 2>(kv, s, a, p, st);
}
template <int F16, int E8>
void launch_attend(const bam_kv_t* kv, const kv_seqs& s, const kv_att& a, const kv_plan& p, hipStream_t st)
{
    if (kv->g.dim <= 64) launch_attend<64, F16, E8>(kv, s, a, p, st);
    else if (kv->g.dim <= 128) launch_attend<128, F16, E8>(kv, s, a, p, st);
    else launch_attend<256, F16, E8>(kv, s, a, p, st);
}

} // namespace
#endif /* __BAM_KV_ATTEND_H__ */
