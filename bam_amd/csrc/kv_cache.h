// The key-value cache in the pages of an array: the handle, where tokens lie, visits of pages, and rows into the cache and out of it.
//
// The cache is cut into blocks of T tokens.  A block has two pages for each key-value head: one of keys and one of values, T the largest power of
// two for which T rows of `dim` 16-bit numbers fit a page.  Within a page the numbers lie in pieces of 16 bytes, in the order in
// which the matrix instructions take them:
//   keys    piece (c, t) at (c * T + place(t)) * 16: numbers 8c .. 8c+7 of token t             c < dim / 8
//   values  piece (t, d) at (t * dim + d) * 16: number d of tokens 8t .. 8t+7           t < T / 8
// and in 8 bits (T rows of `dim` bytes fit a page, sixteen at least)
//   keys    piece (c, t) at (c * T + place(t)) * 16: numbers 16c .. 16c+15 of token t           c < dim / 16
//   values  piece (t, x) at (t * dim/2 + x) * 16: numbers 2x and 2x+1 of token 8t, of 8t+1, ..       t < T / 8
// place(t) is t with its bits 2 and 3 exchanged (t itself where a page holds eight tokens).  What neighbouring lanes of a wave load lies next to each other, and
// is an operand as it stands: with the scores taken as S^T = K Q^T and the output as O^T = V^T P^T, a lane's accumulators of the scores are its
// part of P^T if the rows of K come in that order.
#ifndef __BAM_KV_CACHE_H__
#define __BAM_KV_CACHE_H__
#include "bam_capi_internal.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// what a kernel knows about the cache: the range's tables do not move while the array is there
struct kv_geom {
    range_d_t<uint64_t>* r;
    data_page_t* pages;
    uint8_t* base;
    uint64_t first_page, n_blocks;
    uint32_t heads, dim, tokens, tokens_log, page_log;
    uint8_t* scales;                    /* 8 bits: powers of two of the rows, [pages of the cache][tokens], each 127 more than it is; 16 bits: NULL */
};
struct bam_kv {
    bam_array_t* a;
    kv_geom g;
    int f16, e8;                        /* e8: 8 bits in the pages */
    uint64_t cache_pages;
    bool unheld;                        /* reads of resident pages without a reference are switched on */
};
struct kv_seqs {
    const int32_t* starts;              /* [n + 1] first row of each sequence's new tokens; NULL: one new token each */
    const int32_t* lens;                /* [n] tokens of each sequence, the new ones among them */
    const int32_t* table;               /* [n][width] blocks */
    int64_t stride;
    uint32_t n, rows, width;
};
struct kv_rows {
    const uint16_t *q, *k, *v;          /* rows of heads; k and v are where rows go to when the cache is read */
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    uint16_t* q_out;
    const uint16_t *q_norm, *k_norm;
    const float *cos, *sin;
    uint32_t positions, q_heads, rot, pairs, aligned;      /* aligned: q, k, v in whole pieces of 16 bytes */
    float eps;
    double of_dim;                      /* 1 / dim */
    uint32_t window, piece;             /* rows that a wave looks for beginnings of runs among, and the most rows it takes at a time */
    uint32_t q_heads_each, q_waves;     /* heads of queries that a wave takes; waves that do */
    uint32_t kv_blocks, among;          /* workgroups for keys and values, which are spread among so many from the first on */
    uint32_t by_head;                   /* waves in the order of the heads, each one's windows side by side */
};

namespace {

// sequence of row i, which is one of [lo, hi): the last that starts at or before it
__device__ __forceinline__ uint32_t seq_of(const kv_seqs& s, const uint32_t i, uint32_t lo, uint32_t hi)
{
    if (!s.starts) return i;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (s.starts[mid] <= (int32_t)i) lo = mid; else hi = mid;
    }
    return lo;
}
/* the same for a row that is the whole wave's: 64 places are looked at at a time (a look takes a microsecond of what a small call takes; 512 sequences are two looks and not nine) */
__device__ __forceinline__ uint32_t seq_of_wave(const kv_seqs& s, const uint32_t i)
{
    if (!s.starts) return i;
    uint32_t lo = 0, hi = s.n;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 63u) / 64u, at = lo + step * bam::lane();
        const uint64_t m = bam::ballot(at < hi && s.starts[at < hi ? at : lo] <= (int32_t)i) | 1ull;
        lo += step * (63u - (uint32_t)__builtin_clzll(m));
        hi = hi - lo < step ? hi : lo + step;
    }
    return lo;
}
// a row's place: sequence, position, rows of its sequence from it on (those that there are: starts may say more than `rows`), position of its sequence's first new
// row; false where the row has none (no such sequence, before the first position, past the table)
struct kv_place { uint32_t seq, pos, rest, first; };
__device__ __forceinline__ bool place_of(const kv_seqs& s, const kv_geom& g, const uint32_t i, const uint32_t lo, const uint32_t hi, kv_place& p)
{
    p.seq = seq_of(s, i, lo, hi);
    if (p.seq >= s.n) return false;
    const int32_t end = s.starts ? s.starts[p.seq + 1] : (int32_t)i + 1;
    int32_t begin = s.starts ? s.starts[p.seq] : (int32_t)i;
    if (begin < 0) begin = 0;
    const int64_t len = s.lens[p.seq], pos = len - (end - (int64_t)i);
    if ((int32_t)i < begin || (int64_t)i >= end || pos < 0 || (pos >> g.tokens_log) >= s.width) return false;
    p.pos = (uint32_t)pos;
    p.rest = ((uint32_t)end < s.rows ? (uint32_t)end : s.rows) - i;
    const int64_t first = len - ((int64_t)end - begin);
    p.first = first < 0 ? 0u : (uint32_t)first;
    return true;
}
// the page of keys of a block (the page of values is the next one), or false: no such block
__device__ __forceinline__ bool page_of_block(const kv_geom& g, const kv_seqs& s, const uint32_t seq, const uint32_t i, const uint32_t head, uint64_t& page)
{
    if (i >= s.width) return false;
    const int32_t b = s.table[(int64_t)seq * s.stride + i];
    if (b < 0 || (uint64_t)b >= g.n_blocks) return false;
    page = g.first_page + ((uint64_t)b * g.heads + head) * 2u;
    return true;
}

/* where a token of a block lies among its block's keys */
__device__ __forceinline__ uint32_t place_in(const kv_geom& g, const uint32_t t) { return g.tokens < 16 ? t : (t & ~12u) | (t & 4u) << 1 | (t & 8u) >> 1; }

template <int F16> __device__ __forceinline__ float from16(const uint32_t x)
{
    if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)x);
    else return __builtin_bit_cast(float, x << 16);
}
template <int F16> __device__ __forceinline__ uint32_t to16(const float lo, const float hi)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), _Float16 __attribute__((ext_vector_type(2)))));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), __bf16 __attribute__((ext_vector_type(2)))));
}
template <bool ALIGNED> __device__ __forceinline__ u32x4 load_piece(const uint16_t* p)
{
    if constexpr (ALIGNED) return *(const u32x4*)p;
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return x;
}

// ---- the cache in 8 bits ----
/*
 * A row y (a token's keys of a head, or its values) is kept as e4m3 numbers (a sign, four bits of exponent, three of mantissa; the largest is 448) and a power of two: k is
 * the least whole number with max |y| <= 448 * 2^k, between the bounds below, and what is kept of a number is y / 2^k rounded to the nearest, ties to even.
 * A power of two and not max |y| / 448: what a row stands for is then exact in the 16-bit types (4 significant bits, and a range that the bounds keep inside theirs; in
 * float16 but for what is smaller than that type's steps of 2^-24), so the matrix unit takes it without a second rounding; and a number of 4 significant bits is no nearer for another
 * scale.  For the same reason there is no need of e5m2's range.
 * Bounds: 448 * 2^k is over the type's largest for the upper one; the lower one keeps 2^(k - 9), the smallest step, a normal number (bfloat16), or the type's smallest numbers
 * whole (float16).  A number of 1.9375 and more times the type's largest power of two would be rounded up past the type: it is kept as 1.875 times that, less than a step of an
 * eighth away.  What is not finite is kept as NaN, and has no part in k.
 */
template <int F16> constexpr int32_t LEAST_POWER = F16 ? -24 : -110;
template <int F16> constexpr int32_t MOST_POWER = F16 ? 8 : 120;
template <int F16> constexpr float MOST_KEPT = F16 ? 1.875f * 0x1p15f : 1.875f * 0x1p127f;
/* largest of the numbers of magnitude |x|, those that are not finite left out */
__device__ __forceinline__ float larger_finite(const float a, const float x) { const float m = fabsf(x); return m < INFINITY ? fmaxf(a, m) : a; }
__device__ __forceinline__ float scale_of(const uint32_t power) { return __builtin_bit_cast(float, power << 23); }
__device__ __forceinline__ float inverse_of(const uint32_t power) { return __builtin_bit_cast(float, (254u - power) << 23); }
/* 127 + k for a largest number of a 2^down (numbers that are larger than the type's largest are in 32 bits with a power of two less) */
template <int F16> __device__ __forceinline__ uint32_t power_of(const float a, const uint32_t down)
{
    const uint32_t bits = __builtin_bit_cast(uint32_t, fminf(a, MOST_KEPT<F16> * inverse_of(127u + down)));
    const int32_t k = (int32_t)(bits >> 23) + (int32_t)down - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return 127u + (uint32_t)(k < LEAST_POWER<F16> ? LEAST_POWER<F16> : k > MOST_POWER<F16> ? MOST_POWER<F16> : k);
}
/* a number, the largest that is kept, and 2^-k, the first two 2^-down of what they are and the last 2^down of it */
__device__ __forceinline__ float for8(const float y, const float most, const float inverse)
{
    return fabsf(y) < INFINITY ? fminf(fmaxf(y, -most), most) * inverse : __builtin_nanf("");
}
/* two numbers in the low or the high half of a word */
template <int F16, bool HIGH> __device__ __forceinline__ uint32_t to8(const uint32_t word, const float a, const float b, const float inverse, const float most = MOST_KEPT<F16>)
{
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(for8(a, most, inverse), for8(b, most, inverse), (int)word, HIGH);
}
/* two numbers of the low or the high half of a word, times a power of two, in 16 bits */
template <int F16, bool HIGH> __device__ __forceinline__ uint32_t from8(const uint32_t word, const float scale)
{
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, HIGH));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, HIGH));
}

// ---------------------------------------------------------------------------
// pages held for the length of a visit
// ---------------------------------------------------------------------------
#define KV_PASS_FRESH 512u
#define KV_PASS_CLEARED 1024u
__attribute__((noinline)) __device__ bam_pass_t kv_pass(range_d_t<uint64_t>* r, const uint64_t pg, const uint32_t queue, uint64_t sv, const uint32_t in)
{
    bool hit = false, progressed = false, wants = false;
    uint32_t slot = 0;
    const bool resolved = r->template slow_step<true>(pg, (in & BAM_PASS_WRITE) != 0, queue, sv, slot, hit, progressed, (in & BAM_PASS_TAKE_PART) != 0, true, &wants, BAM_PLACE_NORMAL,
                                                      (in & KV_PASS_FRESH) != 0, (in & KV_PASS_CLEARED) != 0);
    bam_pass_t out;
    out.sv = sv;
    out.slot = slot;
    out.flags = (resolved ? BAM_PASS_RESOLVED : 0u) | (hit ? BAM_PASS_HIT : 0u) | (progressed ? BAM_PASS_PROGRESSED : 0u);
    return out;
}

/*
 * use(address of the slot of the keys or NULL, and of the values) by the whole wave, with those pages held: two neighbouring pages, as range_view::acquire_helped would
 * have them, what is resident first and nothing held while the other is fetched, with what a writer of rows can say besides (`fresh`, `cleared`:
 * range_d_t::slow_step).  It stores past the caches (st16_sys and the like), so a wait for the wave's own stores is all that giving a page back needs: the
 * write-back of the cluster's cache that a release costs would come once per wave.  The miss path is a call: what the rows need is loaded in `use`, behind it (loaded
 * before, it would be kept across the call, in so many registers that one wave is left to a SIMD).  Returns the pages that were not visited since the wait was given up
 * (1: keys, 2: values).
 */
template <bool WRITE, typename F>
__device__ __forceinline__ uint32_t visit(const kv_geom& g, const uint64_t page, const bool fresh, const bool cleared, F&& use)
{
    using namespace bam;
    const uint32_t me = lane();
    data_page_t* const dp = g.pages + page + (me & 1u);
    uint64_t sv = 0;
    uint32_t slot = 0, n_hit = 0;
    bool open = me < 2, in = false;
    if (open) in = bam_try_hit(dp, 1, WRITE, sv, slot);
    uint32_t todo = 3;
    spin_t sp;
    const uint32_t queue = wave_slot_hash();
    for (bool again = false;; again = true) {
        uint32_t got = (uint32_t)ballot(in && open);
        if (!again) n_hit = popc(got);
        if (got) {
            use(got & 1u ? g.base + ((uint64_t)bcast(slot, 0) << g.page_log) : nullptr, got & 2u ? g.base + ((uint64_t)bcast(slot, 1) << g.page_log) : nullptr);
            fence_meta();
            if (in && open) { __hip_atomic_fetch_add(&dp->state, 0u - 1u, __ATOMIC_RELAXED, BAM_AGENT); open = false; }
            todo &= ~got;
        }
        if (__builtin_expect(todo == 0, 1)) break;
        const bam_pass_t ps = kv_pass(g.r, page + (me & 1u), queue, sv, (WRITE ? BAM_PASS_WRITE : 0u) | (open ? BAM_PASS_TAKE_PART : 0u) | (fresh ? KV_PASS_FRESH : 0u) | (cleared ? KV_PASS_CLEARED : 0u));
        if (open) { sv = ps.sv; slot = ps.slot; in = (ps.flags & BAM_PASS_RESOLVED) != 0; n_hit += in && (ps.flags & BAM_PASS_HIT) ? 1u : 0u; }
        if (ballot((ps.flags & BAM_PASS_PROGRESSED) != 0)) sp = spin_t();
        else if (!ballot(in && open) && g.r->cache.spin_giveup(sp)) {
            if (open) __hip_atomic_fetch_add(&dp->state, 0u - 1u, __ATOMIC_RELAXED, BAM_AGENT);
            break;
        }
    }
    if (me == 0) {
        bam_stat_shard_t* const shard = g.r->shard();
        __hip_atomic_fetch_add(&shard->access_cnt, 2ull, __ATOMIC_RELAXED, BAM_AGENT);
        if (n_hit) __hip_atomic_fetch_add(&shard->hit_cnt, (unsigned long long)n_hit, __ATOMIC_RELAXED, BAM_AGENT);
    }
    return todo;
}

// the wave's accesses into the range's counters
__device__ __forceinline__ void count_accesses(const kv_geom& g, const uint32_t n_access, const uint32_t n_hit)
{
    bam_stat_shard_t* const shard = g.r->shard();
    bam::stat_add<32>(&shard->access_cnt, n_access);
    bam::stat_add<32>(&shard->hit_cnt, n_hit);
}

// ---------------------------------------------------------------------------
// rows into the cache and out of it
// ---------------------------------------------------------------------------

/* the angles of eight neighbouring numbers of a row; lanes whose numbers are not turned load some, and do not use them */
struct kv_turn { f32x4 c[2], s[2]; };
__device__ __forceinline__ kv_turn turn_of(const kv_rows& io, const uint32_t piece, const uint32_t pos)
{
    kv_turn t;
    if (!io.rot) return t;
    const uint32_t half = io.rot / 2, hp = io.rot / 16;
    const bool known = pos < io.positions;
    const uint64_t row = (uint64_t)(known ? pos : 0u) * half;
    if (io.pairs) {
        const uint64_t at = row + (piece < 2u * hp ? piece : 0u) * 4u;
        t.c[0] = *(const f32x4*)(io.cos + at);
        t.s[0] = *(const f32x4*)(io.sin + at);
    } else {
        const uint64_t at = row + (piece < hp ? piece : piece < 2u * hp ? piece - hp : 0u) * 8u;
        t.c[0] = *(const f32x4*)(io.cos + at); t.c[1] = *(const f32x4*)(io.cos + at + 4);
        t.s[0] = *(const f32x4*)(io.sin + at); t.s[1] = *(const f32x4*)(io.sin + at + 4);
    }
    if (!known) {
        const float nan = __builtin_nanf("");
        t.c[0] = t.c[1] = t.s[0] = t.s[1] = f32x4{nan, nan, nan, nan};
    }
    return t;
}

/*
 * Eight neighbouring numbers of a row per lane, LPR lanes to a row: x * rsqrt(mean x^2 + eps) * w, then the rotation of the pairs (i, i + rot/2), or
 * (2i, 2i+1), i < rot/2, by the angles of the row's position; in 32 bits, rounded once.  A position past the tables gives NaN.
 */
template <int F16> __device__ __forceinline__ void in_32_bits(const u32x4 x, float (&f)[8])
{
#pragma unroll
    for (int i = 0; i < 4; i++) { const uint32_t y = x[i]; f[2 * i] = from16<F16>(y & 0xffffu); f[2 * i + 1] = from16<F16>(y >> 16); }
}
template <int LPR, int F16>
__device__ __forceinline__ void norm_and_rotate(const kv_rows& io, const kv_geom& g, float (&f)[8], const bool norm, const u32x4 w, const kv_turn& t, const uint32_t piece)
{
    if (norm) {
        float ss = 0;                            /* (pieces past the row's end are zero) */
#pragma unroll
        for (int i = 0; i < 8; i++) ss += f[i] * f[i];
#pragma unroll
        for (int o = LPR / 2; o; o >>= 1) ss += __shfl_xor(ss, o);
        const float by = rsqrtf(ss / (float)g.dim + io.eps);
#pragma unroll
        for (int i = 0; i < 4; i++) { const uint32_t y = w[i]; f[2 * i] *= by * from16<F16>(y & 0xffffu); f[2 * i + 1] *= by * from16<F16>(y >> 16); }
    }
    if (io.rot) {
        const uint32_t pieces = io.rot / 8, hp = pieces / 2;
        const bool turns = piece < pieces;
        if (io.pairs) {
            if (turns) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float a = f[2 * i], b = f[2 * i + 1];
                    f[2 * i] = a * t.c[0][i] - b * t.s[0][i];
                    f[2 * i + 1] = b * t.c[0][i] + a * t.s[0][i];
                }
            }
        } else {
            const uint32_t from = (bam::lane() & ~(uint32_t)(LPR - 1)) + (turns ? (piece < hp ? piece + hp : piece - hp) : piece);
            const float sign = piece < hp ? -1.0f : 1.0f;
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = __shfl(f[i], (int)from);
            if (turns) {
#pragma unroll
                for (int i = 0; i < 8; i++) f[i] = f[i] * t.c[i / 4][i % 4] + sign * o[i] * t.s[i / 4][i % 4];
            }
        }
    }
}
template <int LPR, int F16>
__device__ __forceinline__ u32x4 norm_and_rotate(const kv_rows& io, const kv_geom& g, u32x4 x, const bool norm, const u32x4 w, const kv_turn& t, const uint32_t piece)
{
    if (!norm && !io.rot) return x;
    float f[8];
    in_32_bits<F16>(x, f);
    norm_and_rotate<LPR, F16>(io, g, f, norm, w, t, piece);
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = to16<F16>(f[2 * i], f[2 * i + 1]);
    return x;
}
/* to 32 bits so that what is rounded to fewer next comes out as if from the 64: towards zero, and the last bit set where something was cut off */
__device__ __forceinline__ float to_odd(const double x)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)b;
    return (float)__builtin_bit_cast(double, (b & ~0xffffffffull) | (((lo & 0x1fffffffu) + 0x1fffffffu | lo) & 0xe0000000u));
}
/*
 * The same for what goes into 8 bits, with the sums and the turned numbers in 64 bits: a step of 8 bits is a sixteenth of a number, and one that lies within the error of the arithmetic of a border between
 * two of them comes out a whole step off (of 20 million, 32 in 32 bits, 11 with 64 that were rounded to 32 on the way, none like this; 9 us of 127).  On the borders themselves are rows of one
 * magnitude, which the norm makes plus or minus the weights: with a factor that is 2^-45 off, always downwards, a third of them went to the wrong side.  What is multiplied in 32 bits is exact: 16-bit
 * numbers and weights, the numbers scaled by a power of two near one over their mean size.
 *   What comes out is 2^-5 of the row, which is in range whatever the weights are (a number is at most sqrt(256) of the mean size, sqrt(2) of that turned): a normed key past the type's largest number is kept as
 * that and not as NaN.  The 5 is returned; 0 where there is nothing to do, and the row is as it was.
 */
template <int LPR, int F16>
__device__ __forceinline__ uint32_t norm_and_rotate_for_8(const kv_rows& io, const uint32_t dim, const u32x4 x, float (&f)[8], const bool norm, const u32x4 w, const kv_turn& t, const uint32_t piece)
{
    constexpr int DOWN = 5;
    in_32_bits<F16>(x, f);
    if (!norm && !io.rot) return 0;
    double by = 1.0 / (1 << DOWN), more = 0;
    auto normed = [&](const double y) { return to_odd(__builtin_fma(by, y, more * y)); };      /* (by + more) y, rounded to 64 bits once */
    if (norm) {
        double ss = 0;                           /* (pieces past the row's end are zero) */
#pragma unroll
        for (int i = 0; i < 8; i++) ss = __builtin_fma((double)f[i], (double)f[i], ss);
#pragma unroll
        for (int o = LPR / 2; o; o >>= 1) ss += __shfl_xor(ss, o);
        /* (the quotient by the head's dimension, whose reciprocal is rounded where it is no power of two) */
        const double mean = ss * io.of_dim, rest = __builtin_fma(-mean, (double)dim, ss), v = (rest - rest == 0 ? __builtin_fma(rest, io.of_dim, mean) : mean) + (double)io.eps;
        /* v = u 4^e with u from one to four, and so not at the ends of a float's range; 1 / sqrt(u) in 32 bits, a step of Newton's, 2^-45 off, and what a second one adds, kept beside it (zero, infinity and NaN
         * without) */
        const int e = v > 0 && v < __builtin_inf() ? (int)(((__builtin_bit_cast(uint64_t, v) >> 52) + 1u) >> 1) - 512 : 0;
        const double u = ldexp(v, -2 * e), first = (double)rsqrtf((float)u);
        by = first;
        if (u > 0 && u < __builtin_inf()) {
            by = __builtin_fma(0.5 * first, __builtin_fma(-u * first, first, 1.0), first);
            const double h = u * by, cut = __builtin_fma(u, by, -h);
            more = 0.5 * by * (__builtin_fma(-h, by, 1.0) - cut * by);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t y = w[i];
            f[2 * i] = ldexpf(f[2 * i], -e - DOWN) * from16<F16>(y & 0xffffu);
            f[2 * i + 1] = ldexpf(f[2 * i + 1], -e - DOWN) * from16<F16>(y >> 16);
        }
    }
    const uint32_t pieces = io.rot / 8, hp = pieces / 2;
    const bool turns = piece < pieces;
    if (io.rot && io.pairs) {
        if (turns) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const double a = f[2 * i], b = f[2 * i + 1], c = t.c[0][i], sn = t.s[0][i];
                f[2 * i] = normed(a * c - b * sn);
                f[2 * i + 1] = normed(b * c + a * sn);
            }
            return DOWN;
        }
    } else if (io.rot) {
        const uint32_t from = (bam::lane() & ~(uint32_t)(LPR - 1)) + (turns ? (piece < hp ? piece + hp : piece - hp) : piece);
        const float sign = piece < hp ? -1.0f : 1.0f;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = __shfl(f[i], (int)from);
        if (turns) {
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = normed((double)f[i] * (double)t.c[i / 4][i % 4] + (double)(sign * o[i]) * (double)t.s[i / 4][i % 4]);
            return DOWN;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = normed((double)f[i]);
    return DOWN;
}
/* the power of two of a row whose numbers LPR lanes have */
template <int LPR, int F16> __device__ __forceinline__ uint32_t power_of_row(const float (&f)[8], const uint32_t down = 0)
{
    float a = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) a = larger_finite(a, f[i]);
#pragma unroll
    for (int o = LPR / 2; o; o >>= 1) a = fmaxf(a, __shfl_xor(a, o));
    return power_of<F16>(a, down);
}

/*
 * A wave takes some heads of queries of one row, or one head's keys and values of the runs of rows that begin among io.window rows: a run is the new rows of
 * a sequence in one block, gone through in pieces of up to io.piece tokens (eight or sixteen that begin at a multiple of that).  A page's rows all belong to one
 * wave: a page that holds new rows only is not read, and one that a second wave found gone again would come without the rows of the first.
 *   Bound by memory where there are many rows: 19 459 rows of 32 heads on 8 of 128 numbers, normed and turned, 480 MB in 118 us (4.1 TB/s), 160 MB out again in 55, in 8 bits
 * 440 MB in 130 and 120 MB in 42; a wave for each four rows took 288 and 112 (each looked its sequence up for 1 KiB).  Few rows: the chain of looks, table, references, rows, 6 to 7 us.
 */
template <int LPR, int F16, int E8, bool WRITE, bool ALIGNED>
__global__ __launch_bounds__(256, LPR < 32 ? 4 : 3) void k_kv_rows(const kv_geom g, const kv_seqs s, const kv_rows io)
{
    using namespace bam;
    constexpr uint32_t RPW = 64 / LPR, TRIPS = 16 / RPW, DT = LPR / 8;           /* trips of a piece's keys; of its values: a trip is 64 times two numbers of eight tokens */
    const uint32_t lane = bam::lane();
    uint32_t its_block = blockIdx.x;
    bool queries = false;
    if constexpr (WRITE) {
        auto in_front = [&](const uint32_t b) { return b < io.among ? (uint32_t)((uint64_t)b * io.kv_blocks / io.among) : io.kv_blocks; };
        const uint32_t before = in_front(blockIdx.x), behind = in_front(blockIdx.x + 1u);
        queries = before == behind;
        its_block = queries ? blockIdx.x - before : before;
    }
    const uint32_t wave = first(its_block * 4u + threadIdx.x / 64u);
    const uint32_t sub = lane / LPR, piece = lane % LPR;
    const bool in_row = piece * 8u < g.dim;
    const uint32_t col = in_row ? piece * 8u : 0u;           /* lanes past the row's end load its beginning, and count as zeros */
    if (WRITE && queries) {
        if (wave >= io.q_waves) return;
        const uint32_t per = (io.q_heads + io.q_heads_each - 1) / io.q_heads_each, i = wave / per, h0 = wave % per * io.q_heads_each;
        const uint32_t h1 = h0 + io.q_heads_each < io.q_heads ? h0 + io.q_heads_each : io.q_heads;
        kv_place p{0, 0, 0, 0};
        const uint32_t seq = seq_of_wave(s, i);
        const bool known = place_of(s, g, i, seq, seq + 1u, p);
        const kv_turn t = turn_of(io, piece, known ? p.pos : 0xffffffffu);
        u32x4 w{0, 0, 0, 0};
        if (io.q_norm) w = load_piece<true>(io.q_norm + col);
        const uint16_t* const from = io.q + (int64_t)i * io.q_row + col;
        uint16_t* const to = io.q_out + (uint64_t)i * io.q_heads * g.dim + col;
        for (uint32_t h = h0; h < h1; h += 4u * RPW) {
            u32x4 x[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint32_t hh = h + e * RPW + sub;
                x[e] = load_piece<ALIGNED>(from + (int64_t)(hh < h1 ? hh : h0) * io.q_head);
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint32_t hh = h + e * RPW + sub;
                if (h + e * RPW >= h1) break;
                x[e] = norm_and_rotate<LPR, F16>(io, g, in_row ? x[e] : u32x4{0, 0, 0, 0}, io.q_norm != nullptr, w, t, piece);
                if (hh < h1 && in_row) *(u32x4*)(to + hh * g.dim) = x[e];
            }
        }
        return;
    }
    const uint32_t n = wave, windows = (s.rows + io.window - 1u) / io.window, head = io.by_head ? n / windows : n % g.heads;
    const uint64_t first_row = (uint64_t)(io.by_head ? n % windows : n / g.heads) * io.window;
    if (head >= g.heads) return;
    if (first_row >= s.rows) return;
    kv_place p{0, 0, 0, 0};
    const uint32_t mine = (uint32_t)first_row + lane;
    /* the sequence of the first row, and from the beginnings of the 64 behind it, loaded at once, those of the others */
    const uint32_t first_seq = seq_of_wave(s, (uint32_t)first_row);
    uint32_t lo = first_seq, hi = first_seq + 1u;
    if (s.starts && io.window > 1u) {
        const int32_t begin = first_seq + 1u + lane < s.n ? s.starts[first_seq + 1u + lane] : 0x7fffffff;
        uint32_t k = 0;
#pragma unroll
        for (uint32_t x = 32; x; x >>= 1) k += __shfl(begin, (int)(k + x - 1u)) <= (int32_t)mine ? x : 0u;
        lo += k;
        hi = k == 63u ? s.n : lo + 1u;
    }
    const bool has = lane < io.window && mine < s.rows && place_of(s, g, mine, lo, hi, p);
    const bool begins = has && ((p.pos & (g.tokens - 1u)) == 0 || p.pos == p.first || (s.starts && s.starts[p.seq] == (int32_t)mine));
    if constexpr (!WRITE) {
        /* rows without a place come out as zeros */
        for (uint64_t m = ballot(lane < io.window && mine < s.rows && !has); m; m &= m - 1)
            for (uint32_t d = lane; d < g.dim; d += 64u) {
                ((uint16_t*)io.k)[(int64_t)(first_row + first_lane(m)) * io.k_row + (int64_t)head * io.k_head + d] = 0;
                ((uint16_t*)io.v)[(int64_t)(first_row + first_lane(m)) * io.v_row + (int64_t)head * io.v_head + d] = 0;
            }
    }
    uint64_t its_page = 0;                       /* where a lane's run begins */
    const bool is_there = begins && page_of_block(g, s, p.seq, p.pos >> g.tokens_log, head, its_page);
    const uint64_t theres = ballot(is_there);
    for (uint64_t m = ballot(begins); m; m &= m - 1) {
        const uint32_t j = first_lane(m), pos = bcast(p.pos, j), rest = bcast(p.rest, j), row = (uint32_t)first_row + j;
        const uint64_t page = bcast(its_page, j);
        const bool there = (theres >> j) & 1u;
        uint8_t* const powers = g.scales + (page - g.first_page) * g.tokens;      /* of the block's keys, and of its values behind them (only used where the block is there) */
        const uint32_t run_first = pos & (g.tokens - 1u), block_first = pos - run_first, run_end = rest < g.tokens - run_first ? run_first + rest : g.tokens;
        const uint32_t groups = io.piece / 8u, pairs = g.dim / 2u;
        /* a piece: `cnt` tokens from `in_block` of the block on; `none`: rows out are `fill` in place of keys (1), of values (2) */
        auto use_piece = [&](uint8_t* const keys, uint8_t* const values, const uint32_t none, const uint32_t fill, const uint32_t in_block, const uint32_t cnt) {
            const uint32_t off = in_block - run_first;
            uint16_t* const k_rows = (uint16_t*)io.k + (int64_t)(row + off) * io.k_row + (int64_t)head * io.k_head;
            uint16_t* const v_rows = (uint16_t*)io.v + (int64_t)(row + off) * io.v_row + (int64_t)head * io.v_head;
            /* of the values, a lane takes numbers d and d + 1 of the eight tokens from `tok` on, counted from the piece's first row */
            const int32_t piece_first = (int32_t)(in_block & (io.piece - 1u));
            /* what is worked out from the lane's number is worked out here, not kept across the miss path */
            uint32_t l = lane;
            asm volatile("" : "+v"(l));
            if (keys || (none & 1u)) {
                u32x4 x[TRIPS];
                const uint32_t r0 = l / LPR;
                /* in 8 bits the lane has one half of a piece */
                uint8_t* const at = E8 ? keys + (uint64_t)(col / 16u) * g.tokens * 16u + (col & 8u) : keys + (uint64_t)(col / 8u) * g.tokens * 16u;
#pragma unroll
                for (uint32_t e = 0; e < TRIPS; e++) {
                    const uint32_t r = r0 + e * RPW < cnt ? r0 + e * RPW : 0u;
                    if constexpr (WRITE) x[e] = load_piece<ALIGNED>(k_rows + (int64_t)r * io.k_row + col);
                    else if (none & 1u) x[e] = u32x4{fill, fill, fill, fill};
                    else if constexpr (E8) {
                        const uint64_t y = ld_payload((const uint64_t*)(at + place_in(g, in_block + r) * 16u));
                        const float by = scale_of(powers[in_block + r]);
                        x[e] = u32x4{from8<F16, false>((uint32_t)y, by), from8<F16, true>((uint32_t)y, by), from8<F16, false>((uint32_t)(y >> 32), by), from8<F16, true>((uint32_t)(y >> 32), by)};
                    } else x[e] = ld_payload((const u32x4*)(at + place_in(g, in_block + r) * 16u));
                }
                u32x4 w{0, 0, 0, 0};
                if (WRITE && io.k_norm) w = load_piece<true>(io.k_norm + col);
#pragma unroll
                for (uint32_t e = 0; e < TRIPS; e++) {
                    if (e * RPW >= cnt) break;
                    const uint32_t r = r0 + e * RPW;
                    if constexpr (WRITE) {
                        const kv_turn t = turn_of(io, piece, pos + off + (r < cnt ? r : 0u));
                        if constexpr (E8) {
                            float f[8];
                            const uint32_t down = norm_and_rotate_for_8<LPR, F16>(io, g.dim, in_row ? x[e] : u32x4{0, 0, 0, 0}, f, io.k_norm != nullptr, w, t, piece);
                            const uint32_t power = power_of_row<LPR, F16>(f, down);
                            const float by = inverse_of(power - down), most = MOST_KEPT<F16> * inverse_of(127u + down);
                            const uint32_t lo = to8<F16, true>(to8<F16, false>(0, f[0], f[1], by, most), f[2], f[3], by, most), hi = to8<F16, true>(to8<F16, false>(0, f[4], f[5], by, most), f[6], f[7], by, most);
                            if (r < cnt && in_row) {
                                __hip_atomic_store((uint64_t*)(at + place_in(g, in_block + r) * 16u), (uint64_t)hi << 32 | lo, __ATOMIC_RELAXED, BAM_SYSTEM);
                                if (piece == 0) powers[in_block + r] = (uint8_t)power;
                            }
                        } else {
                            x[e] = norm_and_rotate<LPR, F16>(io, g, in_row ? x[e] : u32x4{0, 0, 0, 0}, io.k_norm != nullptr, w, t, piece);
                            if (r < cnt && in_row) st16_sys(at + place_in(g, in_block + r) * 16u, x[e]);
                        }
                    } else if (r < cnt && in_row) *(u32x4*)(k_rows + (int64_t)r * io.k_row + col) = x[e];
                }
            }
            if (values || (none & 2u)) {
                /* in 8 bits: the powers of two of the rows first, those of the sixteen tokens that the piece is of */
                [[maybe_unused]] uint32_t power[16];
                if constexpr (E8 && WRITE) {
#pragma unroll
                    for (uint32_t e = 0; e < TRIPS; e++) {
                        const int32_t r = (int32_t)(l / LPR + e * RPW) - piece_first;
                        const bool mine = r >= 0 && r < (int32_t)cnt;
                        float f[8];
                        in_32_bits<F16>(load_piece<ALIGNED>(v_rows + (int64_t)(mine ? r : 0) * io.v_row + col), f);
                        const uint32_t x = power_of_row<LPR, F16>(f);
                        if (mine && piece == 0) powers[g.tokens + in_block + r] = (uint8_t)x;
#pragma unroll
                        for (uint32_t i = 0; i < RPW; i++) power[e * RPW + i] = (uint32_t)__builtin_amdgcn_readlane((int)x, (int)(i * LPR));
                    }
                }
#pragma unroll
                for (uint32_t e = 0; e < DT; e++) {
                    const uint32_t y = e * 64u + l, group = y / pairs, d = y % pairs * 2u;
                    const int32_t tok = (int32_t)(group * 8u) - piece_first;
                    if (group >= groups || tok + 8 <= 0 || tok >= (int32_t)cnt) continue;
                    uint8_t* const at = E8 ? values + ((uint64_t)((in_block + tok) >> 3) * pairs + d / 2u) * 16u : values + ((uint64_t)((in_block + tok) >> 3) * g.dim + d) * 16u;
                    uint16_t* const rows = v_rows + d;
                    const bool full = tok >= 0 && tok + 8 <= (int32_t)cnt;
                    if constexpr (WRITE) {
                        uint32_t z[8];
#pragma unroll
                        for (int32_t t = 0; t < 8; t++) {
                            const int32_t r = tok + t < 0 ? 0 : tok + t < (int32_t)cnt ? tok + t : (int32_t)cnt - 1;
                            const uint16_t* const from = rows + r * io.v_row;
                            z[t] = ALIGNED ? *(const uint32_t*)from : (uint32_t)from[0] | ((uint32_t)from[1] << 16);
                        }
                        if constexpr (E8) {
                            u32x4 y;
#pragma unroll
                            for (int t = 0; t < 4; t++) {
                                const uint32_t a = z[2 * t], b = z[2 * t + 1];
                                const uint32_t w = to8<F16, false>(0, from16<F16>(a & 0xffffu), from16<F16>(a >> 16), inverse_of(group ? power[8 + 2 * t] : power[2 * t]));
                                y[t] = to8<F16, true>(w, from16<F16>(b & 0xffffu), from16<F16>(b >> 16), inverse_of(group ? power[8 + 2 * t + 1] : power[2 * t + 1]));
                            }
                            if (full) st16_sys(at, y);
                            else {
#pragma unroll
                                for (int32_t t = 0; t < 8; t++) {
                                    const uint32_t w = y[t / 2];
                                    if (tok + t >= 0 && tok + t < (int32_t)cnt) __hip_atomic_store((uint16_t*)at + t, (uint16_t)(t & 1 ? w >> 16 : w), __ATOMIC_RELAXED, BAM_SYSTEM);
                                }
                            }
                        } else if (full) {
                            u32x4 lo, hi;
#pragma unroll
                            for (int t = 0; t < 4; t++) {
                                lo[t] = (z[2 * t] & 0xffffu) | (z[2 * t + 1] << 16);
                                hi[t] = (z[2 * t] >> 16) | (z[2 * t + 1] & 0xffff0000u);
                            }
                            st16_sys(at, lo);
                            st16_sys(at + 16, hi);
                        } else {
#pragma unroll
                            for (int32_t t = 0; t < 8; t++)
                                if (tok + t >= 0 && tok + t < (int32_t)cnt) {
                                    __hip_atomic_store((uint16_t*)at + t, (uint16_t)z[t], __ATOMIC_RELAXED, BAM_SYSTEM);
                                    __hip_atomic_store((uint16_t*)at + 8 + t, (uint16_t)(z[t] >> 16), __ATOMIC_RELAXED, BAM_SYSTEM);
                                }
                        }
                    } else if constexpr (E8) {
                        u32x4 y{0, 0, 0, 0};
                        uint64_t by = 0;
                        if (!(none & 2u)) {
                            y = ld_payload((const u32x4*)at);
                            by = *(const uint64_t*)(powers + g.tokens + in_block + tok);
                        }
#pragma unroll
                        for (int32_t t = 0; t < 8; t++) {
                            const float scale = scale_of((uint32_t)(by >> (8 * t)) & 0xffu);
                            const uint32_t w = y[t / 2];
                            const uint32_t x = none & 2u ? fill : t & 1 ? from8<F16, true>(w, scale) : from8<F16, false>(w, scale);
                            if (full || (tok + t >= 0 && tok + t < (int32_t)cnt)) *(uint32_t*)(rows + (tok + t) * io.v_row) = x;
                        }
                    } else {
                        u32x4 lo{fill, fill, fill, fill}, hi = lo;
                        if (!(none & 2u)) { lo = ld_payload((const u32x4*)at); hi = ld_payload((const u32x4*)(at + 16)); }
#pragma unroll
                        for (int32_t t = 0; t < 8; t++)
                            if (full || (tok + t >= 0 && tok + t < (int32_t)cnt)) {
                                const uint32_t a = lo[t / 2], b = hi[t / 2];
                                *(uint32_t*)(rows + (tok + t) * io.v_row) = (t & 1) ? (a >> 16) | (b & 0xffff0000u) : (a & 0xffffu) | (b << 16);
                            }
                    }
                }
            }
        };
        auto use = [&](uint8_t* const keys, uint8_t* const values, const uint32_t none, const uint32_t fill) {
            for (uint32_t at = run_first; at < run_end;) {
                uint32_t end = (at | (io.piece - 1u)) + 1u;
                if (end > run_end) end = run_end;
                use_piece(keys, values, none, fill, at, end - at);
                at = end;
            }
        };
        uint32_t none = 3;                       /* rows without a block read as zeros, */
        if (there) {
            /* a page whose first token is one of this call's holds nothing in front of them, and what was behind them is not kept: it needs nothing from the store */
            none = visit<WRITE>(g, page, WRITE && block_first >= bcast(p.first, j), WRITE && block_first + g.tokens > pos + rest, [&](uint8_t* keys, uint8_t* values) { use(keys, values, 0, 0); });
        }
        /* those whose page could not be had as NaN */
        if constexpr (!WRITE) if (__builtin_expect(none != 0, 0)) use(nullptr, nullptr, none, !there ? 0u : F16 ? 0x7e007e00u : 0x7fc07fc0u);
    }
}

template <int E8, bool WRITE>
void launch_rows(const bam_kv_t* kv, const kv_seqs& s, kv_rows io, hipStream_t st)
{
    const uint32_t lpr = kv->g.dim <= 64 ? 8 : kv->g.dim <= 128 ? 16 : 32, rpw = 64 / lpr;
    /* few rows: a trip of heads to a wave, a row to a wave; many: eight trips, and the runs that begin among sixteen rows */
    io.q_heads_each = io.q && (uint64_t)s.rows * io.q_heads > 16384 ? 8 * rpw : rpw;
    io.q_waves = io.q ? (uint32_t)((io.q_heads + io.q_heads_each - 1) / io.q_heads_each * s.rows) : 0;
    io.piece = kv->g.tokens < 16 ? 8 : 16;
    io.of_dim = 1.0 / kv->g.dim;
    /*
     * A wave goes through the runs of its window one after the other: no larger than leaves a wave to each place of the device.  Rows of the last blocks of 512 sequences, 1 to 31 tokens each and eight
     * heads, windows of 32 / 16 / 8 / 4 rows: 52 / 51 / 44 / 50 us; 13 rows of four sequences, 32 / 1: 16 / 8.5.
     */
    const uint32_t rows_each = s.starts ? s.rows / s.n : 0;
    io.window = rows_each >= 8 ? (kv->g.tokens < 64 ? kv->g.tokens : 64) : rows_each >= 4 ? 4 : rows_each >= 2 ? 2 : 1;
    while (io.window > 1 && (uint64_t)s.rows / io.window * kv->g.heads < 4096) io.window /= 2;
    /*
     * Windows that are smaller than runs: by heads.  In the order of the rows, the heads of those in which a run begins would lie side by side in a few workgroups, and those on the same compute
     * units.  512 sequences of 4 new rows, eight heads, a wave to a row: in the order of the rows 41 us, by heads 19; (four rows to a wave 12.5); 100 of 16, two rows to a wave, 27 and 14.
     */
    io.by_head = io.window < (rows_each < kv->g.tokens ? rows_each : kv->g.tokens);
    const uint64_t kv_waves = (uint64_t)((s.rows + io.window - 1) / io.window) * kv->g.heads;
    if (io.q_waves + kv_waves > 0x7fffffffull) throw std::runtime_error("more rows of heads than one launch takes");
    io.kv_blocks = (uint32_t)((kv_waves + 3) / 4);
    const dim3 grid(io.kv_blocks + (io.q_waves + 3) / 4), block(256);
    /*
     * Few rows: keys and values first, whose waves work longest.  Many: their workgroups among the queries', not behind them, where they would be left to finish alone, but what is written last is what
     * the caches have for who reads it next.  19 459 rows of 32 heads on 8 of 128 numbers into the cache and out again, keys and values first / over three quarters of the launch / evenly / last: in 8 bits
     * 119 + 52 / 123 + 43 / 134 + 40 / 134 + 37 us, in 16 bits 119 + 65 / 117 + 61 / 118 + 55 / 130 + 47; one row in 8 bits 8.4 + 5 / - / 9.1 + 5 (8 bits with sums in 32, which take 6 us less).
     */
    io.among = io.kv_blocks;
    const uint32_t most = E8 ? grid.x / 4 * 3 : grid.x;
    if (grid.x > 1024 && io.among < most) io.among = most;
#define KV_ROWS(LPR, AL) \
    if (kv->f16) hipLaunchKernelGGL((k_kv_rows<LPR, 1, E8, WRITE, AL>), grid, block, 0, st, kv->g, s, io); \
    else hipLaunchKernelGGL((k_kv_rows<LPR, 0, E8, WRITE, AL>), grid, block, 0, st, kv->g, s, io)
    if (WRITE && !io.aligned) { if (lpr == 8) { KV_ROWS(8, !WRITE); } else if (lpr == 16) { KV_ROWS(16, !WRITE); } else { KV_ROWS(32, !WRITE); } }
    else if (lpr == 8) { KV_ROWS(8, true); } else if (lpr == 16) { KV_ROWS(16, true); } else { KV_ROWS(32, true); }
#undef KV_ROWS
}

} // namespace
#endif /* __BAM_KV_CACHE_H__ */
