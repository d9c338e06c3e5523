// Beam search's selection, of the C-ABI: from the logits of a request's beams, the continuations with the largest sums of log-probabilities.
//
// For beam i with sum s_i and logits x_i the continuation with token v has s_i + x_i[v] - log sum_u exp x_i[u]; of all of a request's beams and tokens the `width` largest are
// wanted, in order, equal ones by i * vocab + v.  Within a beam the order is that of the logits, so one pass over them finds both what the softmax needs and the beam's best.
// The first kernel has a workgroup for a piece of a beam's logits and leaves the piece's `width` best tokens and its part of the sum of exponentials; the second joins
// the pieces and picks among the beams.
#include "bam_capi_internal.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

/* the most that are wanted, and beams; places for candidates of a workgroup */
constexpr uint32_t BEAM_WIDTH = 256, BEAM_BEAMS = 1024, BEAM_ROOM = 2048;
constexpr uint32_t BEAM_THREADS = 256, BEAM_NOTED = 256;      /* BEAM_NOTED: loads that are kept in LDS */
/* the most candidates of a request: a piece to a beam, or several (plan_of) */
constexpr uint32_t BEAM_CANDIDATES = BEAM_BEAMS * BEAM_WIDTH, BEAM_CANDIDATES_OF_PIECES = 8192;
static_assert(BEAM_CANDIDATES < 1u << 22 && BEAM_CANDIDATES_OF_PIECES <= BEAM_CANDIDATES, "k_beam_join divides their numbers in 32-bit floating point");
constexpr float LOG2E = 1.4426950408889634f;

struct beam_args {
    const void* logits;
    int64_t row;
    const float* scores;                /* [requests][beams] */
    int64_t score_row;
    uint32_t requests, beams, vocab, width, splits, per;      /* per: tokens of a split */
    float* sums;
    int32_t *from, *token;              /* [requests][width] each */
    uint64_t* best;                     /* [row][split][width] keys */
    double* part_s;                     /* [row][split]: the sum of exp(x - part_m), part_m the largest */
    float* part_m;
};

/* -0 as 0, minus infinity above NaN (1) and what is not there (0): in the order of the numbers */
__device__ __forceinline__ uint32_t ordered(const float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return x != x ? 1u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float number_of(const uint32_t o)
{
    return o < 2u ? __builtin_nanf("") : __builtin_bit_cast(float, o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint64_t ordered(const double x)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
    return x != x ? 1ull : b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double number_of(const uint64_t o)
{
    return o < 2ull ? __builtin_nan("") : __builtin_bit_cast(double, o & 0x8000000000000000ull ? o ^ 0x8000000000000000ull : ~o);
}
/* a logit and its token as one number: the larger logit first, of equal ones the lower token */
__device__ __forceinline__ uint64_t key_of(const float x, const uint32_t token) { return (uint64_t)ordered(x) << 32 | (uint32_t)~token; }

template <int TYPE> __device__ __forceinline__ float number_in(const u32x4 v, const uint32_t e)
{
    if constexpr (TYPE == 2) { const uint32_t y = v[e]; return __builtin_bit_cast(float, y); }
    const uint32_t y = v[e / 2];
    if constexpr (TYPE == 0) return __builtin_bit_cast(float, e & 1u ? y & 0xffff0000u : y << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(e & 1u ? y >> 16 : y));
}
template <int TYPE> __device__ __forceinline__ float number_at(const void* x, const uint64_t i)
{
    if constexpr (TYPE == 2) return ((const float*)x)[i];
    const uint32_t y = ((const uint16_t*)x)[i];
    if constexpr (TYPE == 0) return __builtin_bit_cast(float, y << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)y);
}
template <int TYPE> constexpr uint32_t NOTHING = TYPE == 0 ? 0xff80ff80u : TYPE == 1 ? 0xfc00fc00u : 0xff800000u;      /* minus infinity */

__device__ __forceinline__ uint64_t larger(const uint64_t a, const uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t low(const uint64_t x) { return (uint32_t)x; }
__device__ __forceinline__ uint32_t high(const uint64_t x) { return (uint32_t)(x >> 32); }
__device__ __forceinline__ uint64_t both(const uint32_t hi, const uint32_t lo) { return (uint64_t)hi << 32 | lo; }
/* f over the lanes of a wave, or of each four (STEPS 2), without LDS: lanes 1 and 2 apart, halves of eight, of sixteen, rows of sixteen, halves of the wave; every lane has the result */
template <int STEPS, typename F> __device__ __forceinline__ uint64_t over_lanes(uint64_t x, F&& f)
{
#define BEAM_DPP(CTRL) f(x, both((uint32_t)__builtin_amdgcn_update_dpp(0, (int)high(x), CTRL, 0xf, 0xf, true), (uint32_t)__builtin_amdgcn_update_dpp(0, (int)low(x), CTRL, 0xf, 0xf, true)))
    x = BEAM_DPP(0xb1);
    x = BEAM_DPP(0x4e);
    if constexpr (STEPS > 2) {
        x = BEAM_DPP(0x141);
        x = BEAM_DPP(0x140);
        {
            const auto l = __builtin_amdgcn_permlane16_swap(low(x), low(x), false, false), h = __builtin_amdgcn_permlane16_swap(high(x), high(x), false, false);
            const uint32_t l0 = l[0], l1 = l[1], h0 = h[0], h1 = h[1];
            x = f(both(h0, l0), both(h1, l1));
        }
        {
            const auto l = __builtin_amdgcn_permlane32_swap(low(x), low(x), false, false), h = __builtin_amdgcn_permlane32_swap(high(x), high(x), false, false);
            const uint32_t l0 = l[0], l1 = l[1], h0 = h[0], h1 = h[1];
            x = f(both(h0, l0), both(h1, l1));
        }
    }
#undef BEAM_DPP
    return x;
}
/* sums of numbers in 64 bits, the largest of numbers in 32 (NaN where there is one), over a wave */
__device__ __forceinline__ double sum_over_lanes(const double x)
{
    return __builtin_bit_cast(double, over_lanes<6>(__builtin_bit_cast(uint64_t, x), [](const uint64_t a, const uint64_t b) { return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b)); }));
}
__device__ __forceinline__ float most_over_lanes(const float x)
{
    return __builtin_bit_cast(float, (uint32_t)over_lanes<6>(__builtin_bit_cast(uint32_t, x), [](const uint64_t a, const uint64_t b) { return (uint64_t)__builtin_bit_cast(uint32_t, __builtin_elementwise_maximum(__builtin_bit_cast(float, low(a)), __builtin_bit_cast(float, low(b)))); }));
}
/* places in a list in LDS for the lanes that have something for it: one addition by the wave */
__device__ __forceinline__ uint32_t place_for(const bool has, uint32_t* const n)
{
    const uint64_t mask = bam::ballot(has);
    if (!mask) return 0;
    uint32_t base = 0;
    if (bam::lane() == 0) base = atomicAdd(n, bam::popc(mask));
    return bam::first(base) + __builtin_amdgcn_mbcnt_hi(high(mask), __builtin_amdgcn_mbcnt_lo(low(mask), 0));
}

/*
 * A bound for the `width`-th largest of many keys: the `width`-th largest among the largest keys of groups of threads, 64 groups for up to 32 that are wanted, else 256.  It is no more than the
 * `width`-th largest of all, and where the keys are spread over the threads not much less.  `none` where there are not that many.  `mine`: the largest of a group's keys.
 */
template <typename K, typename BEFORE>
__device__ __forceinline__ K bound_of(const K mine, const uint32_t group, const bool leads, const uint32_t width, K* const tops, K* const at, const K none, BEFORE&& comes_before)
{
    const uint32_t t = threadIdx.x, groups = width <= 32u ? 64u : 256u;
    if (leads) tops[group] = mine;
    if (t == 0) *at = none;
    __syncthreads();
    if (t < groups) {
        const K its = tops[t];
        uint32_t above = 0;
#pragma unroll 16
        for (uint32_t i = 0; i < groups; i++) above += comes_before(tops[i], its) ? 1u : 0u;
        if (comes_before(its, none) && above == width - 1u) *at = its;
    }
    __syncthreads();
    return *at;
}
__device__ __forceinline__ uint64_t bound_of_keys(uint64_t mine, const uint32_t width, uint64_t* const tops, uint64_t* const at)
{
    const bool four = width <= 32u;
    if (four) mine = over_lanes<2>(mine, larger);
    return bound_of(mine, four ? threadIdx.x / 4u : threadIdx.x, !four || threadIdx.x % 4u == 0, width, tops, at, (uint64_t)0, [](const uint64_t a, const uint64_t b) { return a > b; });
}

/*
 * A piece of a beam's logits, in chunks of LOADS * 4 KiB.  What is wanted of a chunk is not sorted out of it: few more than `width` of its numbers are not below the bound of the threads' largest
 * (bound_of).  The loads that have such numbers are put in LDS, and looked at again by as many threads; what is found goes into `room`.  For the chunks behind the first the same bound holds.  Where
 * the candidates do not fit (numbers in an order that gives a few threads all the large ones), those that did give a higher bound.  The next chunk is on its way meanwhile.
 * Exponentials are of differences to the thread's largest so far (differences first: the type's lowest value times log2 e is out of range); LOADS * 4 or 8 of them are added up in 32 bits, the rest in 64.
 *   Many rows: bound by memory, 768 of 150001 in float32 94 us (4.9 TB/s, what a copy reaches; 104 with loads that are kept in the caches); 128 of 128000 in bfloat16 14 us, two thirds of it the launch and the
 * latencies of the first loads, the bound and the last list.  Few: latencies, 5.6 us for 4 rows of 32000.
 */
template <int TYPE, uint32_t LOADS>
__global__ __launch_bounds__(BEAM_THREADS, 4) void k_beam_rows(const beam_args a)
{
    using namespace bam;
    constexpr uint32_t VEC = TYPE == 2 ? 4 : 8, SIZE = TYPE == 2 ? 4 : 2, CHUNK = BEAM_THREADS * LOADS * VEC;
    __shared__ uint64_t room[BEAM_ROOM + 8], tops[BEAM_THREADS], bound_at;
    __shared__ u32x4 noted[BEAM_NOTED];
    __shared__ uint16_t noted_at[BEAM_THREADS * LOADS];
    __shared__ uint32_t n_room, n_noted[2];
    __shared__ double wave_s[4];
    __shared__ float wave_m[4];
    const uint32_t t = threadIdx.x, lane = bam::lane(), wave = first(t / 64u);
    const uint32_t row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const uint32_t begin = split * a.per < a.vocab ? split * a.per : a.vocab, end = a.vocab - begin < a.per ? a.vocab : begin + a.per;
    const uint8_t* const x = (const uint8_t*)a.logits + (int64_t)row * a.row * SIZE;
    const uint32_t whole = begin + (end - begin) / VEC * VEC;       /* up to here in loads of 16 bytes; the rest, less than that, one by one */
    uint64_t bound = 0;
    double s = 0;
    float m = -INFINITY;
    if (t == 0) n_room = n_noted[0] = n_noted[1] = 0;
    u32x4 raw[LOADS];
    auto load = [&](const uint32_t c) {
        const uint8_t* const at = x + (uint64_t)(c + t * VEC) * SIZE;
        if (c + CHUNK <= whole) {
#pragma unroll
            for (uint32_t j = 0; j < LOADS; j++) raw[j] = __builtin_nontemporal_load((const u32x4_any*)(at + j * BEAM_THREADS * 16u));
        } else {
#pragma unroll
            for (uint32_t j = 0; j < LOADS; j++) {
                raw[j] = u32x4{NOTHING<TYPE>, NOTHING<TYPE>, NOTHING<TYPE>, NOTHING<TYPE>};
                if (c + (j * BEAM_THREADS + t) * VEC < whole) raw[j] = __builtin_nontemporal_load((const u32x4_any*)(at + j * BEAM_THREADS * 16u));
            }
        }
    };
    load(begin);
    uint32_t here = 0, turn = 0;                     /* here: n_room, as all threads know it */
#pragma unroll 1
    for (uint32_t c = begin; c < end; c += CHUNK, turn ^= 1u) {
        float tops_of[LOADS];                        /* NaN where there is one: such a beam's tokens are picked by their numbers (k_beam_join) */
        float rest = -INFINITY;
        uint32_t rest_at = 0xffffffffu;
        if (end - c <= CHUNK && t < end - whole) { rest_at = whole + t; rest = number_at<TYPE>(x, rest_at); }
        float top = rest;
        uint32_t top_at = rest_at;                   /* no token of the thread with that number comes behind this one of its load */
#pragma unroll
        for (uint32_t j = LOADS; j-- > 0;) {
            float y = number_in<TYPE>(raw[j], 0);
#pragma unroll
            for (uint32_t e = 1; e < VEC; e++) y = __builtin_elementwise_maximum(y, number_in<TYPE>(raw[j], e));
            const uint32_t i = c + (j * BEAM_THREADS + t) * VEC;
            if (i >= whole) y = -INFINITY;
            tops_of[j] = y;
            if (i < whole && !(y < top)) { top = y; top_at = i + VEC - 1u; }
        }
        const float larger_m = __builtin_elementwise_maximum(m, top), use = larger_m == -INFINITY ? 0.0f : larger_m;
        float sum[4] = {__builtin_amdgcn_exp2f((rest - use) * LOG2E), 0, 0, 0};
#pragma unroll
        for (uint32_t j = 0; j < LOADS; j++)
#pragma unroll
            for (uint32_t e = 0; e < VEC; e++) sum[e & 3u] += __builtin_amdgcn_exp2f((number_in<TYPE>(raw[j], e) - use) * LOG2E);
        float both_sums = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        asm volatile("" : "+v"(both_sums));          /* (here, and not behind the next chunk's loads, which would take other registers) */
        s = s * (double)__builtin_amdgcn_exp2f((m - use) * LOG2E) + (double)both_sums;
        m = larger_m;
        if (c == begin) bound = bound_of_keys(top_at == 0xffffffffu ? 0ull : key_of(top, top_at), a.width, tops, &bound_at);
        {
            /* the wave's loads with such numbers */
            uint64_t masks[LOADS];
            uint32_t n = 0;
#pragma unroll
            for (uint32_t j = 0; j < LOADS; j++) {
                const uint32_t i = c + (j * BEAM_THREADS + t) * VEC;
                masks[j] = ballot(i < whole && key_of(tops_of[j], i) >= bound);
                n += popc(masks[j]);
            }
            if (n) {
                uint32_t base = 0;
                if (lane == 0) base = atomicAdd(&n_noted[turn], n);
                base = first(base);
#pragma unroll
                for (uint32_t j = 0; j < LOADS; j++) {
                    if (!masks[j]) continue;
                    const uint32_t at = base + __builtin_amdgcn_mbcnt_hi(high(masks[j]), __builtin_amdgcn_mbcnt_lo(low(masks[j]), 0));
                    if (masks[j] >> lane & 1u) {
                        noted_at[at] = (uint16_t)(j * BEAM_THREADS + t);
                        if (at < BEAM_NOTED) noted[at] = raw[j];
                    }
                    base += popc(masks[j]);
                }
            }
        }
        if (end - c > CHUNK) load(c + CHUNK);
        __syncthreads();
        const uint32_t n_loads = n_noted[turn];
        if (t == 0) n_noted[turn ^ 1u] = 0;
        auto put = [&](const uint64_t k, const bool is) {
            const bool has = is && k >= bound;
            const uint32_t at = place_for(has, &n_room);
            if (has && at < BEAM_ROOM) room[at] = k;
        };
        uint32_t n;
        for (;;) {
#pragma unroll 1
            for (uint32_t q0 = wave * 64u; q0 < n_loads; q0 += BEAM_THREADS) {
                const bool is = q0 + lane < n_loads;
                const uint32_t q = is ? q0 + lane : 0u, i = c + noted_at[q] * VEC;
                u32x4 z;
                if (n_loads <= BEAM_NOTED) z = noted[q];
                else {
                    z = *(const u32x4_any*)(x + (uint64_t)i * SIZE);
                    asm volatile("" : "+v"(z));      /* waited for here, or the other way would wait for the next chunk too */
                }
#pragma unroll
                for (uint32_t e = 0; e < VEC; e++) put(key_of(number_in<TYPE>(z, e), i + e), is);
            }
            if (end - c <= CHUNK && whole != end && wave == 0) put(key_of(rest, rest_at), rest_at != 0xffffffffu);
            __syncthreads();
            n = n_room;                              /* (who adds to it next has passed another barrier) */
            const bool again = n > BEAM_ROOM;
            if (!again && (n <= BEAM_ROOM / 2 || end - c <= CHUNK)) break;
            /* what is there gives a higher bound (of the keys in the room, spread over the threads as they came, at most a group's largest ones are left), and what is below it goes; of a chunk that
             * did not fit, everything, and it is gone through again */
            const uint32_t have = again ? BEAM_ROOM : n, keep = again ? here : n;
            uint64_t most = 0;
#pragma unroll 1
            for (uint32_t j = t; j < have; j += BEAM_THREADS) most = larger(most, room[j]);
            bound = larger(bound, bound_of_keys(most, a.width, tops, &bound_at));
            uint64_t mine[BEAM_ROOM / BEAM_THREADS];
#pragma unroll
            for (uint32_t j = 0; j < BEAM_ROOM / BEAM_THREADS; j++) mine[j] = j * BEAM_THREADS + t < keep ? room[j * BEAM_THREADS + t] : 0ull;
            if (t == 0) n_room = 0;
            __syncthreads();
#pragma unroll
            for (uint32_t j = 0; j < BEAM_ROOM / BEAM_THREADS; j++) put(mine[j], mine[j] != 0);
            __syncthreads();
            n = here = n_room;
            if (!again) break;
            __syncthreads();                         /* all have read it */
        }
        here = n;
    }
    const uint32_t n = here;
    const uint64_t to = ((uint64_t)row * a.splits + split) * a.width;
    /* the parts of the sum of exponentials */
    const float wave_top = most_over_lanes(m);
    s = sum_over_lanes(s * (double)__builtin_amdgcn_exp2f((m - (wave_top == -INFINITY ? 0.0f : wave_top)) * LOG2E));
    if (lane == 0) { wave_s[wave] = s; wave_m[wave] = wave_top; }
    if (t < 8) room[n + t] = 0;                      /* (read below, eight at a time) */
    __syncthreads();
#pragma unroll 1
    for (uint32_t j = t; j < n; j += BEAM_THREADS) {
        const uint64_t mine = room[j];
        uint32_t above = 0;
#pragma unroll 1
        for (uint32_t i = 0; i < n; i += 8) {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) above += room[i + e] > mine ? 1u : 0u;
        }
        if (above < a.width) a.best[to + above] = mine;
    }
    for (uint32_t j = n + t; j < a.width; j += BEAM_THREADS) a.best[to + j] = 0;
    if (t == 0) {
        const float top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(wave_m[0], wave_m[1]), __builtin_elementwise_maximum(wave_m[2], wave_m[3])), use = top == -INFINITY ? 0.0f : top;
        double all = 0;
#pragma unroll
        for (uint32_t w = 0; w < 4; w++) all += wave_s[w] * (double)__builtin_amdgcn_exp2f((wave_m[w] - use) * LOG2E);
        a.part_s[(uint64_t)row * a.splits + split] = all;
        a.part_m[(uint64_t)row * a.splits + split] = top;
    }
}

/* a candidate: its sum in order, and beam and token, of which the lower come first; none is {0, all ones} */
struct beam_place { uint64_t sum, at; };
__device__ __forceinline__ bool before(const beam_place& a, const beam_place& b) { return a.sum > b.sum || (a.sum == b.sum && a.at < b.at); }
/*
 * log x in 64 bits: x = 2^n y, y from 3/4 to 3/2, log y = 2 artanh z, z = (y - 1) / (y + 1) within 1/5, by the series z + z^3/3 + ..., whose first term left out is less than 2^-33 of z.  (The
 * library's is three times as many instructions.)
 */
__device__ __forceinline__ double log_of(const double x)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const int32_t n = (int32_t)((b - 0x3fe8000000000000ull) >> 52) - (b < 0x3fe8000000000000ull ? 4096 : 0);
    const double y = __builtin_bit_cast(double, b - ((uint64_t)(int64_t)n << 52)), z = (y - 1) / (y + 1), w = z * z;
    double p = 1.0 / 13;
#pragma unroll
    for (int k = 11; k > 0; k -= 2) p = p * w + 1.0 / k;
    return !(x > 0) || x - x != 0 ? __builtin_nan("") : (double)n * 0.6931471805599453 + 2 * z * p;
}

/*
 * A request: the beams' logarithms of sums of exponentials, and the best of what the pieces left, by a bound as in k_beam_rows.  Sums are compared in 64 bits and not rounded to 32 before.  They are
 * as near as the exponentials under them, which k_beam_rows takes, and adds up by the chunk, in 32: within 2^-19.  Beams whose sums differ by more than twice that come in the right order; a beam's own
 * tokens, which have that error in common, where 64 bits tell them apart; and beams of the same differences and scores have the same sums.
 *   Up to eight candidates to a thread are in registers before the sums are known, and the first bound is of the upper halves of the sums, with candidate q of piece l in group q * (pieces | 1) + l: pieces'
 * candidates come in order, so neighbouring ones in one group would leave most groups without a good one (16 beams, 2048 candidates, 32 wanted: 55 us for 14).
 *   Latencies: 4.4 to 5 us for up to 1024 candidates, of which an empty kernel behind another takes 4; 6.9 for 2560 of 48 requests.
 */
template <uint32_t THREADS>
__global__ __launch_bounds__(THREADS) void k_beam_join(const beam_args a)
{
    using namespace bam;
    constexpr uint32_t WAVES = THREADS / 64u, EACH = BEAM_ROOM / THREADS, HELD = 8;
    __shared__ double offset[BEAM_BEAMS];            /* of a logit's difference to the beam's largest (which may be so far from zero that nothing else would be left) */
    __shared__ float largest[BEAM_BEAMS];
    __shared__ beam_place room[BEAM_ROOM + 8], tops[256], bound_at;
    __shared__ uint32_t n_room, halves[256], half_at, ranks[BEAM_ROOM];
    const uint32_t t = threadIdx.x, lane = bam::lane(), wave = first(t / 64u), request = blockIdx.x;
    const uint32_t each = a.splits * a.width, all = a.beams * each, pieces = a.beams * a.splits, groups = a.width <= 32u ? 64u : 256u;
    const uint64_t* const best = a.best + (uint64_t)request * all;
    const float of_each = 1.0f / (float)each, of_width = 1.0f / (float)a.width;
    uint64_t held[HELD];
#pragma unroll
    for (uint32_t h = 0; h < HELD; h++) held[h] = h * THREADS + t < all ? best[h * THREADS + t] : 0ull;
    if (t == 0) { n_room = 0; half_at = 0; }
    if (t < 256u) halves[t] = 0;
#pragma unroll 1
    for (uint32_t i = wave; i < a.beams; i += WAVES) {
        const uint64_t at = ((uint64_t)request * a.beams + i) * a.splits;
        const float score = a.scores[(int64_t)request * a.score_row + i];
        /* (splits are seldom more than lanes) */
        float top = lane < a.splits ? a.part_m[at + lane] : -INFINITY;
        double sum = lane < a.splits ? a.part_s[at + lane] : 0.0;
#pragma unroll 1
        for (uint32_t k = lane + 64u; k < a.splits; k += 64u) {
            const float its = a.part_m[at + k], more = __builtin_elementwise_maximum(top, its), use = more == -INFINITY ? 0.0f : more;
            sum = sum * (double)__builtin_amdgcn_exp2f((top - use) * LOG2E) + a.part_s[at + k] * (double)__builtin_amdgcn_exp2f((its - use) * LOG2E);
            top = more;
        }
        const float most = most_over_lanes(top);
        sum = sum_over_lanes(sum * (double)__builtin_amdgcn_exp2f((top - (most == -INFINITY ? 0.0f : most)) * LOG2E));
        const double by = (double)score - log_of(sum);
        if (lane == 0) { offset[i] = by; largest[i] = most; }
    }
    __syncthreads();
    /* candidate c; (numbers below 2^22 are divided exactly this way, and there are no more than BEAM_CANDIDATES) */
    auto beam_of = [&](const uint32_t c) { return (uint32_t)(((float)c + 0.5f) * of_each); };
    auto place_of = [&](const uint32_t c, const uint64_t k) {
        const uint32_t i = beam_of(c), j = c - i * each;
        const double by = offset[i];
        /* (a beam of which all tokens have the same, an infinity or NaN: by their numbers) */
        const bool finite = by - by == 0, is = finite ? k != 0 : j < a.width && j < a.vocab;
        return beam_place{!is ? 0ull : ordered(finite ? ((double)number_of(high(k)) - (double)largest[i]) + by : by), (uint64_t)i << 32 | (finite ? ~low(k) : j)};
    };
    const beam_place none = {0, ~0ull};
    beam_place bound = none, mine[EACH > HELD ? EACH : HELD];
    auto put = [&](const beam_place& p) {
        const bool has = p.sum && !before(bound, p);
        const uint32_t at = place_for(has, &n_room);
        if (has && at < BEAM_ROOM) room[at] = p;
    };
    const bool few = all <= HELD * THREADS;
    auto note = [&](const uint32_t c, const beam_place& p) {
        const uint32_t l = (uint32_t)(((float)c + 0.5f) * of_width);
        if (p.sum) atomicMax(&halves[((c - l * a.width) * (pieces | 1u) + l) & (groups - 1u)], high(p.sum));
    };
    if (few) {
#pragma unroll
        for (uint32_t h = 0; h < HELD; h++) {
            const uint32_t c = h * THREADS + t;
            mine[h] = c < all ? place_of(c, held[h]) : none;
            note(c, mine[h]);
        }
    } else {
#pragma unroll 1
        for (uint32_t c = t; c < all; c += THREADS) note(c, place_of(c, best[c]));
    }
    __syncthreads();
    if (t < groups) {
        const uint32_t its = halves[t];
        uint32_t above = 0, not_below = 0;
#pragma unroll 16
        for (uint32_t i = 0; i < groups; i++) { const uint32_t y = halves[i]; above += y > its ? 1u : 0u; not_below += y >= its ? 1u : 0u; }
        if (above < a.width && not_below >= a.width) half_at = its;      /* (by each of those that have the same) */
    }
    __syncthreads();
    bound = beam_place{both(half_at, 0), ~0ull};
    auto put_all = [&]() {
#pragma unroll 1
        for (uint32_t c0 = wave * 64u; c0 < all; c0 += THREADS) put(c0 + lane < all ? place_of(c0 + lane, best[c0 + lane]) : none);
    };
    if (few) {
#pragma unroll
        for (uint32_t h = 0; h < HELD; h++) if (h * THREADS < all) put(mine[h]);
    } else put_all();
    __syncthreads();
    uint32_t n = n_room;
    /* few are left, which can be put in order, each by looking at all; else what is there gives a higher bound, of all 128 bits */
#pragma unroll 1
    while (n > 2u * a.width + 64u) {
        const uint32_t was = n;
        beam_place top = none;
#pragma unroll
        for (uint32_t j = 0; j < EACH; j++) { mine[j] = j * THREADS + t < n ? room[j * THREADS + t] : none; if (before(mine[j], top)) top = mine[j]; }
        const uint32_t of = THREADS / groups;      /* groups of 16, 4 or single threads */
#pragma unroll 1
        for (uint32_t o = 1; o < of; o <<= 1) {
            const beam_place p = {both((uint32_t)__shfl_xor((int)high(top.sum), o), (uint32_t)__shfl_xor((int)low(top.sum), o)), both((uint32_t)__shfl_xor((int)high(top.at), o), (uint32_t)__shfl_xor((int)low(top.at), o))};
            if (before(p, top)) top = p;
        }
        const beam_place higher = bound_of(top, t / of, t % of == 0, a.width, tops, &bound_at, none, before);
        if (before(higher, bound)) bound = higher;
        if (t == 0) n_room = 0;
        __syncthreads();
        if (n > BEAM_ROOM) put_all();                /* not all of them were in the room */
        else {
#pragma unroll
            for (uint32_t j = 0; j < EACH; j++) if (j * THREADS < n) put(mine[j]);
        }
        __syncthreads();
        n = n_room;
        if (n <= BEAM_ROOM && n == was) break;
    }
    const uint64_t to = (uint64_t)request * a.width;
    if (t < 4) room[n + t] = none;                   /* (read below, four at a time) */
    for (uint32_t j = t; j < n; j += THREADS) ranks[j] = 0;
    __syncthreads();
    /* entries that are a power of two's worth, the threads that are more share what each is compared with */
    uint32_t m_log = 5;
    while ((1u << m_log) < n) m_log++;
    const uint32_t parts = (1u << m_log) < THREADS ? THREADS >> m_log : 1u, part = ((n + 3u) / 4u + parts - 1u) / parts * 4u;
#pragma unroll 1
    for (uint32_t j = t & ((1u << m_log) - 1u); j < n; j += THREADS) {
        const beam_place p = room[j];
        const uint32_t i0 = parts > 1u ? (t >> m_log) * part : 0u, i1 = i0 + part < n ? i0 + part : n;
        uint32_t above = 0;
#pragma unroll 1
        for (uint32_t i = i0; i < i1; i += 4) {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) above += before(room[i + e], p) ? 1u : 0u;
        }
        if (above) atomicAdd(&ranks[j], above);
    }
    __syncthreads();
#pragma unroll 1
    for (uint32_t j = t; j < n; j += THREADS) {
        const uint32_t above = ranks[j];
        if (above >= a.width) continue;
        const beam_place p = room[j];
        a.sums[to + above] = (float)number_of(p.sum);
        a.from[to + above] = (int32_t)(request * a.beams + (uint32_t)(p.at >> 32));
        a.token[to + above] = (int32_t)(uint32_t)p.at;
    }
}

struct beam_plan { uint32_t splits, per; uint64_t best_at, s_at, m_at, bytes; };
beam_plan plan_of(const uint64_t requests, const uint64_t beams, const uint64_t vocab, const uint32_t width, const int type)
{
    beam_plan p{};
    /*
     * A workgroup to each place of the device (four to a compute unit), with at least a load to each of its threads; with more rows than that, pieces of four chunks of eight loads.  But no more
     * candidates than the second launch holds in registers (8192 of a request), where that can be had.  Both launches, with 2 / 4 / 8 / 16 / 32 pieces to a row: 64 rows of 128000 in
     * bfloat16 25 / 18 / 16 / 15 / 20 us; 768 rows of 150001 in float32, 32 wanted, with 2 / 3 / 4 / 5 / 6 / 8: 139 / 121 / 112 / 106 / 113 / 126; 32 rows of one request, 160000, 64 wanted, with
     * 2 / 4 / 8 / 16: 53 / 34 / 40 / 53.
     */
    const uint64_t rows = requests * beams, load = BEAM_THREADS * (type == 2 ? 4 : 8);
    uint64_t splits = (1024 + rows - 1) / rows;
    if (splits < (vocab + 32 * load - 1) / (32 * load)) splits = (vocab + 32 * load - 1) / (32 * load);
    const uint64_t most = BEAM_CANDIDATES_OF_PIECES / (beams * width);
    if (splits > most) splits = most ? most : 1;
    if (splits > (vocab + load - 1) / load) splits = (vocab + load - 1) / load;
    p.per = (uint32_t)(((vocab + splits - 1) / splits + 15) / 16 * 16);
    p.splits = (uint32_t)((vocab + p.per - 1) / p.per);
    auto place = [&](uint64_t bytes) { const uint64_t at = p.bytes; p.bytes += (bytes + 255) & ~255ull; return at; };
    p.best_at = place(rows * p.splits * width * 8);
    p.s_at = place(rows * p.splits * 8);
    p.m_at = place(rows * p.splits * 4);
    return p;
}

int bad_sizes(const char* who, const uint64_t requests, const uint64_t beams, const uint64_t vocab, const uint32_t width, const int type)
{
    if (type < 0 || type > 2) return fail(EINVAL, std::string(who) + ": type must be 0 (bfloat16), 1 (float16) or 2 (float32)");
    if (!beams || !vocab || beams > BEAM_BEAMS) return fail(EINVAL, std::string(who) + ": there must be tokens, and 1 to 1024 beams");
    if (vocab > 0x7fffffffull / beams || requests > 0x7fffffffull / beams) return fail(EINVAL, std::string(who) + ": more beams or continuations than 31 bits count");
    if (!width || width > BEAM_WIDTH || width > beams * vocab) return fail(EINVAL, std::string(who) + ": width must be 1 to 256, and at most the number of continuations");
    return 0;
}

} // namespace

extern "C" {

int bam_beam_select_bytes(uint64_t n_requests, uint64_t n_beams, uint64_t vocab, uint32_t width, int type, uint64_t* bytes)
{
    if (!bytes) return fail(EINVAL, "bam_beam_select_bytes: null argument");
    if (int e = bad_sizes("bam_beam_select_bytes", n_requests, n_beams, vocab, width, type)) return e;
    *bytes = n_requests ? plan_of(n_requests, n_beams, vocab, width, type).bytes : 0;
    return 0;
}

int bam_beam_select(const bam_beam_select_t* what, void* stream)
{
    if (!what) return fail(EINVAL, "bam_beam_select: null argument");
    const bam_beam_select_t& w = *what;
    if (int e = bad_sizes("bam_beam_select", w.n_requests, w.n_beams, w.vocab, w.width, w.type)) return e;
    if (!w.n_requests) return 0;
    if (!w.d_logits || !w.d_scores || !w.d_sums || !w.d_beams || !w.d_tokens || !w.d_work) return fail(EINVAL, "bam_beam_select: null argument");
    if (((uintptr_t)w.d_work & 15) || ((uintptr_t)w.d_logits & (w.type == 2 ? 3 : 1))) return fail(EINVAL, "bam_beam_select: the workspace must be aligned to 16 bytes, logits to their size");
    BAM_API_BEGIN
    const beam_plan p = plan_of(w.n_requests, w.n_beams, w.vocab, w.width, w.type);
    if (w.work_bytes < p.bytes) return fail(EINVAL, "bam_beam_select: the workspace is smaller than bam_beam_select_bytes says");
    const uint64_t rows = w.n_requests * w.n_beams, all = w.n_beams * p.splits * w.width;
    if (rows * p.splits > 0x7fffffffull) return fail(EINVAL, "bam_beam_select: more workgroups than 31 bits count");
    beam_args a{};
    a.logits = w.d_logits; a.row = w.logits_row; a.scores = w.d_scores; a.score_row = w.scores_row;
    a.requests = (uint32_t)w.n_requests; a.beams = (uint32_t)w.n_beams; a.vocab = (uint32_t)w.vocab; a.width = w.width; a.splits = p.splits; a.per = p.per;
    a.sums = w.d_sums; a.from = w.d_beams; a.token = w.d_tokens;
    uint8_t* const at = (uint8_t*)w.d_work;
    a.best = (uint64_t*)(at + p.best_at); a.part_s = (double*)(at + p.s_at); a.part_m = (float*)(at + p.m_at);
    const dim3 grid((uint32_t)(rows * p.splits)), block(BEAM_THREADS);
    hipStream_t const st = (hipStream_t)stream;
#define BEAM_ROWS(LOADS) \
    if (w.type == 0) hipLaunchKernelGGL((k_beam_rows<0, LOADS>), grid, block, 0, st, a); \
    else if (w.type == 1) hipLaunchKernelGGL((k_beam_rows<1, LOADS>), grid, block, 0, st, a); \
    else hipLaunchKernelGGL((k_beam_rows<2, LOADS>), grid, block, 0, st, a)
    /*
     * Loads of a thread at a time: no more than a piece has, and four where that makes no more than two chunks.  1 / 4 / 8: 4 rows of 32000 in 16 pieces 5.7 / 6.3 / 7.3 us; 128 rows of 128000 in 8
     * pieces 25 / 13.8 / 14.7; 768 rows of 150001 in float32, in 5 pieces, - / 131 / 95.
     */
    const uint64_t load = BEAM_THREADS * (w.type == 2 ? 4 : 8);
    if (p.per <= load) { BEAM_ROWS(1); } else if (p.per <= 8 * load) { BEAM_ROWS(4); } else { BEAM_ROWS(8); }
#undef BEAM_ROWS
    if (all <= 1024) hipLaunchKernelGGL(k_beam_join<256>, dim3(a.requests), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_beam_join<1024>, dim3(a.requests), dim3(1024), 0, st, a);
    hip_err_chk(hipGetLastError());
    BAM_API_END
}

} // extern "C"
