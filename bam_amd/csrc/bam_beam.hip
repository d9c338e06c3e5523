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
constexpr uint32_t BEAM_THREADS = 256, BEAM_LOADS = 8;      /* loads of 16 bytes that a thread has on their way */
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
__device__ __forceinline__ uint64_t shfl_xor64(const uint64_t x, const int by)
{
    return (uint64_t)(uint32_t)__shfl_xor((int)(x >> 32), by) << 32 | (uint32_t)__shfl_xor((int)x, by);
}

/*
 * A piece of a beam's logits, in chunks of 32 KiB.  What is wanted of a chunk is not sorted out of it: the `width`-th largest among the threads' largest numbers (of four
 * threads each, up to 32 of them) is no more than the chunk's `width`-th largest, and not much less, so few more than `width` are not smaller.  The loads that have such numbers are noted in LDS, and
 * looked at again by as many threads; what is found goes into `room`.  For the chunks behind the first the same bound holds.  Where the candidates would not fit (numbers in an order that
 * gives a few threads all the large ones), the chunk's `width`-th largest is found by going down from the largest one by one.
 * Exponentials are of differences to the thread's largest so far (differences first: the type's lowest value times log2 e is out of range); 32 or 64 of them are added up in 32 bits, the rest in 64.
 */
template <int TYPE>
__global__ __launch_bounds__(BEAM_THREADS, 4) void k_beam_rows(const beam_args a)
{
    using namespace bam;
    constexpr uint32_t VEC = TYPE == 2 ? 4 : 8, SIZE = TYPE == 2 ? 4 : 2, CHUNK = BEAM_THREADS * BEAM_LOADS * VEC;
    __shared__ uint64_t room[BEAM_ROOM], tops[BEAM_THREADS], bound_at;
    __shared__ uint16_t noted[BEAM_THREADS * BEAM_LOADS];
    __shared__ uint32_t n_room, n_noted;
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
    if (t == 0) n_room = n_noted = 0, bound_at = 0;
    __syncthreads();
    uint32_t here = 0;                               /* n_room, as all threads know it */
    for (uint32_t c = begin; c < end; c += CHUNK) {
        u32x4 raw[BEAM_LOADS];
        float tops_of[BEAM_LOADS];                   /* NaN where there is one: such a beam's tokens are picked by their numbers (k_beam_join) */
#pragma unroll
        for (uint32_t j = 0; j < BEAM_LOADS; j++) {
            const uint32_t i = c + (j * BEAM_THREADS + t) * VEC;
            raw[j] = u32x4{NOTHING<TYPE>, NOTHING<TYPE>, NOTHING<TYPE>, NOTHING<TYPE>};
            if (c + j * BEAM_THREADS * VEC < whole && i < whole) raw[j] = *(const u32x4_any*)(x + (uint64_t)i * SIZE);
        }
        /* (of the last chunk) */
        const uint32_t rest_at = end - c <= CHUNK && t < end - whole ? whole + t : 0xffffffffu;
        const float rest = rest_at != 0xffffffffu ? number_at<TYPE>(x, rest_at) : -INFINITY;
        float top = rest;
        uint32_t top_at = rest_at;                   /* no token of the thread with that number comes behind this one of its load */
#pragma unroll
        for (uint32_t j = BEAM_LOADS; j-- > 0;) {
            float y = number_in<TYPE>(raw[j], 0);
#pragma unroll
            for (uint32_t e = 1; e < VEC; e++) y = __builtin_elementwise_maximum(y, number_in<TYPE>(raw[j], e));
            tops_of[j] = y;
            const uint32_t i = c + (j * BEAM_THREADS + t) * VEC;
            if (i < whole && !(y < top)) { top = y; top_at = i + VEC - 1u; }
        }
        const float larger_m = __builtin_elementwise_maximum(m, top), use = larger_m == -INFINITY ? 0.0f : larger_m;
        float sum[4] = {__builtin_amdgcn_exp2f((rest - use) * LOG2E), 0, 0, 0};
#pragma unroll
        for (uint32_t j = 0; j < BEAM_LOADS; j++) {
            if (c + j * BEAM_THREADS * VEC >= whole) break;
#pragma unroll
            for (uint32_t e = 0; e < VEC; e++) sum[e & 3u] += __builtin_amdgcn_exp2f((number_in<TYPE>(raw[j], e) - use) * LOG2E);
        }
        s = s * (double)__builtin_amdgcn_exp2f((m - use) * LOG2E) + (double)((sum[0] + sum[1]) + (sum[2] + sum[3]));
        m = larger_m;
        if (c == begin) {
            uint64_t mine = top_at == 0xffffffffu ? 0ull : key_of(top, top_at);
            const uint32_t groups = a.width <= 32u ? 64u : 256u;
            if (groups == 64u) {
                mine = larger(mine, shfl_xor64(mine, 1));
                mine = larger(mine, shfl_xor64(mine, 2));
                if ((t & 3u) == 0) tops[t / 4u] = mine;
            } else tops[t] = mine;
            __syncthreads();
            if (t < groups) {
                mine = tops[t];
                uint32_t above = 0;
                for (uint32_t i = 0; i < groups; i++) above += tops[i] > mine ? 1u : 0u;
                if (mine && above == a.width - 1u) bound_at = mine;
            }
            __syncthreads();
            bound = bound_at;
        }
        auto put = [&](const float y, const uint32_t i) {
            const uint64_t k = key_of(y, i);
            if (k < bound) return;
            const uint32_t at = atomicAdd(&n_room, 1u);
            if (at < BEAM_ROOM) room[at] = k;
        };
        auto load_of = [&](const uint32_t p) { return *(const u32x4_any*)(x + (uint64_t)(c + p * VEC) * SIZE); };
        auto put_noted = [&](const uint32_t n) {
            for (uint32_t m = t; m < n; m += BEAM_THREADS) {
                const uint32_t p = noted[m];
                const u32x4 z = load_of(p);
#pragma unroll
                for (uint32_t e = 0; e < VEC; e++) put(number_in<TYPE>(z, e), c + p * VEC + e);
            }
            if (rest_at != 0xffffffffu) put(rest, rest_at);
        };
#pragma unroll
        for (uint32_t j = 0; j < BEAM_LOADS; j++) {
            const uint32_t p = j * BEAM_THREADS + t, i = c + p * VEC;
            if (i < whole && key_of(tops_of[j], i) >= bound) noted[atomicAdd(&n_noted, 1u)] = (uint16_t)p;
        }
        __syncthreads();
        const uint32_t n_loads = n_noted;
        put_noted(n_loads);
        __syncthreads();
        uint32_t n = n_room;
        if (t == 0) n_noted = 0;
        __syncthreads();                             /* before somebody adds to them */
        if (n > BEAM_ROOM) {
            /* the chunk's largest, the next one, ... */
            uint64_t last = ~0ull;
            for (uint32_t r = 0; r < a.width && last; r++) {
                uint64_t mine = 0;
                auto take = [&](const float y, const uint32_t i) { const uint64_t k = key_of(y, i); if (k < last && k > mine) mine = k; };
                for (uint32_t m = t; m < n_loads; m += BEAM_THREADS) {
                    const uint32_t p = noted[m];
                    const u32x4 z = load_of(p);
#pragma unroll
                    for (uint32_t e = 0; e < VEC; e++) take(number_in<TYPE>(z, e), c + p * VEC + e);
                }
                if (rest_at != 0xffffffffu) take(rest, rest_at);
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) mine = larger(mine, shfl_xor64(mine, o));
                if (lane == 0) tops[wave] = mine;
                __syncthreads();
                last = larger(larger(tops[0], tops[1]), larger(tops[2], tops[3]));
                __syncthreads();
            }
            if (last > bound) bound = last;
            if (t == 0) n_room = here;
            __syncthreads();
            put_noted(n_loads);                      /* no more than `width` */
            __syncthreads();
            n = n_room;
            __syncthreads();
        }
        /* the room left has to hold `width` more: what is there is reduced to the best */
        if (n > BEAM_ROOM / 2 && end - c > CHUNK) {
            uint64_t mine[BEAM_ROOM / BEAM_THREADS];
            uint32_t above[BEAM_ROOM / BEAM_THREADS];
#pragma unroll
            for (uint32_t j = 0; j < BEAM_ROOM / BEAM_THREADS; j++) { mine[j] = j * BEAM_THREADS + t < n ? room[j * BEAM_THREADS + t] : 0ull; above[j] = 0; }
            for (uint32_t i = 0; i < n; i++) {
                const uint64_t k = room[i];
#pragma unroll
                for (uint32_t j = 0; j < BEAM_ROOM / BEAM_THREADS; j++) above[j] += k > mine[j] ? 1u : 0u;
            }
            __syncthreads();
#pragma unroll
            for (uint32_t j = 0; j < BEAM_ROOM / BEAM_THREADS; j++) if (mine[j] && above[j] < a.width) room[above[j]] = mine[j];
            n = a.width;                             /* (at most half the room) */
            if (t == 0) n_room = n;
            __syncthreads();
            if (room[n - 1u] > bound) bound = room[n - 1u];
        }
        here = n;
    }
    const uint32_t n = here;
    const uint64_t to = ((uint64_t)row * a.splits + split) * a.width;
    for (uint32_t j = t; j < n; j += BEAM_THREADS) {
        const uint64_t mine = room[j];
        uint32_t above = 0;
        for (uint32_t i = 0; i < n; i++) above += room[i] > mine ? 1u : 0u;
        if (above < a.width) a.best[to + above] = mine;
    }
    for (uint32_t j = n + t; j < a.width; j += BEAM_THREADS) a.best[to + j] = 0;
    /* the parts of the sum of exponentials */
    auto join = [](double& s, float& m, const double s2, const float m2) {
        const float top = __builtin_elementwise_maximum(m, m2), use = top == -INFINITY ? 0.0f : top;
        s = s * (double)__builtin_amdgcn_exp2f((m - use) * LOG2E) + s2 * (double)__builtin_amdgcn_exp2f((m2 - use) * LOG2E);
        m = top;
    };
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double s2 = __builtin_bit_cast(double, shfl_xor64(__builtin_bit_cast(uint64_t, s), o));
        join(s, m, s2, __shfl_xor(m, o));
    }
    if (lane == 0) wave_s[wave] = s, wave_m[wave] = m;
    __syncthreads();
    if (t == 0) {
        for (uint32_t w = 1; w < 4; w++) join(s, m, wave_s[w], wave_m[w]);
        a.part_s[(uint64_t)row * a.splits + split] = s;
        a.part_m[(uint64_t)row * a.splits + split] = m;
    }
}

/* a candidate: its sum in order, and beam * vocab + token; none is all zeros */
struct beam_place { uint64_t sum; uint32_t at; };
__device__ __forceinline__ bool before(const beam_place& a, const beam_place& b) { return a.sum > b.sum || (a.sum == b.sum && a.at < b.at); }
__device__ __forceinline__ beam_place first_of(const beam_place& a, const int by)
{
    const beam_place o = {shfl_xor64(a.sum, by), (uint32_t)__shfl_xor((int)a.at, by)};
    return before(o, a) ? o : a;
}

/*
 * A request: the beams' logarithms of sums of exponentials, and the best of what the pieces left, by the same bound as in k_beam_rows.  Sums are compared in 64 bits:
 * the beams' own sums are rounded to 32, what is added to them is not, and of two beams that differ in their last place the right one is taken.
 */
template <uint32_t THREADS>
__global__ __launch_bounds__(THREADS) void k_beam_join(const beam_args a)
{
    using namespace bam;
    __shared__ double offset[BEAM_BEAMS];            /* of a logit's difference to the beam's largest (which may be so far from zero that nothing else would be left) */
    __shared__ float largest[BEAM_BEAMS];
    __shared__ uint64_t room_sum[BEAM_ROOM], tops_sum[256];
    __shared__ uint32_t room_at[BEAM_ROOM], tops_at[256], n_room;
    __shared__ beam_place bound_at;
    const uint32_t t = threadIdx.x, lane = bam::lane(), wave = first(t / 64u), request = blockIdx.x;
    if (t == 0) n_room = 0, bound_at = beam_place{0, 0};
    for (uint32_t i = wave; i < a.beams; i += THREADS / 64u) {
        const uint64_t at = ((uint64_t)request * a.beams + i) * a.splits;
        float top = -INFINITY;
        for (uint32_t k = lane; k < a.splits; k += 64u) top = __builtin_elementwise_maximum(top, a.part_m[at + k]);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, o));
        double sum = 0;
        for (uint32_t k = lane; k < a.splits; k += 64u) sum += a.part_s[at + k] * exp((double)a.part_m[at + k] - (double)top);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sum += __builtin_bit_cast(double, shfl_xor64(__builtin_bit_cast(uint64_t, sum), o));
        if (lane == 0) { offset[i] = (double)a.scores[(int64_t)request * a.score_row + i] - log(sum); largest[i] = top; }
    }
    __syncthreads();
    const uint32_t each = a.splits * a.width, all = a.beams * each;
    const uint64_t* const best = a.best + (uint64_t)request * all;
    auto candidate = [&](const uint32_t c) {
        const uint32_t i = c / each, j = c % each;
        const double by = offset[i];
        beam_place p = {0, 0};
        if (by - by == 0) {
            const uint64_t k = best[c];
            if (k) { p.at = i * a.vocab + ~(uint32_t)k; p.sum = ordered(((double)number_of((uint32_t)(k >> 32)) - (double)largest[i]) + by); }
        } else if (j < a.width && j < a.vocab) {
            /* all tokens of the beam have the same, an infinity or NaN: by their numbers */
            p.at = i * a.vocab + j;
            p.sum = ordered(by);
        }
        return p;
    };
    beam_place mine = {0, 0};
    for (uint32_t c = t; c < all; c += THREADS) { const beam_place p = candidate(c); if (before(p, mine)) mine = p; }
    /* the bound: of 64 groups of threads where that is enough, else of 256 */
    const uint32_t groups = a.width <= 32u ? 64u : 256u;
#pragma unroll
    for (uint32_t o = 1; o < THREADS / 64u; o <<= 1) if (o < THREADS / groups) mine = first_of(mine, (int)o);
    if (t % (THREADS / groups) == 0) { tops_sum[t / (THREADS / groups)] = mine.sum; tops_at[t / (THREADS / groups)] = mine.at; }
    __syncthreads();
    if (t < groups) {
        mine = beam_place{tops_sum[t], tops_at[t]};
        uint32_t above = 0;
        for (uint32_t i = 0; i < groups; i++) above += before(beam_place{tops_sum[i], tops_at[i]}, mine) ? 1u : 0u;
        if (mine.sum && above == a.width - 1u) bound_at = mine;
    }
    __syncthreads();
    const beam_place bound = bound_at;
    for (uint32_t c = t; c < all; c += THREADS) {
        const beam_place p = candidate(c);
        if (!p.sum || (bound.sum && before(bound, p))) continue;
        const uint32_t at = atomicAdd(&n_room, 1u);
        if (at < BEAM_ROOM) { room_sum[at] = p.sum; room_at[at] = p.at; }
    }
    __syncthreads();
    const uint32_t n = n_room;
    const uint64_t to = (uint64_t)request * a.width;
    auto give = [&](const uint32_t r, const beam_place& p) {
        a.sums[to + r] = (float)number_of(p.sum);
        a.from[to + r] = (int32_t)(request * a.beams + p.at / a.vocab);
        a.token[to + r] = (int32_t)(p.at % a.vocab);
    };
    if (n <= BEAM_ROOM) {
        for (uint32_t j = t; j < n; j += THREADS) {
            const beam_place p = {room_sum[j], room_at[j]};
            uint32_t above = 0;
            for (uint32_t i = 0; i < n; i++) above += before(beam_place{room_sum[i], room_at[i]}, p) ? 1u : 0u;
            if (above < a.width) give(above, p);
        }
        return;
    }
    /* they do not fit: the first, the next one, ... */
    beam_place last = {~0ull, 0};
    for (uint32_t r = 0; r < a.width; r++) {
        mine = beam_place{0, 0};
        for (uint32_t c = t; c < all; c += THREADS) { const beam_place p = candidate(c); if (p.sum && before(last, p) && before(p, mine)) mine = p; }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) mine = first_of(mine, o);
        __syncthreads();
        if (lane == 0) { tops_sum[wave] = mine.sum; tops_at[wave] = mine.at; }
        __syncthreads();
        last = beam_place{0, 0};
        for (uint32_t w = 0; w < THREADS / 64u; w++) { const beam_place p = {tops_sum[w], tops_at[w]}; if (before(p, last)) last = p; }
        if (t == 0) give(r, last);
    }
}

struct beam_plan { uint32_t splits, per; uint64_t best_at, s_at, m_at, bytes; };
beam_plan plan_of(const uint64_t requests, const uint64_t beams, const uint64_t vocab, const uint32_t width, const int type)
{
    beam_plan p{};
    const uint64_t rows = requests * beams, load = BEAM_THREADS * (type == 2 ? 4 : 8);
    uint64_t splits = (2048 + rows - 1) / rows;
    const uint64_t most = (vocab + load - 1) / load;
    if (splits > most) splits = most;
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
    if (rows * p.splits > 0x7fffffffull || all > 0x7fffffffull) return fail(EINVAL, "bam_beam_select: more workgroups or candidates than 31 bits count");
    beam_args a{};
    a.logits = w.d_logits; a.row = w.logits_row; a.scores = w.d_scores; a.score_row = w.scores_row;
    a.requests = (uint32_t)w.n_requests; a.beams = (uint32_t)w.n_beams; a.vocab = (uint32_t)w.vocab; a.width = w.width; a.splits = p.splits; a.per = p.per;
    a.sums = w.d_sums; a.from = w.d_beams; a.token = w.d_tokens;
    uint8_t* const at = (uint8_t*)w.d_work;
    a.best = (uint64_t*)(at + p.best_at); a.part_s = (double*)(at + p.s_at); a.part_m = (float*)(at + p.m_at);
    const dim3 grid((uint32_t)(rows * p.splits)), block(BEAM_THREADS);
    hipStream_t const st = (hipStream_t)stream;
    if (w.type == 0) hipLaunchKernelGGL(k_beam_rows<0>, grid, block, 0, st, a);
    else if (w.type == 1) hipLaunchKernelGGL(k_beam_rows<1>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(k_beam_rows<2>, grid, block, 0, st, a);
    if (all <= 2048) hipLaunchKernelGGL(k_beam_join<256>, dim3(a.requests), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_beam_join<1024>, dim3(a.requests), dim3(1024), 0, st, a);
    hip_err_chk(hipGetLastError());
    BAM_API_END
}

} // extern "C"
