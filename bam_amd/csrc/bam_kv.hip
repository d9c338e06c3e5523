// Key-value cache in the pages of an array, of the C-ABI: appending keys and values (with norms of queries and keys and the
// position rotation on the way), reading rows back, and attention of the newest tokens over what the cache holds.
//
// The cache is cut into blocks of T tokens.  A block has two pages for each key-value head: one of keys and one of values, T the largest power of
// two for which T rows of `dim` 16-bit numbers fit a page.  Within a page the numbers lie in pieces of 16 bytes, in the order in
// which the matrix instructions take them:
//   keys    piece (c, t) at (c * T + place(t)) * 16: numbers 8c .. 8c+7 of token t             c < dim / 8
//   values  piece (t, d) at (t * dim + d) * 16: number d of tokens 8t .. 8t+7           t < T / 8
// place(t) is t with its bits 2 and 3 exchanged (t itself where a page holds eight tokens).  What neighbouring lanes of a wave load lies next to each other, and
// is an operand as it stands: with the scores taken as S^T = K Q^T and the output as O^T = V^T P^T, a lane's accumulators of the scores are its
// part of P^T if the rows of K come in that order.
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
};
struct bam_kv {
    bam_array_t* a;
    kv_geom g;
    int f16;
    uint64_t cache_pages;
    bool unheld;                        /* reads of resident pages without a reference are switched on */
};

namespace {

struct kv_seqs {
    const int32_t* starts;              /* [n + 1] first row of each sequence's new tokens; NULL: one new token each */
    const int32_t* lens;                /* [n] tokens of each sequence, the new ones among them */
    const int32_t* table;               /* [n][width] blocks */
    int64_t stride;
    uint32_t n, rows, width;
};

// sequence of row i
__device__ __forceinline__ uint32_t seq_of(const kv_seqs& s, const uint32_t i)
{
    if (!s.starts) return i;
    uint32_t lo = 0, hi = s.n;          /* the last sequence that starts at or before row i */
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (s.starts[mid] <= (int32_t)i) lo = mid; else hi = mid;
    }
    return lo;
}
// a row's place: sequence, position, rows of its sequence from it on (those that there are: starts may say more than `rows`), position of its sequence's first new
// row; false where the row has none (no such sequence, before the first position, past the table)
struct kv_place { uint32_t seq, pos, rest, first; };
__device__ __forceinline__ bool place_of(const kv_seqs& s, const kv_geom& g, const uint32_t i, kv_place& p)
{
    p.seq = seq_of(s, i);
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
struct kv_rows {
    const uint16_t *q, *k, *v;          /* rows of heads; k and v are where rows go to when the cache is read */
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    uint16_t* q_out;
    const uint16_t *q_norm, *k_norm;
    const float *cos, *sin;
    uint32_t positions, q_heads, rot, pairs, aligned;      /* aligned: q, k, v in whole pieces of 16 bytes */
    float eps;
    uint32_t window, piece;             /* rows that a wave looks for beginnings of runs among, and the most rows it takes at a time */
    uint32_t q_heads_each, q_waves;     /* heads of queries that a wave takes */
};

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
template <int LPR, int F16>
__device__ __forceinline__ u32x4 norm_and_rotate(const kv_rows& io, const kv_geom& g, u32x4 x, const bool norm, const u32x4 w, const kv_turn& t, const uint32_t piece)
{
    if (!norm && !io.rot) return x;
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; i++) { const uint32_t y = x[i]; f[2 * i] = from16<F16>(y & 0xffffu); f[2 * i + 1] = from16<F16>(y >> 16); }
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
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = to16<F16>(f[2 * i], f[2 * i + 1]);
    return x;
}

/*
 * A wave takes some heads of queries of one row, or one head's keys and values of the runs of rows that begin among io.window rows: a run is the new rows of
 * a sequence in one block, gone through in pieces of up to io.piece tokens (eight or sixteen that begin at a multiple of that).  A page's rows all belong to one
 * wave: a page that holds new rows only is not read, and one that a second wave found gone again would come without the rows of the first.
 *   Bound by memory where there are many rows: 19 459 rows of 32 heads on 8 of 128 numbers, normed and turned, 480 MB in 124 us (3.9 TB/s), 160 MB out again in 43; a wave for
 * each four rows took 288 and 112 (each looked its sequence up for 1 KiB).  Few rows: the chain of looks, table, references, rows, 6 to 7 us.
 */
template <int LPR, int F16, bool WRITE, bool ALIGNED>
__global__ __launch_bounds__(256, LPR < 32 ? 4 : 3) void k_kv_rows(const kv_geom g, const kv_seqs s, const kv_rows io)
{
    using namespace bam;
    constexpr uint32_t RPW = 64 / LPR, TRIPS = 16 / RPW, DT = LPR / 8;           /* trips of a piece's keys; of its values: a trip is 64 times two numbers of eight tokens */
    const uint32_t wave = first(blockIdx.x * 4u + threadIdx.x / 64u), lane = bam::lane();
    const uint32_t sub = lane / LPR, piece = lane % LPR;
    const bool in_row = piece * 8u < g.dim;
    const uint32_t col = in_row ? piece * 8u : 0u;           /* lanes past the row's end load its beginning, and count as zeros */
    if (WRITE && wave < io.q_waves) {
        const uint32_t per = (io.q_heads + io.q_heads_each - 1) / io.q_heads_each, i = wave / per, h0 = wave % per * io.q_heads_each;
        const uint32_t h1 = h0 + io.q_heads_each < io.q_heads ? h0 + io.q_heads_each : io.q_heads;
        kv_place p{0, 0, 0, 0};
        const bool known = place_of(s, g, i, p);
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
    const uint32_t n = wave - (WRITE ? io.q_waves : 0u), head = n % g.heads;
    const uint64_t first_row = (uint64_t)(n / g.heads) * io.window;
    if (first_row >= s.rows) return;
    kv_place p{0, 0, 0, 0};
    const uint32_t mine = (uint32_t)first_row + lane;
    const bool has = lane < io.window && mine < s.rows && place_of(s, g, mine, p);
    const bool begins = has && ((p.pos & (g.tokens - 1u)) == 0 || p.pos == p.first || (s.starts && s.starts[p.seq] == (int32_t)mine));
    if constexpr (!WRITE) {
        /* rows without a place come out as zeros */
        for (uint64_t m = ballot(lane < io.window && mine < s.rows && !has); m; m &= m - 1)
            for (uint32_t d = lane; d < g.dim; d += 64u) {
                ((uint16_t*)io.k)[(int64_t)(first_row + first_lane(m)) * io.k_row + (int64_t)head * io.k_head + d] = 0;
                ((uint16_t*)io.v)[(int64_t)(first_row + first_lane(m)) * io.v_row + (int64_t)head * io.v_head + d] = 0;
            }
    }
    for (uint64_t m = ballot(begins); m; m &= m - 1) {
        const uint32_t j = first_lane(m), pos = bcast(p.pos, j), rest = bcast(p.rest, j), seq = bcast(p.seq, j), row = (uint32_t)first_row + j;
        uint64_t page = 0;
        const bool there = page_of_block(g, s, seq, pos >> g.tokens_log, head, page);
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
                uint8_t* const at = keys + (uint64_t)(col / 8u) * g.tokens * 16u;
#pragma unroll
                for (uint32_t e = 0; e < TRIPS; e++) {
                    const uint32_t r = r0 + e * RPW < cnt ? r0 + e * RPW : 0u;
                    if constexpr (WRITE) x[e] = load_piece<ALIGNED>(k_rows + (int64_t)r * io.k_row + col);
                    else x[e] = none & 1u ? u32x4{fill, fill, fill, fill} : ld_payload((const u32x4*)(at + place_in(g, in_block + r) * 16u));
                }
                u32x4 w{0, 0, 0, 0};
                if (WRITE && io.k_norm) w = load_piece<true>(io.k_norm + col);
#pragma unroll
                for (uint32_t e = 0; e < TRIPS; e++) {
                    if (e * RPW >= cnt) break;
                    const uint32_t r = r0 + e * RPW;
                    if constexpr (WRITE) {
                        const kv_turn t = turn_of(io, piece, pos + off + (r < cnt ? r : 0u));
                        x[e] = norm_and_rotate<LPR, F16>(io, g, in_row ? x[e] : u32x4{0, 0, 0, 0}, io.k_norm != nullptr, w, t, piece);
                        if (r < cnt && in_row) st16_sys(at + place_in(g, in_block + r) * 16u, x[e]);
                    } else if (r < cnt && in_row) *(u32x4*)(k_rows + (int64_t)r * io.k_row + col) = x[e];
                }
            }
            if (values || (none & 2u)) {
#pragma unroll
                for (uint32_t e = 0; e < DT; e++) {
                    const uint32_t y = e * 64u + l, group = y / pairs, d = y % pairs * 2u;
                    const int32_t tok = (int32_t)(group * 8u) - piece_first;
                    if (group >= groups || tok + 8 <= 0 || tok >= (int32_t)cnt) continue;
                    uint8_t* const at = values + ((uint64_t)((in_block + tok) >> 3) * g.dim + d) * 16u;
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
                        if (full) {
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

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
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
template <int DP, int F16, int NT, bool HELD>
__device__ __forceinline__ bool kv_steps(const kv_geom& g, const kv_seqs& s, const kv_att& a, const kv_span& sp, const uint32_t seq, const uint32_t head, const uint32_t v0, const uint32_t v1,
                                         const u32x4 (&q)[NT][DP / 32], const int32_t (&pos)[NT], f32x4 (&o)[NT][DP / 16], float (&m)[NT], float (&l)[NT], bool& gone, uint32_t& n_access, uint32_t& n_hit)
{
    using namespace bam;
    const uint32_t lane = bam::lane(), row = lane & 15u, grp = lane >> 4;
    const uint32_t T = g.tokens, D = g.dim;
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
        for (uint32_t t0 = t_first; t0 < t_end; t0 += 32u) {
            /* this lane's tokens as a row of K (8 (row / 4) + row % 4, and 4 further on) and as its part of V (8 grp .. + 7) lie in one block each */
            const uint32_t kt = T < 16 ? t0 + 8u * (row >> 2) : t0 + 16u * (row >> 3), vt = t0 + 8u * grp;
            const uint32_t kb = (kt >> g.tokens_log) - b_first, vb = (vt >> g.tokens_log) - b_first;
            const uint8_t* kp = g.base + ((uint64_t)bam::shfl(slot, kb) << g.page_log) + ((kt & (T - 1u)) + (T < 16 ? row & 3u : row & 7u)) * 16u;
            const uint8_t* vp = g.base + ((uint64_t)bam::shfl(slot, 32u + vb) << g.page_log) + (((vt & (T - 1u)) >> 3) * D + row) * 16u;
            /* keys (part 0) or values (part 32) of the step, page by page: `load` for the lanes whose block came, which is `mine` for this lane */
            auto by_page = [&](const uint32_t part, const uint32_t mine, auto&& load) {
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
            u32x4 k0[DP / 32], k1[DP / 32], vv[DP / 16];
            /* what lies past a row's end is not loaded: its place takes the row's beginning, zero among the keys, of no row among the values */
            const uint8_t *k_at[DP / 32], *v_at[DP / 16];
#pragma unroll
            for (uint32_t j = 0; j < DP / 32; j++) k_at[j] = kp + ((4u * j + grp) * 8u < D ? (4u * j + grp) * T * 16u : 0u);
#pragma unroll
            for (uint32_t i = 0; i < DP / 16; i++) v_at[i] = 16u * i < D ? vp + i * 256u : vp;
            if (HELD && !all) {
#pragma unroll
                for (int j = 0; j < DP / 32; j++) k0[j] = k1[j] = u32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < DP / 16; i++) vv[i] = u32x4{0, 0, 0, 0};
                by_page(0, kb, [&](const uint64_t by) {
#pragma unroll
                    for (int j = 0; j < DP / 32; j++) { k0[j] = ld_payload((const u32x4*)(k_at[j] + by)); k1[j] = ld_payload((const u32x4*)(k_at[j] + by + (T < 16 ? 64 : 128))); }
                });
                if (gone) return true;
            } else if constexpr (DP <= 128) {
                if (T < 16) load_step<64>(k_at, v_at, k0, k1, vv); else load_step<128>(k_at, v_at, k0, k1, vv);
            } else {
                if (T < 16) load_keys<64>(k_at, k0, k1); else load_keys<128>(k_at, k0, k1);
            }
            if (D < DP) {
#pragma unroll
                for (uint32_t j = 0; j < DP / 32; j++) { const bool in = (4u * j + grp) * 8u < D; k0[j] = in ? k0[j] : u32x4{0, 0, 0, 0}; k1[j] = in ? k1[j] : u32x4{0, 0, 0, 0}; }
            }
            const bool whole = !((holes >> ((t0 >> g.tokens_log) - b_first)) & step_blocks) && (int64_t)t0 + 31 <= sp.first_pos && (!a.window || (int64_t)sp.last_pos - t0 < a.window || t0 + 32u <= a.sinks);
            f32x4 s0[NT], s1[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                s0[n] = s1[n] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < DP / 32; j++) { s0[n] = mma<F16>(k0[j], q[n][j], s0[n]); s1[n] = mma<F16>(k1[j], q[n][j], s1[n]); }
            }
            if (HELD && !all) {
                by_page(32, vb, [&](const uint64_t by) {
#pragma unroll
                    for (int i = 0; i < DP / 16; i++) vv[i] = ld_payload((const u32x4*)(v_at[i] + by));
                });
                if (gone) return true;
            } else if constexpr (DP > 128) {         /* wide heads: the values behind the scores, for which they would not leave registers */
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint8_t* at[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) at[i] = v_at[8 * h + i];
                    load_pieces(at, vv + 8 * h);
                }
            }
            const bool hole = (holes >> vb) & 1u;
            bool slow = false;
            if (!whole) {
                /* values of tokens that no row sees may be anything: none of it may meet the zeros of P */
                const uint32_t any = hole ? 0u : seen_of_eight((int32_t)vt, sp.last_pos, low_of(a, sp.first_pos), (int32_t)a.sinks);
#pragma unroll
                for (int i = 0; i < DP / 16; i++) vv[i] = only(vv[i], any);
                if (sp.first_pos != sp.last_pos) {
                    bool odd = false;
#pragma unroll
                    for (int i = 0; i < DP / 16; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) odd |= odd16<F16>(vv[i][e]);
                    slow = ballot(odd) != 0;
                    if (!HELD && slow) return false;             /* row by row, in the launch that holds its pages: the sums of this one stay where they are */
                }
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
                    for (int i = 0; i < DP / 16; i++) o[n][i] = mma<F16>(vv[i], p, o[n][i]);
                } else {
                    /* an infinity or NaN among the values of tokens that some rows see and others do not: row by row, what the row does not see as zero */
                    for (uint32_t c = 0; c < 16; c++) {
                        const uint32_t sc = bam::shfl(sees, (lane & 48u) + c);
#pragma unroll
                        for (int i = 0; i < DP / 16; i++) {
                            const f32x4 with = mma<F16>(only(vv[i], sc), p, o[n][i]);
                            if (row == c) o[n][i] = with;
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

/* a workgroup's split of an item, of its rows from s0 on: its four waves a quarter of the steps each, joined over LDS; the sums to their rows where there is one split, else to a.part */
template <int DP, int F16, int NT, bool HELD>
__device__ __forceinline__ bool kv_split(const kv_geom& g, const kv_seqs& s, const kv_att& a, const uint32_t item, const kv_item& it, const uint32_t s0, const uint32_t split, float* lds, bool& gone)
{
    using namespace bam;
    constexpr uint32_t R = 16 * NT;
    const uint32_t lane = bam::lane(), wave = first(threadIdx.x / 64u), row = lane & 15u, grp = lane >> 4, D = g.dim;
    const uint32_t s1 = s0 + R < it.r1 ? s0 + R : it.r1;
    kv_span sp = span_of(a, s.width << g.tokens_log, it.pos0, it.r0, it.r1);                     /* the item's splits, */
    sp.first_pos = it.pos0 + (int32_t)(s0 / a.group);                           /* as these rows see them */
    sp.last_pos = it.pos0 + (int32_t)((s1 - 1) / a.group);
    uint32_t v0 = split * a.steps, v1 = v0 + a.steps;
    if (v1 > sp.n_steps || split + 1 == a.splits) v1 = sp.n_steps;              /* the last takes what is beyond the length that was announced */
    if (v0 > v1) v0 = v1;
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
            if (has && (4u * j + grp) * 8u < D) q[n][j] = a.aligned ? load_piece<true>(from + (4u * j + grp) * 8u) : load_piece<false>(from + (4u * j + grp) * 8u);
        }
        m[n] = -INFINITY;
        l[n] = 0;
#pragma unroll
        for (int i = 0; i < DP / 16; i++) o[n][i] = f32x4{0, 0, 0, 0};
    }
    uint32_t n_access = 0, n_hit = 0;
    const bool ok = kv_steps<DP, F16, NT, HELD>(g, s, a, sp, it.seq, it.head, w0, w1, q, pos, o, m, l, gone, n_access, n_hit);
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
        f32x4 lo = *(const f32x4*)(os + r * DP + c), hi = *(const f32x4*)(os + r * DP + c + 4);
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

template <int DP, int F16, int NT>
__global__ __launch_bounds__(256) void k_kv_attend(const kv_geom g, const kv_seqs s, const kv_att a)
{
    extern __shared__ float lds[];
    const uint32_t item = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    kv_item it;
    bool gone = false, ok = true;
    if (item_of(g, s, a, item, it)) ok = kv_split<DP, F16, NT, false>(g, s, a, item, it, it.r0, split, lds, gone);
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
template <int DP, int F16, int NW, bool EXACT>
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
    uint32_t v0 = split * a.steps, v1 = v0 + a.steps;
    if (v1 > sp.n_steps || split + 1 == a.splits) v1 = sp.n_steps;
    if (v0 > v1) v0 = v1;
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
    auto load_tile = [&](const uint32_t buf) {
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
        at_first = t_next; at_end = t_end < sp.len ? t_end : sp.len; at_holes = holes; at_block = b_first;          /* (the last step may go on behind the table's end) */
        t_next += KT;
    };
    next_blocks();
    bool more = there;
    if (more) { enter_next(); load_tile(0); }
    /* the lane's row of K among the places of 32 tokens: the one that puts the scores of tokens 8 half .. + 7 of each 16 into its accumulators */
    const uint32_t k_row = T < 16 ? (row & 0x13u) | ((row & 4u) << 1) | ((row & 8u) >> 1) : row;
    const uint32_t k_read = (k_row >> 3) * DP * 16u + (k_row & 7u) * 16u + (half ^ (k_row >> 3 & 1u)) * 128u;
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
        if (idle || (int32_t)t0 > last_pos) continue;
        /*
         * The operands from LDS are read eight ahead of the products that take them, and the order is held (sched_barrier): left to itself the compiler reads each right before
         * its product and waits for it, a hundred cycles for every 32 of the matrix unit.
         */
        constexpr uint32_t NK = DP / 16 * (KT / 32), NV = DP / 32 * (KT / 16);
        auto key_piece = [&](const uint32_t n) { return *(const u32x4*)(keys + (n / (KT / 32)) * 256u + (n % (KT / 32)) * (DP * 64u) + k_read); };
        auto value_piece = [&](const uint32_t n) { return *(const u32x4*)(values + ((2u * (n / (DP / 32)) + half) * DP + 32u * (n % (DP / 32)) + row) * 16u); };
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
                o[i] = mma32<F16>(f[n % 8], p[k], o[i]);
                if (n + 8 < NV) f[n % 8] = value_piece(n + 8);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
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
template <int DP, int F16, int NT>
__global__ __launch_bounds__(256) void k_kv_attend_once(const kv_geom g, const kv_seqs s, const kv_att a)
{
    extern __shared__ float lds[];
    const uint32_t item = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    kv_item it;
    bool gone = false;
    if (!item_of(g, s, a, item, it)) return;
    if (kv_split<DP, F16, NT, false>(g, s, a, item, it, it.r0, split, lds, gone)) return;
    __syncthreads();
    gone = false;
    kv_split<DP, F16, NT, true>(g, s, a, item, it, it.r0, split, lds, gone);
}

/* what the first launch left, with its pages held; ends at once where that is nothing */
template <int DP, int F16, int NT>
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
            kv_split<DP, F16, NT, true>(g, s, a, (uint32_t)(x / a.splits), it, s0, (uint32_t)(x % a.splits), lds, gone);
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
struct kv_plan { uint32_t nt, waves, rows, tiles, splits, steps; uint64_t items, left_at, m_at, l_at, part_at, bytes; };

/* steps of 32 tokens that a tile of `rows` rows can have to look at, of sequences of up to max_len tokens */
uint64_t most_steps(const uint64_t max_len, const uint64_t new_tokens, const uint32_t window, const uint32_t sinks)
{
    const uint64_t all = (max_len + 31) / 32;
    if (!window) return all;
    const uint64_t seen = (window + new_tokens + 31) / 32 + 1 + (sinks + 31ull) / 32;
    return seen < all ? seen : all;
}

kv_plan plan_of(const bam_kv_t* kv, const uint64_t n_seqs, const uint64_t max_new, const uint32_t q_heads, const uint64_t max_len, const uint32_t window, const uint32_t sinks)
{
    kv_plan p{};
    const uint64_t group = q_heads / kv->g.heads, rows = max_new * group;
    p.nt = rows <= 16 ? 1 : 2;
    p.waves = rows <= 32 ? 0 : rows <= 64 ? 2 : 4;
    p.rows = p.waves ? 32 * p.waves : 16 * p.nt;
    const uint64_t R = p.rows;
    p.tiles = (uint32_t)((rows + R - 1) / R);
    p.items = n_seqs * p.tiles * kv->g.heads;
    const uint64_t steps = most_steps(max_len, (R + group - 1) / group + 1, window, sinks);
    /*
     * Workgroups: as many as keep the memory busy, and no more, since each has its latencies before its first token and behind its last, and its split is written and
     * read again.  Few rows, four waves: one to a compute unit where a step of 32 tokens is 16 KiB, two where it is 8.  32 heads on 8 of 128 numbers, one token each, with
     * a workgroup for 512 / 256 of the device: 8 sequences of up to 8000 tokens 51 / 45 us, one of 262121 179 / 167; heads of 64 numbers, 32 sequences of
     * up to 4000, 1024 / 512 / 256: 30 / 28 / 34.
     */
    uint64_t splits = (kv->g.dim <= 64 ? 512 : 256) / p.items;
    /*
     * Tiles of rows: as many workgroups as the LDS of the compute units has room for, but no splits where there is one to each already.  The same heads, with
     * splits for 1024 / 512 / 256 workgroups whatever there is: 1000 new tokens (256 tiles) 41 / 40 / 32 us, 500 after 32500 (128 tiles) 325 / 309 / 377;
     * 10 after 16000 of eight sequences (64 tiles of two waves) 99 / 94 / 101; heads of 64 numbers, the same 45 / 59.
     */
    if (p.waves) splits = p.items >= 256 ? 1 : (kv->g.dim <= 64 ? 2048 / p.waves : 512) / p.items;
    /*
     * The shortest split: 16 steps, and 8 where that makes no more than 32 splits, whose join is short; for few rows only above 1024 tokens, below them the join costs more than
     * is gained, and 32 for tiles that half the compute units have one of.  At least 32 / 16 / 8 steps: 10 new tokens of 2000 34 / 24 / 19 us, of 16000
     * 35 / 26 / 28 (63 splits), 500 of 600 (128 tiles) 24 / 27 / 31; one token of 600, heads of 64, - / 13 / 15, of 2500 - / 14 / 13, heads of 256 - / 31 / 24.
     */
    uint64_t most = (steps + 15) / 16;
    if (p.waves && p.items >= 128) most = (steps + 31) / 32;
    else if (most < 32 && (p.waves || steps > 32)) most = (steps + 7) / 8 < 32 ? (steps + 7) / 8 : 32;
    if (splits > most) splits = most;
    if (splits > 256) splits = 256;
    if (splits < 1) splits = 1;
    p.steps = (uint32_t)((steps + splits - 1) / splits + 3) & ~3u;
    if (p.steps < 4) p.steps = 4;
    p.splits = (uint32_t)((steps + p.steps - 1) / p.steps);
    if (p.splits < 1) p.splits = 1;
    auto place = [&](uint64_t bytes) { const uint64_t at = p.bytes; p.bytes += (bytes + 255) & ~255ull; return at; };
    p.left_at = place(p.items * p.splits);
    if (p.splits > 1) {
        p.m_at = place(p.items * R * p.splits * 4);
        p.l_at = place(p.items * R * p.splits * 4);
        p.part_at = place(p.items * R * p.splits * kv->g.dim * 4);
    }
    return p;
}

/* a kernel and not a memset: the stream may be captured */
__global__ void k_kv_all_left(uint8_t* left, const uint64_t n)
{
    const uint64_t i = blockIdx.x * 256ull + threadIdx.x;
    if (i < n) left[i] = 1;
}

template <int DP, int F16, int NT>
void launch_attend(const bam_kv_t* kv, const kv_seqs& s, kv_att a, const kv_plan& p, hipStream_t st)
{
    constexpr uint32_t lds = split_lds<DP, NT>(), lds_tiles = tile_lds<DP>();
    static_assert(lds <= 65536 && lds_tiles <= 65536, "more LDS than a launch has without asking for it");
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
        if constexpr (DP <= 128) hipLaunchKernelGGL((k_kv_attend_once<DP, F16, NT>), grid, dim3(256), lds, st, kv->g, s, a);
    } else {
        if (!kv->unheld) hipLaunchKernelGGL(k_kv_all_left, dim3((uint32_t)((all + 255) / 256)), dim3(256), 0, st, a.left, all);
        else if (!p.waves) hipLaunchKernelGGL((k_kv_attend<DP, F16, NT>), grid, dim3(256), lds, st, kv->g, s, a);
        else if constexpr (NT == 2) {
            const bool exact = kv->g.dim == DP;
            if (p.waves == 2 && exact) hipLaunchKernelGGL((k_kv_attend_tiles<DP, F16, 2, true>), grid, dim3(128), lds_tiles, st, kv->g, s, a);
            else if (p.waves == 2) hipLaunchKernelGGL((k_kv_attend_tiles<DP, F16, 2, false>), grid, dim3(128), lds_tiles, st, kv->g, s, a);
            else if (exact) hipLaunchKernelGGL((k_kv_attend_tiles<DP, F16, 4, true>), grid, dim3(256), lds_tiles, st, kv->g, s, a);
            else hipLaunchKernelGGL((k_kv_attend_tiles<DP, F16, 4, false>), grid, dim3(256), lds_tiles, st, kv->g, s, a);
        }
        hipLaunchKernelGGL((k_kv_rest<DP, F16, NT>), dim3((uint32_t)groups), dim3(256), lds, st, kv->g, s, a);
    }
    if (p.splits == 1) return;
    constexpr int LPR = DP / 4;
    const uint64_t rows = p.items * p.rows, rpw = 64 / LPR;
    if (p.splits >= 16) hipLaunchKernelGGL((k_kv_join<LPR, F16, true>), dim3((uint32_t)((rows + rpw - 1) / rpw)), dim3(256), 0, st, kv->g, s, a);
    else hipLaunchKernelGGL((k_kv_join<LPR, F16, false>), dim3((uint32_t)((rows + 4 * rpw - 1) / (4 * rpw))), dim3(256), 0, st, kv->g, s, a);
}
template <int DP, int F16>
void launch_attend(const bam_kv_t* kv, const kv_seqs& s, const kv_att& a, const kv_plan& p, hipStream_t st)
{
    if (p.nt == 1) launch_attend<DP, F16, 1>(kv, s, a, p, st);
    else launch_attend<DP, F16, 2>(kv, s, a, p, st);
}
template <int F16>
void launch_attend(const bam_kv_t* kv, const kv_seqs& s, const kv_att& a, const kv_plan& p, hipStream_t st)
{
    if (kv->g.dim <= 64) launch_attend<64, F16>(kv, s, a, p, st);
    else if (kv->g.dim <= 128) launch_attend<128, F16>(kv, s, a, p, st);
    else launch_attend<256, F16>(kv, s, a, p, st);
}

template <bool WRITE>
void launch_rows(const bam_kv_t* kv, const kv_seqs& s, kv_rows io, hipStream_t st)
{
    const uint32_t lpr = kv->g.dim <= 64 ? 8 : kv->g.dim <= 128 ? 16 : 32, rpw = 64 / lpr;
    /* few rows: a trip of heads to a wave, a row to a wave; many: eight trips, and the runs that begin among sixteen rows */
    io.q_heads_each = io.q && (uint64_t)s.rows * io.q_heads > 16384 ? 8 * rpw : rpw;
    io.q_waves = io.q ? (uint32_t)((io.q_heads + io.q_heads_each - 1) / io.q_heads_each * s.rows) : 0;
    io.piece = kv->g.tokens < 16 ? 8 : 16;
    io.window = s.starts && s.rows / s.n >= 8 ? (kv->g.tokens < 64 ? kv->g.tokens : 64) : 1;
    const uint64_t waves = (uint64_t)io.q_waves + (uint64_t)((s.rows + io.window - 1) / io.window) * kv->g.heads;
    if (waves > 0x7fffffffull) throw std::runtime_error("more rows of heads than one launch takes");
    const dim3 grid((uint32_t)((waves + 3) / 4)), block(256);
#define KV_ROWS(LPR, AL) \
    if (kv->f16) hipLaunchKernelGGL((k_kv_rows<LPR, 1, WRITE, AL>), grid, block, 0, st, kv->g, s, io); \
    else hipLaunchKernelGGL((k_kv_rows<LPR, 0, WRITE, AL>), grid, block, 0, st, kv->g, s, io)
    if (WRITE && !io.aligned) { if (lpr == 8) { KV_ROWS(8, !WRITE); } else if (lpr == 16) { KV_ROWS(16, !WRITE); } else { KV_ROWS(32, !WRITE); } }
    else if (lpr == 8) { KV_ROWS(8, true); } else if (lpr == 16) { KV_ROWS(16, true); } else { KV_ROWS(32, true); }
#undef KV_ROWS
}

int bad_seqs(const char* who, const bam_kv_t* kv, const bam_kv_seqs_t& s)
{
    if (!kv || (s.n_rows && (!s.d_lens || !s.d_table))) return fail(EINVAL, std::string(who) + ": null argument");
    if (s.n_seqs > 0x7fffffffull || s.n_rows > 0x7fffffffull) return fail(EINVAL, std::string(who) + ": more rows or sequences than 31 bits count");
    if (!s.d_starts && s.n_seqs != s.n_rows) return fail(EINVAL, std::string(who) + ": without starts every sequence has one new token");
    if (!s.n_rows) return 0;
    if (!s.n_seqs) return fail(EINVAL, std::string(who) + ": rows and no sequences");
    if (s.table_width == 0 || s.table_width > 0x7fffffffull || s.table_stride < 0) return fail(EINVAL, std::string(who) + ": table of no width, or with its rows in reverse");
    if (s.table_width > 0x7ffffc00ull >> kv->g.tokens_log) return fail(EINVAL, std::string(who) + ": the table has room for more positions than 31 bits count");
    return 0;
}
kv_seqs seqs_of(const bam_kv_seqs_t& s) { return kv_seqs{s.d_starts, s.d_lens, s.d_table, s.table_stride, (uint32_t)s.n_seqs, (uint32_t)s.n_rows, (uint32_t)s.table_width}; }
bool whole_pieces(const void* p, int64_t row, int64_t head) { return ((uintptr_t)p & 15) == 0 && row % 8 == 0 && head % 8 == 0; }

} // namespace

extern "C" {

int bam_kv_create(bam_kv_t** out, bam_array_t* a, uint64_t first_page, uint64_t n_blocks, uint32_t n_heads, uint32_t dim, int f16)
{
    if (!out || !a) return fail(EINVAL, "bam_kv_create: null argument");
    *out = nullptr;
    if (!n_heads || !n_blocks) return fail(EINVAL, "bam_kv_create: no heads or no blocks");
    if (!dim || dim % 16 || dim > 256) return fail(EINVAL, "bam_kv_create: head dimension must be a multiple of 16, at most 256");
    if (f16 != 0 && f16 != 1) return fail(EINVAL, "bam_kv_create: type must be 0 (bfloat16) or 1 (float16)");
    if (a->a->adt.n_ranges != 1) return fail(EINVAL, "bam_kv_create: the array must have one range");
    BAM_API_BEGIN
    const range_d_t<uint64_t>& r = a->a->h_ranges[0];
    if (r.page_start_offset) return fail(EINVAL, "bam_kv_create: the array's range must begin a page");
    const uint64_t row = 2ull * dim;
    if (r.page_size < 8 * row) return fail(EINVAL, "bam_kv_create: a page must hold eight rows of a head");
    if (n_heads > 65535 || n_blocks > 0x7fffffffull || first_page > r.page_count || n_blocks * n_heads > (r.page_count - first_page) / 2)
        return fail(EINVAL, "bam_kv_create: the blocks do not fit the array (two pages for each block and head)");
    bam_kv_t* kv = new bam_kv();
    kv->a = a;
    kv->f16 = f16;
    kv->cache_pages = r.cache.n_pages;
    kv->unheld = r.cache.fast_reads != 0;
    kv_geom& g = kv->g;
    g.r = a->a->adt.d_ranges;
    g.pages = r.pages;
    g.base = r.cache.base_addr;
    g.first_page = first_page;
    g.n_blocks = n_blocks;
    g.heads = n_heads;
    g.dim = dim;
    g.page_log = (uint32_t)r.cache.page_size_log;
    for (g.tokens_log = 3; (row << (g.tokens_log + 1)) <= r.page_size; g.tokens_log++) {}
    g.tokens = 1u << g.tokens_log;
    if (kv->cache_pages < 16 * (g.tokens < 32 ? 32 / g.tokens : 1)) { delete kv; return fail(EINVAL, "bam_kv_create: the page cache must have 16 pages, 32 where a page holds 16 tokens, 64 where it holds 8"); }
    *out = kv;
    BAM_API_END
}

void bam_kv_destroy(bam_kv_t* kv) { delete kv; }

int bam_kv_info(bam_kv_t* kv, uint64_t* out)
{
    if (!kv || !out) return fail(EINVAL, "bam_kv_info: null argument");
    out[0] = kv->g.tokens; out[1] = kv->g.n_blocks; out[2] = 2ull * kv->g.heads; out[3] = 1ull << kv->g.page_log;
    return 0;
}

int bam_kv_append(bam_kv_t* kv, const bam_kv_append_t* what, void* stream)
{
    if (!kv || !what) return fail(EINVAL, "bam_kv_append: null argument");
    const bam_kv_append_t& w = *what;
    if (int e = bad_seqs("bam_kv_append", kv, w.seqs)) return e;
    if (!w.seqs.n_rows) return 0;
    if (!w.d_k || !w.d_v || (w.d_q && (!w.d_q_out || !w.q_heads)) || (w.rot && (!w.d_cos || !w.d_sin))) return fail(EINVAL, "bam_kv_append: null argument");
    if (w.rot % 16 || w.rot > kv->g.dim) return fail(EINVAL, "bam_kv_append: the rotated part must be a multiple of 16, at most the head dimension");
    if (((uintptr_t)w.d_q_norm | (uintptr_t)w.d_k_norm | (uintptr_t)w.d_cos | (uintptr_t)w.d_sin | (uintptr_t)w.d_q_out) & 15) return fail(EINVAL, "bam_kv_append: weights, tables and output must be aligned to 16 bytes");
    if ((w.d_q_norm || w.d_k_norm) && (!(w.eps >= 0) || w.eps - w.eps != 0)) return fail(EINVAL, "bam_kv_append: eps must be finite and not negative");
    if (w.n_positions > 0x7fffffffull || (w.rot && !w.n_positions)) return fail(EINVAL, "bam_kv_append: no positions, or more than 31 bits count");
    BAM_API_BEGIN
    kv_rows io{};
    io.q = (const uint16_t*)w.d_q; io.k = (const uint16_t*)w.d_k; io.v = (const uint16_t*)w.d_v;
    io.q_row = w.q_row; io.q_head = w.q_head; io.k_row = w.k_row; io.k_head = w.k_head; io.v_row = w.v_row; io.v_head = w.v_head;
    io.q_out = (uint16_t*)w.d_q_out; io.q_norm = (const uint16_t*)w.d_q_norm; io.k_norm = (const uint16_t*)w.d_k_norm;
    io.cos = w.d_cos; io.sin = w.d_sin; io.positions = (uint32_t)w.n_positions; io.q_heads = w.q_heads; io.rot = w.rot; io.pairs = w.pairs != 0; io.eps = w.eps;
    io.aligned = whole_pieces(w.d_k, w.k_row, w.k_head) && whole_pieces(w.d_v, w.v_row, w.v_head) && (!w.d_q || whole_pieces(w.d_q, w.q_row, w.q_head));
    launch_rows<true>(kv, seqs_of(w.seqs), io, (hipStream_t)stream);
    hip_err_chk(hipGetLastError());
    BAM_API_END
}

int bam_kv_read(bam_kv_t* kv, const bam_kv_seqs_t* seqs, void* d_k, void* d_v, void* stream)
{
    if (!kv || !seqs) return fail(EINVAL, "bam_kv_read: null argument");
    if (int e = bad_seqs("bam_kv_read", kv, *seqs)) return e;
    if (!seqs->n_rows) return 0;
    if (!d_k || !d_v) return fail(EINVAL, "bam_kv_read: null argument");
    if (((uintptr_t)d_k | (uintptr_t)d_v) & 15) return fail(EINVAL, "bam_kv_read: output must be aligned to 16 bytes");
    BAM_API_BEGIN
    kv_rows io{};
    io.k = (const uint16_t*)d_k; io.v = (const uint16_t*)d_v;
    io.k_row = io.v_row = (int64_t)kv->g.heads * kv->g.dim;
    io.k_head = io.v_head = kv->g.dim;
    io.aligned = 1;
    launch_rows<false>(kv, seqs_of(*seqs), io, (hipStream_t)stream);
    hip_err_chk(hipGetLastError());
    BAM_API_END
}

int bam_kv_attend_bytes(bam_kv_t* kv, uint64_t n_seqs, uint64_t max_new, uint32_t q_heads, uint64_t max_len, uint32_t window, uint32_t sinks, uint64_t* bytes)
{
    if (!kv || !bytes) return fail(EINVAL, "bam_kv_attend_bytes: null argument");
    if (!q_heads || q_heads % kv->g.heads) return fail(EINVAL, "bam_kv_attend_bytes: heads of queries must be a multiple of the heads of keys");
    *bytes = n_seqs && max_new ? plan_of(kv, n_seqs, max_new, q_heads, max_len, window, sinks).bytes : 0;
    return 0;
}

int bam_kv_attend(bam_kv_t* kv, const bam_kv_attend_t* what, void* stream)
{
    if (!kv || !what) return fail(EINVAL, "bam_kv_attend: null argument");
    const bam_kv_attend_t& w = *what;
    if (int e = bad_seqs("bam_kv_attend", kv, w.seqs)) return e;
    if (!w.q_heads || w.q_heads % kv->g.heads) return fail(EINVAL, "bam_kv_attend: heads of queries must be a multiple of the heads of keys");
    if (!(w.scale == w.scale) || w.scale - w.scale != 0) return fail(EINVAL, "bam_kv_attend: scale must be finite");
    if (w.window > 0x7fffffffu || w.sinks > 0x7fffffffu || w.max_len > 0x7fffffffull) return fail(EINVAL, "bam_kv_attend: window, sinks and lengths are 31-bit numbers");
    if (!w.seqs.n_rows) return 0;
    if (!w.d_q || !w.d_out || !w.d_work) return fail(EINVAL, "bam_kv_attend: null argument");
    if (((uintptr_t)w.d_out | (uintptr_t)w.d_work) & 15) return fail(EINVAL, "bam_kv_attend: output and workspace must be aligned to 16 bytes");
    const uint64_t max_new = w.seqs.d_starts ? w.max_new : 1;
    if (!max_new || max_new > w.seqs.n_rows) return fail(EINVAL, "bam_kv_attend: max_new must be at least 1 and at most the number of rows");
    if (max_new * (w.q_heads / kv->g.heads) > 0x7fffffffull) return fail(EINVAL, "bam_kv_attend: more rows than 31 bits count");
    BAM_API_BEGIN
    const kv_plan p = plan_of(kv, w.seqs.n_seqs, max_new, w.q_heads, w.max_len, w.window, w.sinks);
    if (p.tiles > 0x7fffffffull / kv->g.heads || w.seqs.n_seqs > 0x7fffffffull / ((uint64_t)p.tiles * kv->g.heads) || p.items * p.splits > 0x7fffffffull || p.items * p.rows > 0x7fffffffull) return fail(EINVAL, "bam_kv_attend: more workgroups than 31 bits count");
    if (w.work_bytes < p.bytes) return fail(EINVAL, "bam_kv_attend: the workspace is smaller than bam_kv_attend_bytes says");
    kv_att a{};
    a.q = (const uint16_t*)w.d_q; a.q_row = w.q_row; a.q_head = w.q_head; a.aligned = whole_pieces(w.d_q, w.q_row, w.q_head); a.q_heads = w.q_heads; a.group = w.q_heads / kv->g.heads;
    a.scale = w.scale * 1.4426950408889634f; a.window = w.window; a.sinks = w.sinks; a.out = (uint16_t*)w.d_out; a.lse = w.d_lse;
    a.tiles = p.tiles; a.splits = p.splits; a.steps = p.steps; a.items = (uint32_t)p.items; a.max_new = (uint32_t)max_new;
    uint8_t* const at = (uint8_t*)w.d_work;
    a.left = at + p.left_at; a.part_m = (float*)(at + p.m_at); a.part_l = (float*)(at + p.l_at); a.part = (float*)(at + p.part_at);
    if (kv->f16) launch_attend<1>(kv, seqs_of(w.seqs), a, p, (hipStream_t)stream);
    else launch_attend<0>(kv, seqs_of(w.seqs), a, p, (hipStream_t)stream);
    hip_err_chk(hipGetLastError());
    BAM_API_END
}

} // extern "C"
