// Key-value cache in the pages of an array, of the C-ABI: appending keys and values (with norms of queries and keys and the
// position rotation on the way), reading rows back, and attention of the newest tokens over what the cache holds.
#include "kv_attend.h"

namespace {

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
     * up to 4000, 1024 / 512 / 256: 30 / 28 / 34.  In 8 bits, 512 / 256: 8 of 8000 33 / 37, 24 of 9000 87 / 116, one of 262121 97 / 111; heads of 256 numbers, 8 of 8000, 63 / 54.
     */
    uint64_t splits = (kv->g.dim <= 64 || (kv->e8 && kv->g.dim <= 128) ? 512 : 256) / p.items;
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

int create(const char* name, bam_kv_t** out, bam_array_t* a, const uint64_t first_page, const uint64_t n_blocks, const uint32_t n_heads, const uint32_t dim, const int f16, const int e8,
           uint8_t* const scales, const uint64_t scales_bytes)
{
    const std::string who = name;
    if (!out || !a) return fail(EINVAL, who + ": null argument");
    *out = nullptr;
    if (!n_heads || !n_blocks) return fail(EINVAL, who + ": no heads or no blocks");
    if (!dim || dim % 16 || dim > 256) return fail(EINVAL, who + ": head dimension must be a multiple of 16, at most 256");
    if (f16 != 0 && f16 != 1) return fail(EINVAL, who + ": type must be 0 (bfloat16) or 1 (float16)");
    if (a->a->adt.n_ranges != 1) return fail(EINVAL, who + ": the array must have one range");
    BAM_API_BEGIN
    const range_d_t<uint64_t>& r = a->a->h_ranges[0];
    if (r.page_start_offset) return fail(EINVAL, who + ": the array's range must begin a page");
    const uint64_t row = e8 ? dim : 2ull * dim, least = e8 ? 16 : 8;
    if (r.page_size < least * row) return fail(EINVAL, who + (e8 ? ": a page must hold sixteen rows of a head" : ": a page must hold eight rows of a head"));
    if (n_heads > 65535 || n_blocks > 0x7fffffffull || first_page > r.page_count || n_blocks * n_heads > (r.page_count - first_page) / 2)
        return fail(EINVAL, who + ": the blocks do not fit the array (two pages for each block and head)");
    bam_kv_t* kv = new bam_kv();
    kv->a = a;
    kv->f16 = f16;
    kv->e8 = e8;
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
    g.scales = scales;
    if (e8 && (!scales || ((uintptr_t)scales & 15) || scales_bytes < 2 * n_blocks * n_heads * g.tokens)) {
        delete kv;
        return fail(EINVAL, who + ": the powers of two of the rows need a byte for each token of each page, aligned to 16");
    }
    if (kv->cache_pages < 16 * (g.tokens < 32 ? 32 / g.tokens : 1)) { delete kv; return fail(EINVAL, who + ": the page cache must have 16 pages, 32 where a page holds 16 tokens, 64 where it holds 8"); }
    *out = kv;
    BAM_API_END
}

/* ---- the sequences that go on behind a choice of beams ---- */
struct kv_order {
    const int32_t *parents, *lens, *table;
    int64_t stride;
    uint32_t width, n_old, n_new;
    const int32_t* spare;
    int32_t *lens_out, *table_out, *spare_out;
    int32_t *freed, *copies;            /* [n_old], [n_new]: the last blocks that nobody goes on with; whether a child has one of its own */
};
constexpr uint32_t ORDER_OLD = 4096, ORDER_PIECES = 512;      /* old sequences that are looked at at a time; pieces of each page that a wave has in LDS, */
static_assert(ORDER_OLD * 4 == 2 * ORDER_PIECES * 16, "in the same LDS");
/* the last block of old sequence p, if it is there and not full; `rest` tokens in it */
__device__ __forceinline__ bool last_block(const kv_geom& g, const kv_order& o, const uint32_t p, uint32_t& block, uint32_t& rest)
{
    const int32_t len = o.lens[p];
    const uint32_t i = (uint32_t)len >> g.tokens_log;
    rest = (uint32_t)len & (g.tokens - 1u);
    if (len <= 0 || !rest || i >= o.width) return false;
    block = (uint32_t)o.table[(int64_t)p * o.stride + i];
    return block < g.n_blocks;
}

/*
 * Workgroup 0, one wave: the spare blocks that are left.  The others, a wave each: head h of child i, whose last block is copied where an earlier child has the parent's; head 0 writes
 * the child's length and row of blocks besides.  Whether there is an earlier child each wave finds by itself, in the parents in front of its own: one launch, nobody waits for anybody.
 *   A page is copied by way of LDS, 8 KiB at a time, by one wave: nothing is held while the other page is waited for, and the new page needs no read (kv_cache.h, visit).  Only
 * pieces that have tokens move.  4 beams 7.1 us, the launch and a chain of looks, references and stores; 512 sequences of which 256 are copied, eight heads, pages of 8 KiB, 22 us (33 MB).
 */
template <int F16>
__global__ __launch_bounds__(64) void k_kv_reorder(const kv_geom g, const kv_order o)
{
    using namespace bam;
    __shared__ u32x4 room[2 * ORDER_PIECES];
    const uint32_t lane = threadIdx.x;
    if (blockIdx.x == 0) {
        int32_t* const first_child = (int32_t*)room;
        uint32_t n_freed = 0;
        for (uint32_t base = 0; base < o.n_old; base += ORDER_OLD) {
            const uint32_t here = o.n_old - base < ORDER_OLD ? o.n_old - base : ORDER_OLD;
            for (uint32_t x = lane; x < here; x += 64u) first_child[x] = 0x7fffffff;
            __syncthreads();
            for (uint32_t i = lane; i < o.n_new; i += 64u) {
                const uint32_t p = (uint32_t)o.parents[i] - base;
                if (p < here) atomicMin(&first_child[p], (int32_t)i);
            }
            __syncthreads();
            for (uint32_t i = lane; i < o.n_new; i += 64u) {
                const uint32_t p = (uint32_t)o.parents[i] - base;
                uint32_t block, rest;
                if (p < here) o.copies[i] = first_child[p] != (int32_t)i && last_block(g, o, base + p, block, rest);
                else if (base == 0 && (uint32_t)o.parents[i] >= o.n_old) o.copies[i] = 0;
            }
            for (uint32_t x = 0; x < here; x += 64u) {
                uint32_t block = 0, rest;
                const bool is = x + lane < here && first_child[x + lane] == 0x7fffffff && last_block(g, o, base + x + lane, block, rest);
                const uint64_t m = ballot(is);
                if (is) __hip_atomic_store(&o.freed[n_freed + popc(m & ((1ull << lane) - 1u))], (int32_t)block, __ATOMIC_RELAXED, BAM_AGENT);
                n_freed += popc(m);
            }
            __syncthreads();
        }
        wait_stores();
        uint32_t n_copies = 0;
        for (uint32_t x = 0; x < o.n_new; x += 64u) {
            const bool in = x + lane < o.n_new, is = in && o.copies[x + lane];      /* (this lane's own) */
            const uint64_t m = ballot(is);
            const uint32_t rank = n_copies + popc(m & ((1ull << lane) - 1u));
            if (in) o.spare_out[x + lane] = !is ? o.spare[x + lane] : rank < n_freed ? __hip_atomic_load(&o.freed[rank], __ATOMIC_RELAXED, BAM_AGENT) : -1;
            n_copies += popc(m);
        }
        return;
    }
    const uint32_t i = (blockIdx.x - 1u) / g.heads, head = (blockIdx.x - 1u) % g.heads;
    const int32_t parent = o.parents[i];
    const uint32_t p = (uint32_t)parent;
    if (p >= o.n_old) {
        if (head) return;
        for (uint32_t x = lane; x < o.width; x += 64u) o.table_out[(uint64_t)i * o.width + x] = -1;
        if (lane == 0) o.lens_out[i] = 0;
        return;
    }
    uint32_t block = 0, rest = 0;
    bool copy = false;
    if (last_block(g, o, p, block, rest))
        for (uint32_t x = 0; x < i && !copy; x += 256u) {
            bool same = false;
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) { const uint32_t y = x + e * 64u + lane; same |= y < i && o.parents[y < i ? y : i] == parent; }
            copy = ballot(same) != 0;
        }
    const uint32_t own = copy ? (uint32_t)o.spare[i] : block;
    if (head == 0) {
        const int32_t len = o.lens[p];
        const uint32_t n = len > 0 ? ((uint32_t)len + g.tokens - 1u) >> g.tokens_log : 0u, last = copy ? n - 1u : 0xffffffffu;
        for (uint32_t x = lane; x < o.width; x += 64u) o.table_out[(uint64_t)i * o.width + x] = x >= n ? -1 : x == last ? (int32_t)own : o.table[(int64_t)p * o.stride + x];
        if (lane == 0) o.lens_out[i] = len;
    }
    if (!copy || own >= g.n_blocks) return;
    const uint64_t from = ((uint64_t)block * g.heads + head) * 2u, to = ((uint64_t)own * g.heads + head) * 2u;      /* pages of the cache */
    const bool e8 = g.scales != nullptr;
    /* pieces of a page, of eight tokens' values; those of `rest` tokens */
    const uint32_t pieces = g.tokens * g.dim / (e8 ? 16u : 8u), eight = e8 ? g.dim / 2u : g.dim, v_pieces = (rest + 7u) / 8u * eight;
    const u32x4 lost = e8 ? u32x4{0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu} : F16 ? u32x4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u} : u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
    /* the powers of two of the rows, while their page is held: of one that could not be had (`not_had`, as visit has it), neither the numbers nor their powers change, then or later */
    uint32_t not_had = 0;
    const bool has = e8 && lane < rest;
    const uint8_t its[2] = {has ? g.scales[from * g.tokens + lane] : (uint8_t)0, has ? g.scales[(from + 1u) * g.tokens + lane] : (uint8_t)0};      /* (of the first 64 tokens: on their way while the source is looked for) */
    auto powers = [&](const uint32_t part) {
        if (has) g.scales[(to + part) * g.tokens + lane] = its[part];
        for (uint32_t t = lane + 64u; t < rest; t += 64u) g.scales[(to + part) * g.tokens + t] = g.scales[(from + part) * g.tokens + t];
    };
    for (uint32_t x0 = 0; x0 < pieces; x0 += ORDER_PIECES) {
        auto wanted = [&](const uint32_t part, const uint32_t x) { return part ? x < v_pieces : x < pieces && place_in(g, x & (g.tokens - 1u)) < rest; };
        auto load = [&](const uint32_t part, const uint8_t* const page) {
            const uint8_t* at[8];
            u32x4 y[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) { const uint32_t x = x0 + e * 64u + lane; at[e] = page + (wanted(part, x) ? (uint64_t)x * 16u : 0u); }
            load_pieces(at, y);
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) room[part * ORDER_PIECES + e * 64u + lane] = y[e];
        };
        auto store = [&](const uint32_t part, uint8_t* const page) {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) {
                const uint32_t x = x0 + e * 64u + lane;
                if (wanted(part, x)) st16_sys(page + (uint64_t)x * 16u, room[part * ORDER_PIECES + e * 64u + lane]);
            }
        };
        const uint32_t none = visit<false>(g, g.first_page + from, false, false, [&](uint8_t* keys, uint8_t* values) {
            if (keys) load(0, keys);
            if (values) load(1, values);
        });
        if (__builtin_expect(none != 0, 0))
            for (uint32_t x = lane; x < ORDER_PIECES; x += 64u) {
                if (none & 1u) room[x] = lost;
                if (none & 2u) room[ORDER_PIECES + x] = lost;
            }
        /* (behind the first part, the page holds what this call has put there) */
        not_had |= visit<true>(g, g.first_page + to, x0 == 0, true, [&](uint8_t* keys, uint8_t* values) {
            if (e8 && x0 == 0) {
                if (keys) powers(0);
                if (values) powers(1);
            }
            if (keys && !(not_had & 1u)) store(0, keys);
            if (values && !(not_had & 2u)) store(1, values);
        });
    }
}

} // namespace

extern "C" {

int bam_kv_create(bam_kv_t** out, bam_array_t* a, uint64_t first_page, uint64_t n_blocks, uint32_t n_heads, uint32_t dim, int f16)
{
    return create("bam_kv_create", out, a, first_page, n_blocks, n_heads, dim, f16, 0, nullptr, 0);
}

int bam_kv_create_e4m3(bam_kv_t** out, bam_array_t* a, uint64_t first_page, uint64_t n_blocks, uint32_t n_heads, uint32_t dim, int f16, uint8_t* d_scales, uint64_t scales_bytes)
{
    return create("bam_kv_create_e4m3", out, a, first_page, n_blocks, n_heads, dim, f16, 1, d_scales, scales_bytes);
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
    if (kv->e8) kv8_rows(kv, seqs_of(w.seqs), io, true, (hipStream_t)stream);
    else launch_rows<0, true>(kv, seqs_of(w.seqs), io, (hipStream_t)stream);
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
    if (kv->e8) kv8_rows(kv, seqs_of(*seqs), io, false, (hipStream_t)stream);
    else launch_rows<0, false>(kv, seqs_of(*seqs), io, (hipStream_t)stream);
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
    if (kv->e8) kv8_attend(kv, seqs_of(w.seqs), a, p, (hipStream_t)stream);
    else if (kv->f16) launch_attend<1, 0>(kv, seqs_of(w.seqs), a, p, (hipStream_t)stream);
    else launch_attend<0, 0>(kv, seqs_of(w.seqs), a, p, (hipStream_t)stream);
    hip_err_chk(hipGetLastError());
    BAM_API_END
}

int bam_kv_reorder(bam_kv_t* kv, const bam_kv_reorder_t* what, void* stream)
{
    if (!kv || !what) return fail(EINVAL, "bam_kv_reorder: null argument");
    const bam_kv_reorder_t& w = *what;
    if (!w.n_new) return 0;
    if (!w.d_parents || !w.d_lens || !w.d_table || !w.d_spare || !w.d_lens_out || !w.d_table_out || !w.d_spare_out || !w.d_work) return fail(EINVAL, "bam_kv_reorder: null argument");
    if (!w.n_old || w.n_old > 0x7fffffffull || w.n_new > 0x7ffffffeull / kv->g.heads) return fail(EINVAL, "bam_kv_reorder: no old sequences, or more sequences than 31 bits count");
    if (w.table_width == 0 || w.table_width > 0x7fffffffull || w.table_stride < 0) return fail(EINVAL, "bam_kv_reorder: table of no width, or with its rows in reverse");
    if (w.table_width > 0x7ffffc00ull >> kv->g.tokens_log) return fail(EINVAL, "bam_kv_reorder: the table has room for more positions than 31 bits count");
    if (((uintptr_t)w.d_work & 3) || w.work_bytes / 4 < w.n_old + w.n_new) return fail(EINVAL, "bam_kv_reorder: the workspace must be aligned, and have 4 bytes for each sequence");
    BAM_API_BEGIN
    kv_order o{};
    o.parents = w.d_parents; o.lens = w.d_lens; o.table = w.d_table; o.stride = w.table_stride; o.width = (uint32_t)w.table_width; o.n_old = (uint32_t)w.n_old; o.n_new = (uint32_t)w.n_new;
    o.spare = w.d_spare; o.lens_out = w.d_lens_out; o.table_out = w.d_table_out; o.spare_out = w.d_spare_out;
    o.freed = (int32_t*)w.d_work; o.copies = o.freed + w.n_old;
    const dim3 grid(1u + o.n_new * kv->g.heads);
    if (kv->f16) hipLaunchKernelGGL(k_kv_reorder<1>, grid, dim3(64), 0, (hipStream_t)stream, kv->g, o);
    else hipLaunchKernelGGL(k_kv_reorder<0>, grid, dim3(64), 0, (hipStream_t)stream, kv->g, o);
    hip_err_chk(hipGetLastError());
    BAM_API_END
}

} // extern "C"
