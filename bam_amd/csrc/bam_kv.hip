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

} // extern "C"
