// attention.hip -- attention over the paged pool for a batch that shares a prefix:
// which blocks of attention_kernels.h take what, argument checks and launches.
#include "attention_kernels.h"

namespace kvec {

struct AttnPlan {
    bool flat, flat_tile, own_tile;
    uint32_t parts_flat, parts_own, tiles_flat, req_tiles, first;
    uint64_t rows, tiles_own, blocks_flat, blocks;
    // pools with block scales: K/V heads of a wave, groups of a block's, runs, and see AttnArgs
    uint32_t wave_heads, run_heads, groups, run_keys, few_keys, runs_flat, runs_own;
    bool direct() const { return parts_flat + parts_own == 1; }
    int64_t bytes(int64_t dim) const {
        return direct() ? 0 : int64_t(uint64_t(parts_flat + parts_own) * rows * (uint64_t(dim) * 4 + 8)) + 16;
    }
};

// Which blocks take which part, and in how many splits of the keys.
inline AttnPlan plan_attention(const kvec_attention* s) {
    AttnPlan p{};
    const uint64_t group = uint64_t(s->heads / s->kv_heads), N = uint64_t(s->tokens), B = uint64_t(s->batch);
    const uint64_t max_q = s->cu_q ? min(uint64_t(s->max_q), N) : 1, Hk = uint64_t(s->kv_heads);
    const uint64_t req_rows = max_q * group, all_rows = N * group, prefix = uint64_t(s->prefix);
    const uint64_t cap = uint64_t(s->pages_per_seq) * uint64_t(s->page_tokens);
    const uint64_t len = s->max_len > 0 && uint64_t(s->max_len) < cap ? uint64_t(s->max_len) : cap;
    p.rows = N * uint64_t(s->heads);
    // Splits of `keys` keys: a block's time falls with them, the writing and
    // joining of partial results (rows * dim) grows with them, so about the root
    // of the quotient; no more than two blocks a compute unit, and 128 keys each.
    // Measured, bf16, us: 2048 rows behind 8192 keys 49 (32 splits), 42 (16);
    // 512 rows behind 4096 22 (32), 19 (16); 128 rows behind 512 16.6 (1), 11.7
    // (4), 12.2 (8); one request of 32768 keys 43 (16), 33.5 (64).
    auto splits = [&](uint64_t blocks, uint64_t keys, uint64_t room) {
        blocks = blocks ? blocks : 1;
        uint64_t n = min((room + blocks / 2) / blocks, 512 / blocks);
        if (n > keys / 128) n = keys / 128;
        while (n > 1 && n * n * p.rows * uint64_t(s->dim) > keys * 6400) --n;
        return uint32_t(n < 1 ? 1 : n > 256 ? 256 : n);
    };
    // A request's rows as tiles of 128, which read the prefix with the own keys,
    // or as stream blocks of 16 behind the shared part: by the keys that either's
    // blocks go through, a stream block's at three fifths of a tile's.  Measured,
    // bf16, four query heads to a K/V head, us (stream, tile): 64 requests of
    // 1024 own keys with 16 rows 36, 41, with 64 rows 79, 42; 64 of 500 behind
    // 4096 with 64 rows 110, 149, with 128 rows 182, 156; behind 512 with 48
    // rows 60, 44.  Where few requests leave compute units idle the stream
    // blocks, being more, can be ahead for longer (16 of 500 behind 4096 with
    // 128 rows 57, 62).  All of that is for requests of equally many rows.  The
    // choice is one for the call, by the longest request, so in a step of few long
    // and many short ones the short ones go through the prefix by tiles of their
    // own: 255 requests of one token and one of 512 behind 8192 take 1125 us, in two
    // calls 160 and 106; 60 and four 538, in two calls 45 and 299.
    // Pools with block scales, whose stream blocks are runs, go by the same: us (runs, tiles),
    // 8 bits, 64 requests of 1024 own keys with 16 rows a K/V head 60, 61, with 24 rows 78,
    // 61, with 64 rows 139, 61; 4 bits 50, 52; 61, 52; 111, 54; heads of 64 with 16 rows 38, 51;
    // 64 of 4096 with 32 rows of one head 58, 35; 64 of 512 behind 4096 with 32 rows 110, 169,
    // with 64 rows 185, 165.  It is wrong for the last, and behind 512 (32 rows 72, 51; runs
    // are taken).
    const uint64_t own_keys = len > prefix ? len - prefix : 0;
    const uint64_t by16 = (req_rows + kStreamRows - 1) / kStreamRows, by128 = (req_rows + kTileRows - 1) / kTileRows;
    p.own_tile = 0.6 * double(own_keys) * double(by16) + double(prefix) * double(req_rows) / kTileRows >
                 double(prefix + own_keys) * double(by128);
    p.req_tiles = uint32_t(by16);
    p.tiles_own = p.own_tile ? min(all_rows / kTileRows + B, B * by128) : B * by16;
    const uint64_t own = p.tiles_own * Hk;
    p.flat = prefix > 0 && !p.own_tile;
    if (p.flat) {
        p.first = uint32_t(prefix);
        // Measured, us (stream, tile): 64 rows behind 512 12.2, 13.3, behind 4096
        // 24.8, 19.4; 128 rows behind 512 15.0, 14.9; 32 rows behind 4096 18.4, 16.9,
        // behind 512 11.3, 12.3.
        p.flat_tile = all_rows > 2 * kStreamRows;
        const uint64_t bm = p.flat_tile ? kTileRows : kStreamRows;
        p.tiles_flat = uint32_t((all_rows + bm - 1) / bm);
        // Tile blocks of the shared part leave places to the stream blocks beside
        // them, as the two take time: a tile's keys by the matrix units, a
        // request's by memory, whose bytes a value count in.  Measured, us, with
        // all places and with their share: 256 requests of 1024 own fp8 keys
        // behind 32768 208 (8 splits), 192 (6); 128 of 512 bf16 ones behind
        // 16384 86 (16), 76 (8); 256 of 512 behind 8192, eight K/V heads, 127
        // (5), 114 (3); no own keys, behind 32768, 173 (8), 187 (6).
        const double value_bytes = s->pool_dtype == KVEC_BLOCK_E2M1 ? 0.5 : s->pool_dtype == s->dtype ? 2.0 : 1.0;
        uint64_t room = 512;
        if (p.flat_tile) {
            const double shared = 2.0 * double(p.tiles_flat) * double(prefix);
            const double beside = double(B * by16) * double(own_keys) * value_bytes;
            room = uint64_t(512.0 * shared / (shared + beside));
        }
        p.parts_flat = splits(uint64_t(p.tiles_flat) * Hk, prefix, room);
    }
    p.parts_own = splits(own, len > p.first ? len - p.first : 1, 512);
    p.blocks_flat = p.flat ? uint64_t(p.tiles_flat) * Hk * p.parts_flat : 0;
    p.blocks = p.blocks_flat + own * p.parts_own;
    if (const int bits = block_bits(s->pool_dtype)) {
        // Runs: waves of two heads where the codes have 4 bits and each head's rows of a
        // request are no more than eight; blocks of four times as many heads, or as there
        // are; eight pairs of rows and runs on as many XCDs.
        p.wave_heads = bits == 4 && Hk >= 2 && req_rows <= kStreamRows / 2 ? 2 : 1;
        const uint64_t rows = kStreamRows / p.wave_heads, most = 4 * p.wave_heads;
        p.run_heads = p.wave_heads;
        while (p.run_heads < most && p.run_heads < Hk) p.run_heads *= 2;
        p.groups = uint32_t((Hk + p.run_heads - 1) / p.run_heads);
        const uint64_t subs = most / p.run_heads;         // times 32 keys, each with partial results of its own
        p.few_keys = uint32_t(64 * subs);
        auto run_blocks = [&](uint64_t tiles, uint64_t runs) { return (tiles * runs + 7) / 8 * 8 * p.groups; };
        auto runs = [&](uint64_t tiles, uint64_t keys, uint32_t* count) {
            // One request has all its runs: two blocks a compute unit, once the card over.  Of
            // several most are shorter than the longest, and runs that they do not have end at
            // once: three times over.  Measured, us, by blocks (512, 768, 1024, 1536; all runs
            // counted, 32 / 8 heads of 128): one request of 262144 keys, 8 bits, 106, 124, 113,
            // 112, 4 bits (512 parts at most) 65, 66, 64, 65; 64 of up to 8192, 8 bits, 142, 118,
            // 149, 130, 4 bits 103, 82, 97, 86; 256 of up to 4096, 4 bits, 203, 199, 188, 160.
            // Requests that are all equally long would have fewer: 2 of 131072, 8 bits, 105,
            // 124, 112, 119; 64 of 4096 102, 119, 108, 115, 4 bits 62, 68, 68, 78.  So would heads
            // of 256, of which one block fits: 16 / 4 of them, 64 of 4096, 137, 147, 155, 176, of
            // up to 4096 123, 105, 108, 115.  (A prefix's runs are counted as several requests'.)
            // 64 keys a wave of a run, 512 parts of a row.
            uint64_t n = (B > 1 ? 1536 : 512) / (tiles * p.groups);
            if (n > keys / p.few_keys) n = keys / p.few_keys;
            if (n > 512 / subs) n = 512 / subs;
            n = n < 1 ? 1 : n;
            *count = uint32_t(n);
            return uint32_t((keys + n - 1) / n + kStreamKeys - 1) / kStreamKeys * kStreamKeys;
        };
        if (p.flat && !p.flat_tile) {
            p.tiles_flat = uint32_t((all_rows + rows - 1) / rows);
            runs(p.tiles_flat, prefix, &p.runs_flat);
            p.parts_flat = uint32_t(p.runs_flat * subs);
            p.blocks_flat = run_blocks(p.tiles_flat, p.runs_flat);
        }
        if (!p.own_tile) {
            p.req_tiles = uint32_t((req_rows + rows - 1) / rows);
            p.tiles_own = B * p.req_tiles;
            p.run_keys = runs(p.tiles_own, len > p.first ? len - p.first : 1, &p.runs_own);
            p.parts_own = uint32_t(p.runs_own * subs);
            p.blocks = p.blocks_flat + run_blocks(p.tiles_own, p.runs_own);
        }
    }
    return p;
}

inline int check_attention(const kvec_attention* s, const char* fn) {
    if (!s) return set_error(KVEC_EINVAL, "%s: null descriptor", fn);
    if (s->tokens < 0 || s->batch < 0 || s->heads < 1 || s->kv_heads < 1 || s->heads % s->kv_heads || s->dim < 1 ||
        s->pages_per_seq < 1 || s->pool_pages < 0 || s->prefix < 0)
        return set_error(KVEC_EINVAL, "%s: bad sizes", fn);
    if (s->dtype != KVEC_BF16 && s->dtype != KVEC_F16) return set_error(KVEC_EINVAL, "%s: dtype %d", fn, s->dtype);
    const bool blocks = block_bits(s->pool_dtype) != 0;
    if (s->pool_dtype != s->dtype && s->pool_dtype != KVEC_FP8_E4M3 && !blocks)
        return set_error(KVEC_EINVAL, "%s: pool_dtype %d is neither dtype, fp8 nor one with block scales", fn, s->pool_dtype);
    if (s->pool_dtype != KVEC_FP8_E4M3 && (s->k_scale || s->v_scale))
        return set_error(KVEC_EINVAL, "%s: scales are an fp8 pool's", fn);
    const int unit = blocks ? kScaleBlock : s->pool_dtype == KVEC_FP8_E4M3 ? 16 : 8;
    if (s->dim > 256 || s->dim % unit)
        return set_error(KVEC_EUNSUPPORTED, "%s: dim=%d must be a multiple of %d up to 256", fn, s->dim, unit);
    if (s->page_tokens < 1 || (s->page_tokens & (s->page_tokens - 1)))
        return set_error(KVEC_EINVAL, "%s: page_tokens=%d must be a power of two", fn, s->page_tokens);
    if (s->pool_pages > (int64_t(1) << 31) / s->page_tokens ||
        int64_t(s->pages_per_seq) * s->page_tokens >= (int64_t(1) << 31) - 1024)
        return set_error(KVEC_EUNSUPPORTED, "%s: positions or slots past 2^31", fn);
    if (s->prefix > int64_t(s->pages_per_seq) * s->page_tokens)
        return set_error(KVEC_EINVAL, "%s: prefix=%lld past the page table", fn, (long long)s->prefix);
    if (s->cu_q ? s->max_q < 1 && s->tokens > 0 : s->tokens != s->batch)
        return set_error(KVEC_EINVAL, "%s: max_q=%d tokens=%lld batch=%d", fn, s->max_q, (long long)s->tokens, s->batch);
    if (!(s->scale >= 0.0f) || s->scale > kFloatMax / kLog2e)
        return set_error(KVEC_EINVAL, "%s: scale must not be negative, and finite times log2(e)", fn);
    if (s->tokens * s->heads >= (int64_t(1) << 31) / 64 || int64_t(s->batch) * s->pages_per_seq >= (int64_t(1) << 31))
        return set_error(KVEC_EUNSUPPORTED, "%s: too many rows for one launch", fn);
    return KVEC_OK;
}

// The plan, and that its launches can be.
inline int checked_plan(const kvec_attention* s, const char* fn, AttnPlan* p) {
    *p = plan_attention(s);
    if (!launchable(p->blocks, kAB) || (!p->direct() && !launchable(p->rows, kAB)))
        return set_error(KVEC_EUNSUPPORTED, "%s: too many blocks for one launch", fn);
    return KVEC_OK;
}

}  // namespace kvec

using namespace kvec;

extern "C" int64_t kvec_prefix_attention_workspace(const kvec_attention* s) {
    static const char* fn = "kvec_prefix_attention_workspace";
    if (check_attention(s, fn)) return -1;
    if (s->tokens == 0 || s->batch == 0) return 0;
    AttnPlan p;
    return checked_plan(s, fn, &p) ? -1 : p.bytes(s->dim);
}

extern "C" int kvec_prefix_attention(const kvec_attention* s, void* workspace, int64_t workspace_bytes, void* stream) {
    static const char* fn = "kvec_prefix_attention";
    int rc = check_attention(s, fn);
    if (rc) return rc;
    if (s->tokens == 0 || s->batch == 0) return KVEC_OK;
    if (!s->q || !s->out || !s->pool || !s->page_table || !s->seq_lens || (s->prefix && !s->prefix_pages))
        return set_error(KVEC_EINVAL, "%s: null array", fn);
    if (!aligned16(s->pool)) return set_error(KVEC_EINVAL, "%s: pool not 16-byte aligned", fn);
    const int64_t str[4] = {s->q_stride, s->q_head_stride, s->o_stride, s->o_head_stride};
    for (int64_t x : str)
        if (x < 0 || x > (int64_t(1) << 40)) return set_error(KVEC_EINVAL, "%s: stride %lld", fn, (long long)x);
    if (rows_overlap(s->tokens, s->o_stride, s->heads, s->o_head_stride, s->dim))
        return set_error(KVEC_EINVAL, "%s: rows of out overlap", fn);
    AttnPlan p;
    if ((rc = checked_plan(s, fn, &p))) return rc;
    const int64_t need = p.bytes(s->dim);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return set_error(KVEC_EINVAL, "%s: workspace of %lld bytes, 16-byte aligned, wanted", fn, (long long)need);
    const uint64_t rec = 2 * half_bytes(s->kv_heads, s->dim, s->pool_dtype);
    if (rec / 2 >= (block_bits(s->pool_dtype) ? kMaxBlockHalf : uint64_t(1) << 30))
        return set_error(KVEC_EUNSUPPORTED, "%s: token record too large", fn);
    {
        auto span = [&](const void* q, int64_t st, int64_t hs, const char* name) {
            return Span{q, uint64_t((s->tokens - 1) * st + (s->heads - 1) * hs + s->dim) * 2, name, -1};
        };
        const Span w[2] = {span(s->out, s->o_stride, s->o_head_stride, "out"),
                           {workspace, uint64_t(need), "workspace", -1}};
        const Span r[6] = {span(s->q, s->q_stride, s->q_head_stride, "q"),
                           {s->pool, uint64_t(s->pool_pages) * uint64_t(s->page_tokens) * rec, "pool", -1},
                           {s->page_table, uint64_t(s->batch) * uint64_t(s->pages_per_seq) * 4, "page_table", -1},
                           {s->seq_lens, uint64_t(s->batch) * 4, "seq_lens", -1},
                           {s->cu_q, s->cu_q ? uint64_t(s->batch + 1) * 4 : 0, "cu_q", -1},
                           {s->prefix_pages,
                            s->prefix ? uint64_t((s->prefix + s->page_tokens - 1) / s->page_tokens) * 4 : 0,
                            "prefix_pages", -1}};
        if ((rc = check_no_alias(w, 2, r, 6, fn))) return rc;
    }
    AttnArgs a{};
    a.q = (const uint8_t*)s->q;
    a.out = (uint8_t*)s->out;
    a.qs = s->q_stride, a.qh = s->q_head_stride, a.os = s->o_stride, a.oh = s->o_head_stride;
    a.pool = (const uint8_t*)s->pool;
    a.table = s->page_table;
    a.prefix_pages = s->prefix_pages;
    a.seq_lens = s->seq_lens;
    a.cu = s->cu_q;
    a.k_scale = s->k_scale;
    a.v_scale = s->v_scale;
    a.rec = uint32_t(rec);
    a.token_bytes = uint32_t(rec / 2);
    a.scales = uint32_t(uint64_t(s->kv_heads) * uint64_t(s->dim) * uint64_t(block_bits(s->pool_dtype)) / 8);
    a.tokens = uint32_t(s->tokens);
    a.batch = uint32_t(s->batch);
    a.heads = uint32_t(s->heads);
    a.kv_heads = uint32_t(s->kv_heads);
    a.group = a.heads / a.kv_heads;
    a.dim = uint32_t(s->dim);
    a.width = uint32_t(s->pages_per_seq);
    while ((1 << a.shift) < s->page_tokens) ++a.shift;
    a.pool_pages = uint32_t(s->pool_pages);
    a.cap = a.width << a.shift;
    a.max_rows = uint32_t(s->cu_q ? min(int64_t(s->max_q), s->tokens) : 1) * a.group;
    a.prefix = uint32_t(s->prefix);
    a.first = p.first;
    a.parts_flat = p.parts_flat;
    a.parts_own = p.parts_own;
    a.blocks_flat = uint32_t(p.blocks_flat);
    a.by_group = make_fastdiv(a.group);
    a.by_req_tiles = make_fastdiv(p.req_tiles);
    a.by_flat = make_fastdiv(p.parts_flat ? p.parts_flat : 1);
    a.by_own = make_fastdiv(p.parts_own);
    a.by_heads_flat = make_fastdiv(a.kv_heads * a.by_flat.d);
    a.by_heads_own = make_fastdiv(a.kv_heads * p.parts_own);
    if (p.run_heads) {
        a.run_heads = p.run_heads;
        a.run_keys = p.run_keys;
        a.few_keys = p.few_keys;
        a.by_groups = make_fastdiv(p.groups);
        a.by_tiles_flat = make_fastdiv(p.tiles_flat ? p.tiles_flat : 1);
        a.by_tiles_own = make_fastdiv(uint32_t(p.tiles_own));
        a.by_runs_flat = make_fastdiv(p.runs_flat ? p.runs_flat : 1);
        a.by_runs_own = make_fastdiv(p.runs_own ? p.runs_own : 1);
    }
    a.direct = p.direct();
    a.scale = s->scale;
    a.wide_q = aligned16(s->q) && s->q_stride % 8 == 0 && s->q_head_stride % 8 == 0;
    a.wide_o = aligned16(s->out) && s->o_stride % 8 == 0 && s->o_head_stride % 8 == 0;
    if (need) {
        a.ws_o = (float*)workspace;
        a.ws_ml = (f32x2*)((uint8_t*)workspace + uint64_t(p.parts_flat + p.parts_own) * p.rows * uint64_t(s->dim) * 4);
    }
    const bool fp8 = s->pool_dtype == KVEC_FP8_E4M3, bf = s->dtype == KVEC_BF16;
    const int bits = block_bits(s->pool_dtype);
    AttnFn f = bits ? pick_block_attn(bf, bits, p.flat_tile, p.own_tile, int(p.wave_heads), s->dim)
               : bf ? (fp8 ? pick_attn<__bf16, kFp8>(p.flat_tile, p.own_tile, s->dim)
                           : pick_attn<__bf16, kPlain>(p.flat_tile, p.own_tile, s->dim))
                    : (fp8 ? pick_attn<_Float16, kFp8>(p.flat_tile, p.own_tile, s->dim)
                           : pick_attn<_Float16, kPlain>(p.flat_tile, p.own_tile, s->dim));
    hipLaunchKernelGGL(f, dim3(unsigned(p.blocks)), dim3(kAB), 0, as_stream(stream), a);
    if ((rc = check_launch(fn)) || p.direct()) return rc;
    uint32_t lanes = 16, cut = 1;
    while (lanes * 4 < a.dim) lanes *= 2;
    // Runs can be many: a row by several blocks where rows are few and its parts take several passes.
    // Measured: 32 rows of 128 with 512 parts 34 us by one, 11.3 by eight (8.5 now).
    while (p.run_heads && p.rows * cut < 512 && lanes > 4 && a.parts_flat + a.parts_own > kAB / lanes) lanes /= 2, cut *= 2;
    const dim3 grid(unsigned(p.rows), cut);
    if (bf) hipLaunchKernelGGL(attn_join_kernel<__bf16>, grid, dim3(kAB), 0, as_stream(stream), a, lanes);
    else hipLaunchKernelGGL(attn_join_kernel<_Float16>, grid, dim3(kAB), 0, as_stream(stream), a, lanes);
    return check_launch(fn);
}
