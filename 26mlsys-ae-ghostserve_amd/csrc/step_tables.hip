// step_tables.hip -- a step's page table rows and slots from request lengths.
//
// With P tokens a page, request b holds h_b = ceil(cached_b / P) pages and ends
// with e_b = ceil((cached_b + new_b) / P), both at most the row's width, so it
// takes n_b = e_b - h_b pages of the free list from o_b = sum of n over the
// requests before it.  Entry j of its row is kept (j < h_b), free[o_b + j - h_b]
// (j < e_b), or -1.  Token t of the step belongs to the request with
// cu_b <= t < cu_(b+1), cu the sums of new, and the page it falls in is read
// from the row's kept part or from the free list, never from an entry that
// this launch writes: so rows and tokens need no order between them, and the
// whole step is one launch.
//
// Nothing here is long enough to be bound by memory; a launch and a scan's
// latency are what is paid.  Every block forms the sums that it needs by
// itself from the lengths (a few KB, in cache after the first block) instead
// of waiting for another: block 0 writes the lengths' sums, the next blocks
// clear and fill table rows, the rest place 1024 tokens each.  Measured: 16
// decoding requests 3.7 us (any small launch takes 3.5); 1024 requests, rows of 2048
// pages, 7.7 us.
#include "kvec_internal.h"

namespace kvec {

constexpr int kSTB = 256;                 // threads of a block
constexpr int kReqs = 4 * kSTB;           // requests scanned at a time
constexpr int kTokensPerBlock = 4 * kSTB;
constexpr uint32_t kIntMax = 0x7FFFFFFFu;

struct StepArgs {
    int32_t* table;
    const int32_t* cached;
    const int32_t* fresh;
    const int32_t* free_pages;
    int32_t* slots;
    int32_t* positions;
    int32_t* cu;
    int32_t* lens;
    int32_t* taken;
    uint32_t batch, width, shift, pool_pages, n_free, max_tokens;
    uint32_t rows_per_block, row_blocks;
    FastDiv div_width;                    // by groups of 4 entries (rows of whole groups) or by entries
};

// Sums that stay at 2^31 - 1: associative on values of 31 bits.
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kIntMax); }

struct Req {
    uint32_t cached, fresh, held, need;
};

__device__ __forceinline__ Req request(const StepArgs& a, uint32_t b) {
    Req r{0, 0, 0, 0};
    if (b < a.batch) {
        r.cached = uint32_t(max(a.cached[b], 0));
        r.fresh = uint32_t(max(a.fresh[b], 0));
        const uint32_t up = (1u << a.shift) - 1;
        r.held = min((r.cached + up) >> a.shift, a.width);
        r.need = min((sat_add(r.cached, r.fresh) + up) >> a.shift, a.width) - r.held;
    }
    return r;
}

// Exclusive sums over the block of one value a thread; *total gets the sum.
template <bool SAT>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* lds, uint32_t* total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d, 64);
        if (lane >= uint32_t(d)) x = SAT ? sat_add(x, y) : x + y;
    }
    __syncthreads();                      // lds may still be read from the call before
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSTB / 64; ++w) {
        if (w == wave) before = all;
        all = SAT ? sat_add(all, lds[w]) : all + lds[w];
    }
    *total = all;
    const uint32_t up = __shfl_up(x, 1, 64);
    const uint32_t excl = lane ? up : 0u;
    return SAT ? sat_add(before, excl) : before + excl;
}

__device__ __forceinline__ int32_t free_page(const StepArgs& a, uint32_t i) {
    return i < a.n_free ? a.free_pages[i] : -1;
}

__device__ void step_lengths(const StepArgs& a, uint32_t* lds) {
    uint32_t cu = 0, pages = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += kSTB) {
        const uint32_t b = b0 + threadIdx.x;
        const Req r = request(a, b);
        uint32_t all, allp;
        const uint32_t at = sat_add(cu, block_scan<true>(r.fresh, lds, &all));
        block_scan<false>(r.need, lds, &allp);
        if (b < a.batch) {
            a.cu[b] = int32_t(at);
            a.lens[b] = int32_t(sat_add(r.cached, r.fresh));
        }
        cu = sat_add(cu, all);
        pages += allp;
    }
    if (threadIdx.x == 0) {
        a.cu[a.batch] = int32_t(cu);
        *a.taken = int32_t(pages);
    }
}

// Rows r0 .. of the table: what follows the pages that they hold.
__device__ void step_rows(const StepArgs& a, uint32_t r0, uint32_t* lds, uint32_t (*row)[kSTB]) {
    uint32_t before = 0;
    for (uint32_t b = threadIdx.x; b < r0; b += kSTB) before += request(a, b).need;
    uint32_t base, unused;
    block_scan<false>(before, lds, &base);
    const uint32_t n = min(a.rows_per_block, a.batch - r0);
    const Req r = request(a, threadIdx.x < n ? r0 + threadIdx.x : a.batch);
    const uint32_t off = base + block_scan<false>(r.need, lds, &unused);
    row[0][threadIdx.x] = r.held;
    row[1][threadIdx.x] = r.held + r.need;
    row[2][threadIdx.x] = off - r.held;   // entry j takes free[off - held + j]
    __syncthreads();
    int32_t* t = a.table + uint64_t(r0) * a.width;
    auto entry = [&](uint32_t i, uint32_t j) { return j < row[1][i] ? free_page(a, row[2][i] + j) : -1; };
    if ((a.width & 3) == 0 && (reinterpret_cast<uintptr_t>(a.table) & 15) == 0) {
        typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
        const uint32_t groups = a.width / 4;
        for (uint32_t e = threadIdx.x; e < n * groups; e += kSTB) {
            const uint32_t i = fdiv(e, a.div_width), j = (e - i * groups) * 4;
            if (j + 4 <= row[0][i]) continue;
            i32x4 v = {entry(i, j), entry(i, j + 1), entry(i, j + 2), entry(i, j + 3)};
            int32_t* p = t + uint64_t(i) * a.width + j;
            if (j >= row[0][i]) {
                *reinterpret_cast<i32x4*>(p) = v;
            } else {
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x)
                    if (j + x >= row[0][i]) p[x] = v[x];
            }
        }
    } else {
        for (uint32_t e = threadIdx.x; e < n * a.width; e += kSTB) {
            const uint32_t i = fdiv(e, a.div_width), j = e - i * a.width;
            if (j >= row[0][i]) t[e] = entry(i, j);
        }
    }
}

// Tokens t0 .. t0 + 1023: the requests are scanned 1024 at a time until the
// block's last token is placed.
__device__ void step_tokens(const StepArgs& a, uint32_t t0, uint32_t* lds, uint32_t* cu_l, uint32_t* off_l) {
    const uint32_t t1 = min(t0 + kTokensPerBlock, a.max_tokens);
    uint32_t cu = 0, pages = 0;
    for (uint32_t b0 = 0; b0 < a.batch && cu < t1; b0 += kReqs) {
        Req r[4];
        uint32_t sf = 0, sn = 0, allf, alln;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            r[x] = request(a, b0 + threadIdx.x * 4 + x);
            sf = sat_add(sf, r[x].fresh);
            sn += r[x].need;
        }
        uint32_t f = sat_add(cu, block_scan<true>(sf, lds, &allf));
        uint32_t o = pages + block_scan<false>(sn, lds, &alln);
        // request x of the chunk has the tokens from cu_l[x] on
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            cu_l[threadIdx.x * 4 + x] = f;
            off_l[threadIdx.x * 4 + x] = o;
            f = sat_add(f, r[x].fresh);
            o += r[x].need;
        }
        cu = sat_add(cu, allf);
        pages += alln;
        __syncthreads();
        const uint32_t lo = cu_l[0];
        for (uint32_t t = max(t0, lo) + threadIdx.x; t < min(t1, cu); t += kSTB) {
            uint32_t x = 0;                       // the last request with cu_l[x] <= t
#pragma unroll
            for (uint32_t step = kReqs / 2; step; step >>= 1)
                if (cu_l[x + step] <= t) x += step;
            const Req q = request(a, b0 + x);
            const uint32_t pos = sat_add(q.cached, t - cu_l[x]);
            const uint32_t j = pos >> a.shift;
            int32_t page = -1;
            if (j < q.held) page = a.table[uint64_t(b0 + x) * a.width + j];
            else if (j < q.held + q.need) page = free_page(a, off_l[x] + j - q.held);
            const bool good = uint32_t(page) < a.pool_pages;
            a.positions[t] = int32_t(pos);
            a.slots[t] = good ? int32_t((uint32_t(page) << a.shift) | (pos & ((1u << a.shift) - 1))) : -1;
        }
        __syncthreads();                          // the chunk's sums are read
    }
    for (uint32_t t = max(t0, cu) + threadIdx.x; t < t1; t += kSTB) {
        a.positions[t] = 0;
        a.slots[t] = -1;
    }
}

__global__ __launch_bounds__(kSTB) void step_tables_kernel(StepArgs a) {
    __shared__ uint32_t lds[kSTB / 64];
    __shared__ uint32_t buf[2 * kReqs];
    const uint32_t blk = blockIdx.x;
    if (blk == 0) {
        step_lengths(a, lds);
    } else if (blk <= a.row_blocks) {
        step_rows(a, (blk - 1) * a.rows_per_block, lds, reinterpret_cast<uint32_t(*)[kSTB]>(buf));
    } else {
        step_tokens(a, (blk - 1 - a.row_blocks) * uint32_t(kTokensPerBlock), lds, buf, buf + kReqs);
    }
}

}  // namespace kvec

using namespace kvec;

extern "C" int kvec_step_tables(const kvec_step* s, void* stream) {
    static const char* fn = "kvec_step_tables";
    if (!s) return set_error(KVEC_EINVAL, "%s: null descriptor", fn);
    if (s->batch < 0 || s->pages_per_seq < 1 || s->pool_pages < 0 || s->n_free < 0 || s->max_tokens < 0)
        return set_error(KVEC_EINVAL, "%s: bad sizes", fn);
    if (s->page_tokens < 1 || (s->page_tokens & (s->page_tokens - 1)))
        return set_error(KVEC_EINVAL, "%s: page_tokens=%d must be a power of two", fn, s->page_tokens);
    if (s->pool_pages > (int64_t(1) << 31) / s->page_tokens)
        return set_error(KVEC_EUNSUPPORTED, "%s: slots past 2^31", fn);
    if (int64_t(s->batch) * s->pages_per_seq >= (int64_t(1) << 31) || s->n_free >= (int64_t(1) << 31) ||
        s->max_tokens >= (int64_t(1) << 31) - kTokensPerBlock)
        return set_error(KVEC_EUNSUPPORTED, "%s: arrays past 2^31 entries", fn);
    if (!s->cu_new || !s->taken || (s->batch && (!s->page_table || !s->cached || !s->new_tokens || !s->seq_lens)) ||
        (s->n_free && !s->free_pages) || (s->max_tokens && (!s->slots || !s->positions)))
        return set_error(KVEC_EINVAL, "%s: null array", fn);
    const uint64_t B = uint64_t(s->batch), T = uint64_t(s->max_tokens) * 4;
    const Span w[6] = {{s->page_table, B * uint64_t(s->pages_per_seq) * 4, "page_table", -1},
                       {s->slots, T, "slots", -1},
                       {s->positions, T, "positions", -1},
                       {s->cu_new, (B + 1) * 4, "cu_new", -1},
                       {s->seq_lens, B * 4, "seq_lens", -1},
                       {s->taken, 4, "taken", -1}};
    const Span r[3] = {{s->cached, B * 4, "cached", -1},
                       {s->new_tokens, B * 4, "new_tokens", -1},
                       {s->free_pages, uint64_t(s->n_free) * 4, "free_pages", -1}};
    int rc = check_no_alias(w, 6, r, 3, fn);
    if (rc) return rc;
    StepArgs a{};
    a.table = s->page_table;
    a.cached = s->cached;
    a.fresh = s->new_tokens;
    a.free_pages = s->free_pages;
    a.slots = s->slots;
    a.positions = s->positions;
    a.cu = s->cu_new;
    a.lens = s->seq_lens;
    a.taken = s->taken;
    a.batch = uint32_t(B);
    a.width = uint32_t(s->pages_per_seq);
    while ((1 << a.shift) < s->page_tokens) ++a.shift;
    a.pool_pages = uint32_t(s->pool_pages);
    a.n_free = uint32_t(s->n_free);
    a.max_tokens = uint32_t(s->max_tokens);
    // about 8192 entries a block, and no more rows than a block has threads
    a.rows_per_block = a.width >= 8192 ? 1 : 8192 / a.width;
    if (a.rows_per_block > kSTB) a.rows_per_block = kSTB;
    a.row_blocks = (a.batch + a.rows_per_block - 1) / a.rows_per_block;
    const bool wide = (a.width & 3) == 0 && (reinterpret_cast<uintptr_t>(a.table) & 15) == 0;
    a.div_width = make_fastdiv(wide ? a.width / 4 : a.width);
    const unsigned blocks = 1 + a.row_blocks + (a.max_tokens + kTokensPerBlock - 1) / kTokensPerBlock;
    hipLaunchKernelGGL(step_tables_kernel, dim3(blocks), dim3(kSTB), 0, as_stream(stream), a);
    return check_launch(fn);
}
