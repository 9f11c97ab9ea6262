// attention.hip -- attention over the paged pool for a batch that shares a prefix.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m)
//
// over the keys j that the query sees: positions up to its own, on pages inside
// the pool.  Positions below `prefix` are the same for all requests and are read
// from one list of pages; their part of the sum is computed for the rows of all
// requests together (a row: one query head of one token), so that a tile of keys
// is read once for as many rows as fill a matrix instruction, not once a
// request.  Each request's own keys are a second part; parts are joined by
// their maxima and sums, which are linear once both are brought to one maximum.
//
// Two kinds of blocks, one kernel.  Both form S^T = K Q^T and O^T += V^T P^T, keys
// along the rows of the matrix instructions and query rows along their columns: a
// lane then holds scores of one query row only, so the softmax needs one exchange
// between lane halves (or quarters) for the maximum and none for the sum, and the
// scores that a lane holds are, rounded to 16 bits, just what the second product
// wants from it (the instruction sums over keys in any order, so long as V^T comes
// in the same one: rows 4h .. and 8 + 4h .. of each 16).  V lies [key][value]
// and is needed transposed, which ds_read_b64_tr_b16 does on the way from LDS.
//
// Scores, maxima, sums and outputs are 32-bit; P is rounded to 16 bits for the
// second product (half a step of the inputs' own type relative to each value; a
// product of 32-bit values would run at a sixteenth of the rate), and the output
// once at the end.  The sums are those of the rounded P, so the weights of a row
// add up to one.
//
// Masked keys: a key past a row's last one or on a page outside the pool has
// p = 0 by selection; keys that no row of a tile sees are read as zeros, so what
// a page holds behind its last token (NaN, say) has no part.  Where some rows of
// a tile see a key and others do not, a V value that is not finite would reach
// the others as 0 * NaN: such values are taken out of the product and added to
// the rows that see them after the loop.  (Under a weight that is rounded to 0, in
// fp16 one of less than 2^-32, an infinity that is not taken out becomes NaN.)
#include "lm_types.h"
#include "paged_geom.h"

namespace kvec {

constexpr int kAB = 256;                       // threads of a block: 4 waves
constexpr int kTileRows = 128;                 // rows of a tile block, 32 a wave
constexpr int kTileKeys = 32;
constexpr int kStreamRows = 16;                // rows of a stream block
constexpr int kStreamKeys = 32;                // keys a wave takes at a time
constexpr float kLog2e = 1.44269504088896340736f;
// The running maximum moves only when a score passes it by this much (in
// powers of two): p stays under 2^8, and most tiles rescale nothing.
constexpr float kLazy = 8.0f;
// Powers are formed as 2^(s c - m c), one operation, where m c is up to this; past
// it the rounding of m c counts (from 2^24 on in whole powers of two, so that a row
// could become 0 or infinite), and the maximum is taken off the score first.
constexpr float kFar = 256.0f;
constexpr float kFloatMax = 3.402823466e38f;
// Powers are formed 2^7 times as large where they are rounded to fp16, whose
// smallest numbers, 2^-24, would otherwise be short for a long tail far under a
// peak: 2^18 keys of 2^-25.5 all became 0.  The largest is 2^15 then (fp16 ends at
// 2^16); sums and outputs carry the factor until they are divided.  bf16 has the
// exponents of 32 bits.
template <class T>
constexpr float kLift = __is_same(T, _Float16) ? 7.0f : 0.0f;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c, __bf16*) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c, _Float16*) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c, __bf16*) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c, _Float16*) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Transposed read of 16-bit values: within 16 lanes, lane i gives the address
// of columns 4 (i % 4) .. + 3 of row i / 4 and gets column i of the four rows.
__device__ __forceinline__ u32x2 lds_tr(const uint8_t* p) {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p));
}

// Four e4m3 values to four 16-bit ones: exact in both types.
__device__ __forceinline__ u32x2 fp8_widen(uint32_t v, __bf16*) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, true))};
}
__device__ __forceinline__ u32x2 fp8_widen(uint32_t v, _Float16*) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, 1.0f, true))};
}

// The larger of the two lane halves' values, in both.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// c plus the sum of two 16-bit values.
__device__ __forceinline__ float add2(uint32_t v, float c, __bf16*) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, v), bf16x2{__bf16(1.0f), __bf16(1.0f)}, c, false);
}
__device__ __forceinline__ float add2(uint32_t v, float c, _Float16*) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, v), f16x2{_Float16(1.0f), _Float16(1.0f)}, c, false);
}

// Whether a 16-bit value is infinite or NaN: all its exponent bits are set.
__device__ __forceinline__ uint32_t exponent_bits(__bf16*) { return 0x7F80u; }
__device__ __forceinline__ uint32_t exponent_bits(_Float16*) { return 0x7C00u; }

// The values of four that are not finite, zeros for the others; v: 16-bit pairs.
template <class T>
__device__ __forceinline__ f32x4 not_finite(u32x2 v, T*) {
    f32x4 x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t w = j < 2 ? v.x : v.y;
        const float f = float(__builtin_bit_cast(T, uint16_t(j & 1 ? w >> 16 : w & 0xFFFFu)));
        x[j] = __builtin_fabsf(f) < INFINITY ? 0.0f : f;
    }
    return x;
}

// The lowest n bits, n clamped to 0 .. 32.
__device__ __forceinline__ uint32_t low_bits(int32_t n) {
    return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1;
}

// A value that the compiler takes for a new one: what is compared
// with it is compared again each time, instead of once with a register pair
// held for each lane mask over a whole loop.
__device__ __forceinline__ uint32_t anew(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

struct AttnArgs {
    const uint8_t* q;
    uint8_t* out;
    int64_t qs, qh, os, oh;                    // elements
    const uint8_t* pool;                       // the layer
    const int32_t* table;
    const int32_t* prefix_pages;
    const int32_t* seq_lens;
    const int32_t* cu;                         // null: one token a request
    const float *k_scale, *v_scale;
    float* ws_o;                               // [parts][rows][dim]
    f32x2* ws_ml;                              // [parts][rows]: maximum, sum
    uint32_t rec, token_bytes;                 // bytes of a token record, of its K
    uint32_t tokens, batch, heads, kv_heads, group, dim;
    uint32_t width, shift, pool_pages, cap;    // cap: positions that a table row covers
    uint32_t prefix;                           // keys of the shared part (0: none)
    uint32_t first;                            // first own key: prefix, or 0 with the prefix's pages read there
    uint32_t parts_flat, parts_own;            // splits of the keys of each part
    uint32_t blocks_flat;                      // blocks of the shared part, before those of the own keys
    uint32_t max_rows;                         // rows of a request that are computed (max_q tokens')
    FastDiv by_group, by_req_tiles;            // query heads of a K/V head; stream blocks: row tiles of a request
    FastDiv by_flat, by_own;                   // splits of each part
    FastDiv by_heads_flat, by_heads_own;       // K/V heads times splits
    int direct;                                // one part in all: outputs are final
    int wide_q, wide_o;                        // 16-byte rows
    float scale;
};

__device__ __forceinline__ uint32_t first_token(const AttnArgs& a, uint32_t b) {
    return a.cu ? uint32_t(a.cu[b]) : b;
}
__device__ __forceinline__ uint32_t live_tokens(const AttnArgs& a) {
    return a.cu ? min(uint32_t(max(a.cu[a.batch], 0)), a.tokens) : a.tokens;
}
// The request that token t (a live one) belongs to.
__device__ __forceinline__ uint32_t request_of(const AttnArgs& a, uint32_t t) {
    if (!a.cu) return t;
    uint32_t lo = 0, hi = a.batch;             // cu[lo] <= t < cu[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (uint32_t(a.cu[mid]) <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}
// Whether token t (a live one) is among its request's first max_q.  The request is
// looked for by a wave, 64 entries at a time.
__device__ __forceinline__ bool computed(const AttnArgs& a, uint32_t t) {
    if (!a.cu || a.max_rows >= a.tokens * a.group) return true;
    uint32_t lo = 0, n = a.batch;              // cu[lo] <= t < cu[lo + n]
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, off = ((threadIdx.x & 63) + 1) * step;
        const bool before = off < n && uint32_t(a.cu[lo + min(off, n)]) <= t;
        const uint32_t skip = uint32_t(__builtin_popcountll(__ballot(before))) * step;
        lo += skip;
        n = min(step, n - skip);
    }
    return (t - uint32_t(a.cu[lo])) * a.group < a.max_rows;
}
// Rows of request b that are computed; t0: its first token.
__device__ __forceinline__ uint32_t rows_of(const AttnArgs& a, uint32_t b, uint32_t t0) {
    const uint32_t t1 = min(first_token(a, b + 1), a.tokens);
    return t1 > t0 ? min((t1 - t0) * a.group, a.max_rows) : 0u;
}
// Keys that token t of request b sees.
__device__ __forceinline__ uint32_t seen_by(const AttnArgs& a, uint32_t b, uint32_t t) {
    const int64_t n = int64_t(a.seq_lens[b]) - int64_t(first_token(a, b + 1)) + int64_t(t) + 1;
    return uint32_t(n < 0 ? 0 : n > int64_t(a.cap) ? int64_t(a.cap) : n);
}

// What a block works on: rows row0 .. of a segment's rows, keys k0 .. k1 - 1.
struct Item {
    bool live;
    bool flat;                                 // the shared part: rows of all requests
    uint32_t b;                                // request (own keys)
    uint32_t t0;                               // its first token (0: all requests' rows)
    uint32_t rows;                             // rows of the segment
    uint32_t row0;
    uint32_t head;                             // K/V head
    uint32_t part;                             // where its partial result goes
    uint32_t k0, k1;
};

// Row tiles of the requests before each, for tile blocks of own keys: the
// request of tile `tile` and the first of its tiles; past the last one, the number
// of all tiles in `first` and batch in `b`.  A wave sums 64 requests at a time.
struct TileAt {
    uint32_t b, first;
};
__device__ __forceinline__ uint32_t tiles_of(const AttnArgs& a, uint32_t b) {
    return (rows_of(a, b, first_token(a, b)) + kTileRows - 1) / kTileRows;
}
__device__ __forceinline__ TileAt tile_at(const AttnArgs& a, uint32_t tile) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
        const uint32_t b = b0 + lane, n = b < a.batch ? tiles_of(a, b) : 0u;
        uint32_t x = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t y = uint32_t(__shfl_up(int(x), d, 64));
            if (lane >= uint32_t(d)) x += y;
        }
        const uint64_t past = __ballot(before + x > tile);
        if (past) {
            const int at = __builtin_ctzll(past);
            return TileAt{b0 + uint32_t(at), before + uint32_t(__shfl(int(x - n), at, 64))};
        }
        before += uint32_t(__shfl(int(x), 63, 64));
    }
    return TileAt{a.batch, before};
}

template <bool STREAM>
__device__ __forceinline__ Item make_item(const AttnArgs& a, uint32_t id) {
    constexpr uint32_t BM = STREAM ? kStreamRows : kTileRows;
    constexpr uint32_t KEYS = STREAM ? 4 * kStreamKeys : kTileKeys;
    Item it{};
    it.flat = id < a.blocks_flat;
    if (!it.flat) id -= a.blocks_flat;
    const FastDiv by_parts = it.flat ? a.by_flat : a.by_own, by_hp = it.flat ? a.by_heads_flat : a.by_heads_own;
    const uint32_t parts = by_parts.d, hp = by_hp.d;
    uint32_t tiles = 0;
    if (!STREAM && !it.flat) {
        // as many tiles as there are, not the launch's bound: blocks without
        // work come last then, and no compute unit gets a third block for them
        tiles = __builtin_amdgcn_readfirstlane(tile_at(a, 0xFFFFFFFFu).first);
        if (id >= tiles * hp) return it;
    }
    // Blocks go to the eight XCDs in turn: heads and splits first, so that with
    // eight K/V heads (and any eighth of the sizes that serve) an XCD's blocks
    // share their keys in its L2; and the tiles with the most keys, a request's
    // last ones, before the others (both: 1375 -> 1272 us for 8192 tokens behind
    // 8192 in four requests).
    uint32_t tile = fdiv(id, by_hp);
    const uint32_t rest = id - tile * hp;
    if (!STREAM && !it.flat) tile = tiles - 1 - tile;
    it.head = fdiv(rest, by_parts);
    const uint32_t split = rest - it.head * parts;
    it.part = it.flat ? split : a.parts_flat + split;
    uint32_t first = 0, last;
    if (it.flat) {
        it.rows = live_tokens(a) * a.group;
        it.row0 = tile * BM;
        it.live = it.row0 < it.rows;
        last = a.prefix;
    } else {
        uint32_t local;
        if (STREAM) {
            it.b = fdiv(tile, a.by_req_tiles);
            local = tile - it.b * a.by_req_tiles.d;
        } else {
            const TileAt t = tile_at(a, tile);
            it.b = __builtin_amdgcn_readfirstlane(t.b);
            local = tile - __builtin_amdgcn_readfirstlane(t.first);
        }
        it.t0 = first_token(a, it.b);
        it.rows = rows_of(a, it.b, it.t0);
        it.row0 = local * BM;
        it.live = it.row0 < it.rows;
        first = a.first;
        last = 0;
        if (it.live) {
            const uint32_t end_row = min(it.row0 + BM, it.rows) - 1;
            last = seen_by(a, it.b, it.t0 + fdiv(end_row, a.by_group));
        }
    }
    // equal shares of the keys, in whole steps
    const uint32_t n = last > first ? last - first : 0u;
    const uint32_t steps = (n + KEYS - 1) / KEYS, each = fdiv(steps + parts - 1, by_parts);
    it.k0 = first + min(uint64_t(split) * each * KEYS, uint64_t(n));
    it.k1 = first + min(uint64_t(split + 1) * each * KEYS, uint64_t(n));
    return it;
}

// The page of a key, as the table has it (of the last key past that: its place
// is looked at before it is used), and its slot, or kNoCell where there is none.
// In two steps, so that the table's entry can be on its way for a while.
__device__ __forceinline__ uint32_t key_page(const AttnArgs& a, const Item& it, uint32_t pos) {
    pos = min(pos, it.k1 - 1);
    const int32_t* row = it.flat || pos < a.prefix ? a.prefix_pages : a.table + uint64_t(it.b) * a.width;
    return uint32_t(*as_global(row + (pos >> a.shift)));
}
__device__ __forceinline__ uint32_t page_slot(const AttnArgs& a, const Item& it, uint32_t pos, uint32_t page) {
    const uint32_t slot = (page << a.shift) | (pos & ((1u << a.shift) - 1));
    return pos < it.k1 && page < a.pool_pages ? slot : kNoCell;
}
__device__ __forceinline__ uint32_t key_slot(const AttnArgs& a, const Item& it, uint32_t pos) {
    return page_slot(a, it, pos, key_page(a, it, pos));
}

// A 16-byte chunk of a key's K (or V) row, zeros where there is no key.
__device__ __forceinline__ const uint8_t* chunk_at(const AttnArgs& a, uint32_t slot, uint32_t off, bool inside) {
    return slot != kNoCell && inside ? a.pool + uint64_t(slot) * a.rec + off : reinterpret_cast<const uint8_t*>(kZeroCell);
}

// What a product of a query and a key is multiplied by, in powers of two.
__device__ __forceinline__ float score_factor(const AttnArgs& a) {
    const float c = a.scale * kLog2e * (a.k_scale ? *a.k_scale : 1.0f);
    return c == 0.0f ? 1e-30f : c;
}

// A row's maximum and sum at the end: none for one that sees nothing, and a
// maximum for a sum that is NaN (all its scores were), so that it is not taken
// for a row without keys when parts are joined.
__device__ __forceinline__ f32x2 settle(float m, float l, bool sees) {
    const float top = l != l && m == -INFINITY ? 0.0f : m;
    return f32x2{sees ? top : -INFINITY, sees ? l : 0.0f};
}

// Four values of a key's V row from value d on, zeros where there are none.
template <class T, bool FP8>
__device__ __forceinline__ u32x2 value4(const AttnArgs& a, uint32_t slot, uint32_t head_off, uint32_t d) {
    const uint8_t* p = chunk_at(a, slot, a.token_bytes + head_off + d * (FP8 ? 1 : 2), d < anew(a.dim));
    if constexpr (FP8) return fp8_widen(*as_global(reinterpret_cast<const uint32_t*>(p)), (T*)nullptr);
    else return *as_global(reinterpret_cast<const u32x2*>(p));
}

// Eight values of a query row (zeros past the head's end).
template <class T>
__device__ __forceinline__ u32x4 load_q(const AttnArgs& a, const T* row, uint32_t d) {
    u32x4 v = {0, 0, 0, 0};
    if (!row || d >= a.dim) return v;
    if (a.wide_q) return ld16(reinterpret_cast<const uint8_t*>(row + d));
#pragma unroll
    for (int j = 0; j < 4; ++j)
        v[j] = uint32_t(__builtin_bit_cast(uint16_t, *as_global(row + d + 2 * j))) |
               uint32_t(__builtin_bit_cast(uint16_t, *as_global(row + d + 2 * j + 1))) << 16;
    return v;
}

template <class T>
__device__ __forceinline__ void store4(T* p, f32x4 v, bool wide) {
    T* t = nullptr;
    if (wide) {
        *as_global(reinterpret_cast<u32x2*>(p)) = u32x2{pack2(v.x, v.y, t), pack2(v.z, v.w, t)};
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) put1(p + j, v[j]);
    }
}

// A kernel's arguments, read from memory again where they are used: what only its
// end needs is not held in registers over its loop.  (They are the kernel's one
// argument, so they start its argument segment.)
typedef const __attribute__((address_space(4))) AttnArgs LateArgs;
__device__ __forceinline__ LateArgs& late_args() {
    auto* p = (LateArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
}

// A finished quarter of a row: into the workspace, or the output.
template <class T, class Args>
__device__ __forceinline__ void emit4(Args& a, const Item& it, uint32_t token, uint32_t head, uint32_t d,
                                      f32x4 o, float inv_l) {
    if (d >= anew(a.dim)) return;
    if (a.direct) {
        store4(reinterpret_cast<T*>(a.out) + int64_t(token) * a.os + int64_t(head) * a.oh + d,
               f32x4{o.x * inv_l, o.y * inv_l, o.z * inv_l, o.w * inv_l}, a.wide_o);
    } else {
        const uint64_t row = uint64_t(it.part) * a.tokens * a.heads + uint64_t(token) * a.heads + head;
        *as_global(reinterpret_cast<f32x4*>(a.ws_o + row * a.dim + d)) = o;
    }
}

// -------------------------------------------------------------- tile blocks
// 128 rows against units of 32 keys: for rows enough to be bound by the matrix
// units.  Each wave owns 32 rows (Q in registers); the four waves share the K
// and V units in LDS, a ring of four of each.  A step of the loop forms the
// scores of unit j + 1 while the vector units turn those of unit j into P, and
// adds V of unit j; K of unit j + 3 and V of unit j + 2 are on their way from
// memory meanwhile.  There is a barrier every two steps.  (Scores of 64 keys at a
// time, both buffers of them, would take the registers past 256, and so one
// wave a SIMD less.)
//
// K and V of the queries' type go to LDS without passing registers: a wave's
// load puts 64 chunks of 16 bytes there one after another, so rows cannot be
// padded against bank conflicts, and the chunks of a row are permuted instead
// (chunk c of key r lies at c ^ swz(r); the lane that loads it picks its source
// accordingly).  An fp8 pool's values are widened on the way, by register.
//
// Measured, 32 query heads to 8 K/V heads of 128, bf16: 4 x 2048 tokens behind 8192
// 1216 us, 1017 TFLOP/s, where a library product of 8192 x 8192 x 8192 reaches 1267
// (fp16 1243, fp8 pool 1223); the same at 64 / 16 heads of 64 866 TFLOP/s, 32 / 8 of
// 80 763 and of 96 892 (80 takes rows of 16 chunks in LDS, six of them zeros), of 192
// 562 (in the kernel of 256 values, a quarter of its products by zeros), 16 / 4 of
// 256 741 (one block a compute unit); 16 x 2048 with no prefix 765; 16 x 128 behind
// 4096 151 us, 926 TFLOP/s (512 blocks, all at once: their start and end are not
// hidden behind others).  No one part bounds it: the matrix units are busy 46 % of
// the time and instructions issue in 72 %; when the whole took 1270 us, without the
// powers it took 1186, without either product about 1000, without the loads to LDS
// 1068.
template <int DP>
struct TileGeom {
    static constexpr int ROW = DP == 64 ? 128 : DP <= 128 ? 256 : 512;   // bytes of a key's row in LDS
    static constexpr int POS = ROW / 16;                                 // chunks of it
    static constexpr int BYTES = kTileKeys * ROW;
    // 16 lanes read one chunk of 16 keys: all on different banks
    static __device__ __forceinline__ uint32_t swz_k(uint32_t key) { return DP == 64 ? (key >> 1) & 7 : key & 15; }
    // 64 lanes read two neighbours of chunks of 8 keys: moved by whole pairs
    static __device__ __forceinline__ uint32_t swz_v(uint32_t key) {
        return DP == 64 ? ((key >> 1) & 3) << 1 : (key & 7) << 1;
    }
};

// 16 bytes a lane from memory to LDS, lane after lane from `to` on (the same for
// the wave).
__device__ __forceinline__ void load_to_lds(const uint8_t* from, uint8_t* to) {
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// Says that a condition hardly ever holds (where SAY: at 256 values a head the
// registers come out worse for it, past what a wave has).
template <bool SAY>
__device__ __forceinline__ bool rarely(bool x) {
    return SAY ? __builtin_expect_with_probability(x, 0, 0.99) : x;
}

// A barrier of the block after which its LDS holds what was written before and
// what loads brought.
__device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);                   // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <class T, bool FP8, int DP>
__device__ __forceinline__ void attn_tile(const AttnArgs& a, const Item& it, uint8_t* k0, uint8_t* k1, uint8_t* k2, uint8_t* k3,
                                          uint8_t* v0, uint8_t* v1, uint8_t* v2, uint8_t* v3) {
    using G = TileGeom<DP>;
    constexpr int KS = DP / 16, DB = DP / 32;
    constexpr int CH = FP8 ? DP / 16 : G::POS;             // chunks of a key that are loaded
    constexpr int PER = (kTileKeys * CH + kAB - 1) / kAB;  // of them by a thread
    __shared__ uint32_t odd;                              // V values that are not finite were taken out
    __shared__ uint32_t lows[4];

    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t r = lane & 31, h = lane >> 5;
    T* const ty = nullptr;
    if (tid == 0) odd = 0;
    if constexpr (FP8) __syncthreads();                   // before a value is taken out

    const uint32_t row_bytes = a.dim * (FP8 ? 1 : 2), head_off = it.head * row_bytes;
    // V values that are not finite become 0
    auto scrub = [&](u32x4 v) {
        const uint32_t e = exponent_bits(ty);
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t w = v[j];
            if ((w & e) == e) w &= 0xFFFF0000u, bad = true;
            if (((w >> 16) & e) == e) w &= 0x0000FFFFu, bad = true;
            v[j] = w;
        }
        if (bad) odd = 1;
        return v;
    };
    // A unit's K and V rows on their way; slot: of its key `lane` % 32.  A chunk
    // past the head's end, or of a key that is not there, is read from zeros.
    u32x4 xk[FP8 ? PER : 1], xv[FP8 ? PER : 1];
    const uint8_t *from_k[PER], *from_v[PER];
    uint32_t step_k[PER], step_v[PER];                    // bytes a slot
    const uint8_t* const zeros = reinterpret_cast<const uint8_t*>(kZeroCell);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint32_t idx = FP8 ? i * kAB + tid : (wave * PER + i) * 64 + lane, key = idx / CH, pos = idx % CH;
        const uint32_t ck = (FP8 ? pos : pos ^ G::swz_k(key)) * 16, cv = (FP8 ? pos : pos ^ G::swz_v(key)) * 16;
        const bool in = key < uint32_t(kTileKeys);
        step_k[i] = in && ck < row_bytes ? a.rec : 0u;
        step_v[i] = in && cv < row_bytes ? a.rec : 0u;
        from_k[i] = step_k[i] ? a.pool + head_off + ck : zeros;
        from_v[i] = step_v[i] ? a.pool + a.token_bytes + head_off + cv : zeros;
    }
    uint32_t sl[PER];                                     // the slots that K was loaded from last
    auto load_k = [&](uint32_t slot, uint8_t* k) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t idx = FP8 ? i * kAB + tid : (wave * PER + i) * 64 + lane, key = idx / CH;
            sl[i] = uint32_t(__shfl(int(slot), int(key & 31), 64));
            const bool there = sl[i] != kNoCell;
            const uint8_t* p = (there ? from_k[i] : zeros) + uint64_t(there ? sl[i] : 0u) * step_k[i];
            if constexpr (FP8) xk[i] = ld16(p);
            else load_to_lds(p, k + (wave * PER + i) * 1024);
        }
    };
    // V of the unit whose K was loaded last
    auto load_v = [&](uint8_t* v) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const bool there = sl[i] != kNoCell;
            const uint8_t* p = (there ? from_v[i] : zeros) + uint64_t(there ? sl[i] : 0u) * step_v[i];
            if constexpr (FP8) xv[i] = ld16(p);
            else load_to_lds(p, v + (wave * PER + i) * 1024);
        }
    };
    // fp8: what load() holds in registers, widened into LDS
    auto put_fp8 = [&](const u32x4* from, bool is_v, uint8_t* to, bool careful) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t idx = i * kAB + tid, key = idx / CH, ch = idx % CH;
            if (kTileKeys * CH % kAB && key >= uint32_t(kTileKeys)) break;
            const uint32_t swz = is_v ? G::swz_v(key) : G::swz_k(key);
            const u32x4 x = from[FP8 ? i : 0];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const u32x2 x0 = fp8_widen(x[2 * j], ty), x1 = fp8_widen(x[2 * j + 1], ty);
                u32x4 w = {x0.x, x0.y, x1.x, x1.y};
                if (careful) w = scrub(w);
                *reinterpret_cast<u32x4*>(to + key * G::ROW + ((ch * 2 + j) ^ swz) * 16) = w;
            }
        }
    };
    const uint32_t units = (it.k1 - it.k0 + kTileKeys - 1) / kTileKeys;
    const int32_t* const own_row = a.table + uint64_t(it.b) * a.width;
    // Of a key of the unit at `base`.  The row is chosen by lane: chosen once for the
    // unit, where its keys lie on one side of the prefix's end, the compiler lost the
    // choice for the fifth unit and read the request's own row there (seen in the
    // generated code).
    auto unit_page = [&](uint32_t base, uint32_t key) __attribute__((always_inline)) {
        const uint32_t pos = min(base + key, it.k1 - 1);
        const int32_t* row = it.flat || pos < a.prefix ? a.prefix_pages : own_row;
        return uint32_t(*as_global(row + (pos >> a.shift)));
    };
    const uint32_t key = lane & 31;
    // The first units, asked for before anything else is: the queries and their
    // limits come while these are on their way.
    // of the lane's key: pages of units j + 3 and j + 4; and which keys of units
    // j, j + 1 and j + 2 are there
    uint32_t page3 = 0, page4 = 0, valid0 = 0, valid1 = 0, valid2 = 0, slot2 = 0;
    if (units) {
        const uint32_t pg0 = unit_page(it.k0, key), pg1 = unit_page(it.k0 + kTileKeys, key);
        const uint32_t pg2 = unit_page(it.k0 + 2 * kTileKeys, key);
        page3 = unit_page(it.k0 + 3 * kTileKeys, key);
        page4 = unit_page(it.k0 + 4 * kTileKeys, key);
        const uint32_t s0 = page_slot(a, it, it.k0 + key, pg0), s1 = page_slot(a, it, it.k0 + kTileKeys + key, pg1);
        slot2 = page_slot(a, it, it.k0 + 2 * kTileKeys + key, pg2);
        valid0 = uint32_t(__ballot(s0 != kNoCell));
        valid1 = uint32_t(__ballot(s1 != kNoCell));
        valid2 = uint32_t(__ballot(slot2 != kNoCell));
        if constexpr (!FP8) {
            load_k(s0, k0);
            load_v(v0);
            load_k(s1, k1);
            load_v(v1);
            load_k(slot2, k2);
        } else {
            // one unit at a time in registers; the last one's K stays there
            load_k(s0, k0);
            load_v(v0);
            put_fp8(xk, false, k0, false);
            put_fp8(xv, true, v0, true);
            load_k(s1, k1);
            load_v(v1);
            put_fp8(xk, false, k1, false);
            put_fp8(xv, true, v1, true);
            load_k(slot2, k2);
            put_fp8(xk, false, k2, false);
        }
    }

    // the lane's row
    const uint32_t row = it.row0 + wave * 32 + r;
    const bool has = row < it.rows;
    const uint32_t tok = has ? fdiv(row, a.by_group) : 0u;
    const uint32_t token = it.t0 + tok, head = it.head * a.group + (has ? row - tok * a.group : 0u);
    // rows that are not there, and rows that see nothing, ask for no mask
    const uint32_t seen = has ? seen_by(a, it.flat ? request_of(a, token) : it.b, token) : 0u;
    const uint32_t limit = seen ? seen : 0xFFFFFFFFu;
    // 0 would make NaN of a masked score; a negative one goes to the query
    const float c0 = score_factor(a);
    const uint32_t sign = c0 < 0.0f ? 0x80008000u : 0u;
    u32x4 qf[KS];
    {
        const T* p = has ? reinterpret_cast<const T*>(a.q) + int64_t(token) * a.qs + int64_t(head) * a.qh : nullptr;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = load_q(a, p, uint32_t(s * 16) + h * 8) ^ sign;
    }
    // the fewest keys that a row of the wave, and of the block, sees
    uint32_t low = limit;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) low = min(low, uint32_t(__shfl_xor(int(low), d, 64)));
    low = __builtin_amdgcn_readfirstlane(low);
    if (lane == 0) lows[wave] = low;
    __syncthreads();
    const uint32_t block_low = min(min(lows[0], lows[1]), min(lows[2], lows[3]));

    const float c = fabsf(c0);
    const float lazy = fminf(kLazy / c, kFloatMax);
    float m = -INFINITY, l = 0.0f, mc = 0.0f, bar = -INFINITY;   // bar: the score that moves m
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x16{};

    // places in a unit of K and V that the lane reads
    uint32_t at_k[KS], at_v[DB];
    {
        const uint32_t i16 = lane & 15, gd = (lane >> 4) & 1, kk = 4 * h + i16 / 4;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) at_k[ks] = anew(r * G::ROW + ((ks * 2 + h) ^ G::swz_k(r)) * 16);
#pragma unroll
        for (int d = 0; d < DB; ++d)
            at_v[d] = anew(kk * G::ROW + ((d * 4 + gd * 2 + ((i16 >> 1) & 1)) ^ G::swz_v(kk)) * 16 + (i16 & 1) * 8);
    }
    // S^T: 32 keys x 32 rows
    auto scores = [&](const uint8_t* k) __attribute__((always_inline)) {
        f32x16 s = f32x16{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = mma32(*reinterpret_cast<const u32x4*>(k + at_k[ks]), qf[ks], s, ty);
        return s;
    };
    // the largest score of the lane's row among the scores that it holds
    auto largest = [&](const f32x16& s) __attribute__((always_inline)) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        return top;
    };
    // ... with the masks, where there are any; keys: 8 (i / 4) + 4 h + i % 4
    auto masked = [&](f32x16& s, float top, uint32_t base, uint32_t valid) __attribute__((always_inline)) {
        if (rarely<DP <= 128>(valid != ~0u || base + kTileKeys > low)) {
            const uint32_t see = (valid & low_bits(int32_t(min(limit, 0x7FFFFFFFu) - base))) >> (4 * h);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = see & (1u << (8 * (i / 4) + i % 4)) ? s[i] : -INFINITY;
            top = largest(s);
        }
        return max_halves(top);
    };

    f32x16 sa, sb;
    float top = -INFINITY;
    if (units) {
        meet();
        sa = scores(k0);
        top = masked(sa, largest(sa), it.k0, valid0);
    }
    // Step j: K of unit j + 1 and V of unit j are read, K of unit j + 3 (its
    // lane's slot: `slot`) and V of unit j + 2 loaded.
    auto step = [&](uint32_t base, uint32_t slot, uint32_t valid, const uint8_t* k_next, const uint8_t* v_now, uint8_t* k_to,
                    uint8_t* v_to, f32x16& s, f32x16& s_next) __attribute__((always_inline)) {
        if (rarely<DP <= 128>(__ballot(top > bar) != 0)) {
            const float to = fmaxf(m, top);
            const float f = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - to) * c);
            m = to;
            // a row with scores past kFar comes here with every unit
            const float off = fabsf(m) * c > kFar && m != -INFINITY ? m : 0.0f;
            bar = off != 0.0f ? -INFINITY : m + lazy;
            mc = (off != 0.0f || m == -INFINITY ? 0.0f : m * c) - kLift<T>;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] -= off;
            l *= f;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
            }
        }
        load_v(v_to);
        // (the lane masks of both at once, at four loads each, are too many)
        if constexpr (PER > 2) __builtin_amdgcn_sched_barrier(0);
        load_k(slot, k_to);
        // The next unit's scores beside this one's powers, then O^T += V^T P^T.
        // Left to the compiler's order: barriers between a vector and a matrix
        // part, alternating both products, fixed counts of vector instructions
        // to a matrix one, or raised priority in the matrix part took 0 to 10 %
        // longer (8192 tokens behind 8192, eight K/V heads).
        constexpr int AK = DP > 128 ? 4 : KS < 8 ? KS : 8, AV = 4;   // reads ahead of their use
        u32x4 kf[KS], vf[2 * DB];
        auto read_k = [&](int i) __attribute__((always_inline)) {
            kf[i] = *reinterpret_cast<const u32x4*>(k_next + at_k[i]);
        };
        // keys 16 t + 4 h + (lane % 16) / 4 and 8 further
        auto read_v = [&](int i) __attribute__((always_inline)) {
            const uint8_t* vd = v_now + at_v[i % DB] + 16 * (i / DB) * G::ROW;
            const u32x2 x0 = lds_tr(vd), x1 = lds_tr(vd + 8 * G::ROW);
            vf[i] = u32x4{x0.x, x0.y, x1.x, x1.y};
        };
#pragma unroll
        for (int i = 0; i < AK; ++i) read_k(i);
        s_next = f32x16{};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            s_next = mma32(kf[i], qf[i], s_next, ty);
            if (i + AK < KS) read_k(i + AK);
        }
        u32x4 p[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -mc));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i / 4][i % 4] = pack2(s[2 * i], s[2 * i + 1], ty);
            l = add2(uint32_t(p[i / 4][i % 4]), l, ty);   // the sum is that of the rounded P
        }
#pragma unroll
        for (int i = 0; i < AV; ++i) read_v(i);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            if (i + AV < 2 * DB) read_v(i + AV);
            o[i % DB] = mma32(vf[i], p[i / DB], o[i % DB], ty);
        }
        top = masked(s_next, largest(s_next), base + kTileKeys, valid);
        if constexpr (FP8) {
            put_fp8(xk, false, k_to, false);
            put_fp8(xv, true, v_to, base + 3 * kTileKeys > block_low);
        }
    };
    // Two steps, with a barrier before them: what either reads has come in the
    // pass before, and what either loads goes where nothing is read any more.
    // (The pages, loaded a pass ahead, have come by then too.)
    auto pass = [&](uint32_t j, const uint8_t* ka, const uint8_t* kb, uint8_t* va, uint8_t* vb, uint8_t* kc, uint8_t* vc,
                    uint8_t* kd, uint8_t* vd) __attribute__((always_inline)) {
        const uint32_t base = it.k0 + j * kTileKeys;
        meet();
        if (!FP8 && rarely<DP <= 128>(base + 2 * kTileKeys > block_low)) {
            for (uint32_t e = tid; e < uint32_t(G::BYTES) / 16; e += kAB) {
                const u32x4 x = reinterpret_cast<const u32x4*>(va)[e], y = reinterpret_cast<const u32x4*>(vb)[e];
                reinterpret_cast<u32x4*>(va)[e] = scrub(x);
                reinterpret_cast<u32x4*>(vb)[e] = scrub(y);
            }
            meet();
        }
        const uint32_t slot3 = page_slot(a, it, base + 3 * kTileKeys + key, page3);
        const uint32_t slot4 = page_slot(a, it, base + 4 * kTileKeys + key, page4);
        page3 = unit_page(base + 5 * kTileKeys, key);
        page4 = unit_page(base + 6 * kTileKeys, key);
        step(base, slot3, valid1, ka, va, kc, vc, sa, sb);
        if (j + 1 < units) step(base + kTileKeys, slot4, valid2, kb, vb, kd, vd, sb, sa);
        valid1 = uint32_t(__ballot(slot3 != kNoCell));
        valid2 = uint32_t(__ballot(slot4 != kNoCell));
    };
    for (uint32_t j = 0; j < units; j += 4) {
        pass(j, k1, k2, v0, v1, k3, v2, k0, v3);
        if (j + 2 < units) pass(j + 2, k3, k0, v2, v3, k1, v0, k2, v1);
    }
    meet();

    // V values that were taken out, to the rows that see them
    if (odd) {
        // from the first pass on that was looked through, two units at a time (fp8:
        // the first units are looked through before the limits are known)
        const uint32_t skip = !FP8 && block_low > it.k0 ? (block_low - it.k0) / (2 * kTileKeys) * (2 * kTileKeys) : 0u;
        for (uint32_t kk = it.k0 + skip; kk < it.k1; ++kk) {
            const uint32_t sl = kk < limit ? key_slot(a, it, kk) : kNoCell;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 x = not_finite(value4<T, FP8>(a, sl, head_off, uint32_t(d * 32 + 8 * i) + 4 * h), ty);
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[d][4 * i + j] += x[j];
                    __builtin_amdgcn_sched_barrier(0);    // a rare path: few registers, not speed
                }
        }
    }

    l += __shfl_xor(l, 32, 64);
    {
        const f32x2 ml = settle(m, l, limit != 0xFFFFFFFFu);
        m = ml.x, l = ml.y;
    }
    // where the row goes, worked out anew: not held over the loop
    const uint32_t at_row = it.row0 + wave * 32 + (anew(lane) & 31);
    if (at_row >= it.rows) return;
    LateArgs& e = late_args();
    const FastDiv by_group = {e.by_group.d, e.by_group.m, e.by_group.s1, e.by_group.s2};
    const uint32_t to_tok = fdiv(at_row, by_group);
    const uint32_t to_token = it.t0 + to_tok, to_head = it.head * e.group + at_row - to_tok * e.group;
    const float vs = e.v_scale ? *e.v_scale : 1.0f;
    const float inv = l > 0.0f ? vs / l : l == l ? 0.0f : l;
    if (!e.direct && anew(h) == 0) {
        const uint64_t at = uint64_t(it.part) * e.tokens * e.heads + uint64_t(to_token) * e.heads + to_head;
        *as_global(e.ws_ml + at) = f32x2{m, l};
    }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4 x = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            if (l == 0.0f) x = f32x4{0, 0, 0, 0};
            emit4<T>(e, it, to_token, to_head, uint32_t(d * 32 + 8 * i) + 4 * h, x, inv);
        }
}

// ------------------------------------------------------------ stream blocks
// 16 rows against a run of keys that the block's four waves share out, 32 keys
// at a time: for the few rows of a request that decodes, bound by reading K and
// V.  A wave works alone until the end (its V in a part of LDS of its own, its
// maximum and sum its own), then the four results are joined.  Measured: 64 requests
// of 2048 own keys, 8 K/V heads of 128, bf16: 109 us, 4.9 TB/s (a read stream reaches
// 7.1); 256 such 400 us, 5.4 TB/s; 64 over an fp8 pool 50 us, 5.4 TB/s.  Four requests
// behind 512 tokens 8.4 us, most of it the way to the first keys (table, then keys:
// about 6 us) and the joining of the waves.
template <class T, bool FP8, int DP>
__device__ __forceinline__ void attn_stream(const AttnArgs& a, const Item& it, uint8_t* v0, uint8_t* v1, uint8_t* v2,
                                            uint8_t* v3) {
    using G = TileGeom<DP>;                               // V lies as in the tile blocks
    constexpr int KS = DP / 32, DB = DP / 16;
    constexpr int CH = DP / (FP8 ? 16 : 8);
    constexpr int PER = (kStreamKeys * CH + 63) / 64;
    static_assert(kStreamKeys == kTileKeys && G::BYTES >= kStreamRows * DP * 4, "a unit of V, or the rows' results");
    __shared__ float lm[4][kStreamRows], ll[4][kStreamRows];

    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t r = lane & 15, g = lane >> 4;
    T* const ty = nullptr;
    uint8_t* const lv = wave == 0 ? v0 : wave == 1 ? v1 : wave == 2 ? v2 : v3;

    const uint32_t row_bytes = a.dim * (FP8 ? 1 : 2), head_off = it.head * row_bytes;
    u32x4 xv[PER];
    u32x4 xk[2][KS];                                      // fp8: 8 bytes of each
    auto fetch = [&](uint32_t slot) {                     // slot: of the keys lane % 32
        const uint32_t inside = anew(row_bytes);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const uint32_t s = uint32_t(__shfl(int(slot), int(kb * 16 + r), 64));
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const uint32_t d = ks * 32 + g * 8;
                if constexpr (FP8) {
                    const u32x2 v = *as_global(reinterpret_cast<const u32x2*>(chunk_at(a, s, head_off + d, d < inside)));
                    xk[kb][ks].x = v.x;
                    xk[kb][ks].y = v.y;
                } else {
                    xk[kb][ks] = ld16(chunk_at(a, s, head_off + d * 2, d * 2 < inside));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t idx = i * 64 + lane, key = idx / CH, ch = idx % CH;
            const uint32_t s = uint32_t(__shfl(int(slot), int(key & 31), 64));
            const bool in = ch * 16 < inside && key < uint32_t(kStreamKeys);
            xv[i] = ld16(chunk_at(a, s, a.token_bytes + head_off + ch * 16, in));
        }
    };
    auto scrub = [&](u32x4& v) {
        const uint32_t e = exponent_bits(ty);
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t w = v[j];
            if ((w & e) == e) w &= 0xFFFF0000u, bad = true;
            if (((w >> 16) & e) == e) w &= 0x0000FFFFu, bad = true;
            v[j] = w;
        }
        return bad;
    };

    const uint32_t nblk = (it.k1 - it.k0 + kStreamKeys - 1) / kStreamKeys;
    bool odd = false;
    uint32_t slot = kNoCell, slot_next = kNoCell;
    if (wave < nblk) {
        slot = key_slot(a, it, it.k0 + wave * kStreamKeys + (lane & 31));
        fetch(slot);
        slot_next = key_slot(a, it, it.k0 + (wave + 4) * kStreamKeys + (lane & 31));
    }
    // the queries and their limits, while the first keys are on their way
    const uint32_t row = it.row0 + r;
    const bool has = row < it.rows;
    const uint32_t tok = has ? fdiv(row, a.by_group) : 0u;
    const uint32_t token = it.t0 + tok, head = it.head * a.group + (has ? row - tok * a.group : 0u);
    // rows that are not there, and rows that see nothing, ask for no mask
    const uint32_t seen = has ? seen_by(a, it.flat ? request_of(a, token) : it.b, token) : 0u;
    const uint32_t limit = seen ? seen : 0xFFFFFFFFu;
    // 0 would make NaN of a masked score; a negative one goes to the query
    const float c0 = score_factor(a);
    const uint32_t sign = c0 < 0.0f ? 0x80008000u : 0u;
    u32x4 qf[KS];
    {
        const T* p = has ? reinterpret_cast<const T*>(a.q) + int64_t(token) * a.qs + int64_t(head) * a.qh : nullptr;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = load_q(a, p, uint32_t(s * 32) + g * 8) ^ sign;
    }
    uint32_t low = limit;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) low = min(low, uint32_t(__shfl_xor(int(low), d, 64)));
    low = __builtin_amdgcn_readfirstlane(low);

    const float c = fabsf(c0);
    float m = -INFINITY, l = 0.0f;
    f32x4 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x4{0, 0, 0, 0};

    for (uint32_t n = wave; n < nblk; n += 4) {
        const uint32_t base = it.k0 + n * kStreamKeys;
        const uint32_t valid = uint32_t(__ballot(slot != kNoCell));
        const bool careful = base + kStreamKeys > low;
        // V to LDS; the reads of the block before have all been waited for by
        // its products, and a wave's LDS operations keep their order
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t idx = i * 64 + lane, key = idx / CH, ch = idx % CH;
            if (kStreamKeys * CH % 64 && key >= uint32_t(kStreamKeys)) break;
            uint8_t* pv = lv + key * G::ROW;
            const uint32_t swz = G::swz_v(key);
            if constexpr (FP8) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const u32x2 v0 = fp8_widen(xv[i][2 * j], ty), v1 = fp8_widen(xv[i][2 * j + 1], ty);
                    u32x4 v = {v0.x, v0.y, v1.x, v1.y};
                    if (careful) odd |= scrub(v);
                    *reinterpret_cast<u32x4*>(pv + ((ch * 2 + j) ^ swz) * 16) = v;
                }
            } else {
                u32x4 v = xv[i];
                if (careful) odd |= scrub(v);
                *reinterpret_cast<u32x4*>(pv + (ch ^ swz) * 16) = v;
            }
        }
        f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                u32x4 kf = xk[kb][ks];
                if constexpr (FP8) {
                    const u32x2 k0 = fp8_widen(kf.x, ty), k1 = fp8_widen(kf.y, ty);
                    kf = u32x4{k0.x, k0.y, k1.x, k1.y};
                }
                s[kb] = mma16(kf, qf[ks], s[kb], ty);
            }
        if (n + 4 < nblk) {
            fetch(slot_next);
            slot = slot_next;
            slot_next = key_slot(a, it, base + 8 * kStreamKeys + (lane & 31));
        }
        // keys: 16 kb + 4 g + i
        if (valid != 0xFFFFFFFFu || careful) {
            const uint32_t see = (valid & low_bits(int32_t(min(limit, 0x7FFFFFFFu) - base))) >> (4 * g);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[kb][i] = see & (1u << (kb * 16 + i)) ? s[kb][i] : -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i / 4][i % 4]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (__any((top - m) * c > kLazy || m == -INFINITY)) {
            const float to = fmaxf(m, top);
            const float f = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - to) * c);
            m = to;
            l *= f;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= f;
        }
        const float off = m == -INFINITY ? 0.0f : m;
        const float lift = __uint_as_float(anew(__float_as_uint(kLift<T>)));   // not held in a scalar register
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i / 4][i % 4] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 4][i % 4] - off, c, lift));
        // sum over keys 4 g .. and 16 + 4 g .. : what the lane's scores are of
        const u32x4 p = {pack2(s[0][0], s[0][1], ty), pack2(s[0][2], s[0][3], ty), pack2(s[1][0], s[1][1], ty),
                         pack2(s[1][2], s[1][3], ty)};
#pragma unroll
        for (int i = 0; i < 4; ++i) l = add2(uint32_t(p[i]), l, ty);   // the sum is that of the rounded P
        const uint32_t kk = 4 * g + r / 4, z = G::swz_v(kk);   // keys 8 and 16 apart: the same permutation
        const uint8_t* v = lv + kk * G::ROW + (r & 1) * 8;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            const uint8_t* vd = v + ((d * 2 + ((r >> 1) & 1)) ^ z) * 16;
            const u32x2 x0 = lds_tr(vd), x1 = lds_tr(vd + 16 * G::ROW);
            o[d] = mma16(u32x4{x0.x, x0.y, x1.x, x1.y}, p, o[d], ty);
        }
        __builtin_amdgcn_wave_barrier();
    }

    // V values that were taken out, to the rows that see them
    if (__any(odd)) {
        for (uint32_t n = wave; n < nblk; n += 4) {
            const uint32_t base = it.k0 + n * kStreamKeys;
            if (base + kStreamKeys <= low) continue;
            for (uint32_t key = base; key < min(base + kStreamKeys, it.k1); ++key) {
                const uint32_t sl = key < limit ? key_slot(a, it, key) : kNoCell;
#pragma unroll
                for (int d = 0; d < DB; ++d)
                    o[d] += not_finite(value4<T, FP8>(a, sl, head_off, uint32_t(d * 16) + 4 * g), ty);
            }
        }
    }

    // the four waves' results: brought to one maximum, summed over LDS
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    {
        const f32x2 ml = settle(m, l, seen != 0);
        m = ml.x, l = ml.y;
    }
    if (g == 0) {
        lm[wave][r] = m;
        ll[wave][r] = l;
    }
    __syncthreads();
    const float top = fmaxf(fmaxf(lm[0][r], lm[1][r]), fmaxf(lm[2][r], lm[3][r]));
    auto factor = [&](float x) { return x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((x - top) * c); };
    const float f = factor(m);
    float* lo = reinterpret_cast<float*>(lv);             // [row][dim]
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        f32x4 x = o[d] * f;
        if (m == -INFINITY) x = f32x4{0, 0, 0, 0};
        *reinterpret_cast<f32x4*>(lo + r * DP + d * 16 + 4 * g) = x;
    }
    __syncthreads();
    const float vs = a.v_scale ? *a.v_scale : 1.0f;
    for (uint32_t e = tid; e < uint32_t(kStreamRows) * (DP / 4); e += kAB) {
        const uint32_t rr = e / (DP / 4), d = e % (DP / 4) * 4;
        const uint32_t rw = it.row0 + rr;
        if (rw >= it.rows) continue;
        f32x4 x = {0, 0, 0, 0};
        float sum = 0.0f, mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            x += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(w == 0 ? v0 : w == 1 ? v1 : w == 2 ? v2 : v3) + rr * DP + d);
            mx = fmaxf(mx, lm[w][rr]);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w)
            sum += lm[w][rr] == -INFINITY ? 0.0f : ll[w][rr] * __builtin_amdgcn_exp2f((lm[w][rr] - mx) * c);
        const uint32_t tr = fdiv(rw, a.by_group), tk = it.t0 + tr, hd = it.head * a.group + rw - tr * a.group;
        if (!a.direct && d == 0) {
            const uint64_t at = uint64_t(it.part) * a.tokens * a.heads + uint64_t(tk) * a.heads + hd;
            *as_global(a.ws_ml + at) = f32x2{mx, sum};
        }
        emit4<T>(a, it, tk, hd, d, x, sum > 0.0f ? vs / sum : sum == sum ? 0.0f : sum);
    }
}

// The kernels: FLAT and OWN say what takes the shared part and the own keys (0: no
// such blocks, 1: stream blocks, 2: tile blocks).  Both parts are one launch: the
// one is bound by the matrix units, the other by memory.
template <class T, bool FP8, int DP, int FLAT, int OWN>
__global__ __launch_bounds__(kAB, DP <= 128 ? 2 : 1) void attn_kernel(AttnArgs a) {
    using G = TileGeom<DP>;
    constexpr bool TILE = FLAT == 2 || OWN == 2;
    // separate arrays: the compiler can tell their accesses apart, so a read of
    // one does not wait for a load into another
    __shared__ __attribute__((aligned(16))) uint8_t k0[TILE ? G::BYTES : 16], k1[TILE ? G::BYTES : 16];
    __shared__ __attribute__((aligned(16))) uint8_t k2[TILE ? G::BYTES : 16], k3[TILE ? G::BYTES : 16];
    __shared__ __attribute__((aligned(16))) uint8_t v0[G::BYTES], v1[G::BYTES], v2[G::BYTES], v3[G::BYTES];
    const uint32_t id = blockIdx.x;
    if (TILE && (FLAT != 2 || OWN == 2 || id < a.blocks_flat)) {
        const Item it = make_item<false>(a, id);
        if (it.live) attn_tile<T, FP8, DP>(a, it, k0, k1, k2, k3, v0, v1, v2, v3);
    } else if (OWN == 1) {
        const Item it = make_item<true>(a, id);
        if (it.live) attn_stream<T, FP8, DP>(a, it, v0, v1, v2, v3);
    }
}

// Partial results of a row brought to one maximum, summed, divided and rounded.
// A block takes one row: `lanes` threads a part, the parts shared out to the
// others, so that a row's parts are read side by side.  Measured: 2048 rows of 128
// with 12 parts 6.0 us (6.5 where the row's request is looked for), 8192 rows with 7
// parts 12.7, 128 rows with 5 parts 3.8.
template <class T>
__global__ __launch_bounds__(kAB) void attn_join_kernel(AttnArgs a, uint32_t lanes) {
    __shared__ f32x4 lo[kAB];
    __shared__ float ll[kAB];
    const uint32_t tid = threadIdx.x, rows = a.tokens * a.heads, row = blockIdx.x;
    if (row / a.heads >= live_tokens(a) || row / a.heads < first_token(a, 0) || !computed(a, row / a.heads)) return;
    const uint32_t each = kAB / lanes, mine = tid / lanes, d = tid % lanes * 4;
    const uint32_t parts = a.parts_flat + a.parts_own;
    float top = -INFINITY, l = 0.0f;
    const float c = fabsf(score_factor(a));
    f32x4 o = {0, 0, 0, 0};
    for (uint32_t p = tid & 63; p < parts; p += 64) top = fmaxf(top, as_global(a.ws_ml)[uint64_t(p) * rows + row].x);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
#pragma unroll 4
    for (uint32_t p = mine; p < parts; p += each) {
        const uint64_t at = uint64_t(p) * rows + row;
        const f32x2 ml = as_global(a.ws_ml)[at];
        if (ml.x == -INFINITY) continue;                  // nothing seen there
        const float f = __builtin_amdgcn_exp2f((ml.x - top) * c);
        l += ml.y * f;
        if (d < a.dim) o += *as_global(reinterpret_cast<const f32x4*>(a.ws_o + at * a.dim + d)) * f;
    }
    lo[tid] = o;
    ll[tid] = l;
    __syncthreads();
    if (mine || d >= a.dim) return;
    for (uint32_t p = 1; p < each; ++p) {
        o += lo[p * lanes + tid];
        l += ll[p * lanes + tid];
    }
    const float vs = a.v_scale ? *a.v_scale : 1.0f;
    const float inv = l > 0.0f ? vs / l : l == l ? 0.0f : l;
    store4(reinterpret_cast<T*>(a.out) + int64_t(row / a.heads) * a.os + int64_t(row % a.heads) * a.oh + d, o * inv,
           a.wide_o);
}

typedef void (*AttnFn)(AttnArgs);

template <class T, bool FP8, int FLAT, int OWN>
AttnFn pick_dim(int dim) {
    return dim <= 64    ? &attn_kernel<T, FP8, 64, FLAT, OWN>
           : dim <= 96  ? &attn_kernel<T, FP8, 96, FLAT, OWN>
           : dim <= 128 ? &attn_kernel<T, FP8, 128, FLAT, OWN>
                        : &attn_kernel<T, FP8, 256, FLAT, OWN>;
}
template <class T, bool FP8>
AttnFn pick_attn(bool flat_tile, bool own_tile, int dim) {
    return own_tile ? pick_dim<T, FP8, 0, 2>(dim) : flat_tile ? pick_dim<T, FP8, 2, 1>(dim) : pick_dim<T, FP8, 1, 1>(dim);
}

struct AttnPlan {
    bool flat, flat_tile, own_tile;
    uint32_t parts_flat, parts_own, tiles_flat, req_tiles, first;
    uint64_t rows, tiles_own, blocks_flat, blocks;
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
        uint64_t room = 512;
        if (p.flat_tile) {
            const double shared = 2.0 * double(p.tiles_flat) * double(prefix);
            const double beside = double(B * by16) * double(own_keys) * (s->pool_dtype == KVEC_FP8_E4M3 ? 1.0 : 2.0);
            room = uint64_t(512.0 * shared / (shared + beside));
        }
        p.parts_flat = splits(uint64_t(p.tiles_flat) * Hk, prefix, room);
    }
    p.parts_own = splits(own, len > p.first ? len - p.first : 1, 512);
    p.blocks_flat = p.flat ? uint64_t(p.tiles_flat) * Hk * p.parts_flat : 0;
    p.blocks = p.blocks_flat + own * p.parts_own;
    return p;
}

inline int check_attention(const kvec_attention* s, const char* fn) {
    if (!s) return set_error(KVEC_EINVAL, "%s: null descriptor", fn);
    if (s->tokens < 0 || s->batch < 0 || s->heads < 1 || s->kv_heads < 1 || s->heads % s->kv_heads || s->dim < 1 ||
        s->pages_per_seq < 1 || s->pool_pages < 0 || s->prefix < 0)
        return set_error(KVEC_EINVAL, "%s: bad sizes", fn);
    if (s->dtype != KVEC_BF16 && s->dtype != KVEC_F16) return set_error(KVEC_EINVAL, "%s: dtype %d", fn, s->dtype);
    if (s->pool_dtype != s->dtype && s->pool_dtype != KVEC_FP8_E4M3)
        return set_error(KVEC_EINVAL, "%s: pool_dtype %d is neither dtype nor fp8", fn, s->pool_dtype);
    if (s->pool_dtype == s->dtype && (s->k_scale || s->v_scale))
        return set_error(KVEC_EINVAL, "%s: scales are an fp8 pool's", fn);
    const int unit = s->pool_dtype == KVEC_FP8_E4M3 ? 16 : 8;
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
    const int64_t ps = type_bytes(s->pool_dtype);
    const uint64_t rec = 2 * uint64_t(s->kv_heads) * uint64_t(s->dim) * uint64_t(ps);
    if (rec / 2 >= (uint64_t(1) << 30)) return set_error(KVEC_EUNSUPPORTED, "%s: token record too large", fn);
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
    a.direct = p.direct();
    a.scale = s->scale;
    a.wide_q = aligned16(s->q) && s->q_stride % 8 == 0 && s->q_head_stride % 8 == 0;
    a.wide_o = aligned16(s->out) && s->o_stride % 8 == 0 && s->o_head_stride % 8 == 0;
    if (need) {
        a.ws_o = (float*)workspace;
        a.ws_ml = (f32x2*)((uint8_t*)workspace + uint64_t(p.parts_flat + p.parts_own) * p.rows * uint64_t(s->dim) * 4);
    }
    const bool fp8 = s->pool_dtype == KVEC_FP8_E4M3, bf = s->dtype == KVEC_BF16;
    AttnFn f = bf ? (fp8 ? pick_attn<__bf16, true>(p.flat_tile, p.own_tile, s->dim)
                         : pick_attn<__bf16, false>(p.flat_tile, p.own_tile, s->dim))
                  : (fp8 ? pick_attn<_Float16, true>(p.flat_tile, p.own_tile, s->dim)
                         : pick_attn<_Float16, false>(p.flat_tile, p.own_tile, s->dim));
    hipLaunchKernelGGL(f, dim3(unsigned(p.blocks)), dim3(kAB), 0, as_stream(stream), a);
    if ((rc = check_launch(fn)) || p.direct()) return rc;
    uint32_t lanes = 16;
    while (lanes * 4 < a.dim) lanes *= 2;
    const dim3 grid(unsigned(p.rows));
    if (bf) hipLaunchKernelGGL(attn_join_kernel<__bf16>, grid, dim3(kAB), 0, as_stream(stream), a, lanes);
    else hipLaunchKernelGGL(attn_join_kernel<_Float16>, grid, dim3(kAB), 0, as_stream(stream), a, lanes);
    return check_launch(fn);
}
