// block_read.hip -- tokens of a cache with block scales read back by slot.
//
//   value = code * 2^(byte - 127), rounded to the wanted type
//
// Nothing is computed to speak of: 33 (e4m3) or 17 (e2m1) bytes come in for 64 that
// leave, so the kernel is bound by its stores.  A lane turns 8 neighbours (of 32
// bits: 4) into one 16-byte store, lanes side by side along a token's K and then its V;
// it takes four such pieces, with all their loads in flight before the first
// is used.  32768 tokens of 8 heads of 128 from 8 bits to bf16: 35 to 37 us, 5.6 TB/s;
// 500 tokens 3.1 us.
#include "block_scale.h"

namespace kvec {

constexpr int kBRB = 256;
constexpr int kBRIter = 4;

struct BrArgs {
    const uint8_t* pool;
    const int32_t* slots;
    uint8_t *k, *v;
    int64_t n_slots;
    FastDiv by_token, by_half;                // pieces of a token; of its K
    uint32_t pieces;                          // of all tokens
    uint32_t half;                            // bytes of a half record
    uint32_t scales;                          // where its scales start
};

// A piece: what makes one 16-byte store.
template <class T>
constexpr uint32_t kPiece = 16 / sizeof(T);

// The codes of a piece and their scale as T in memory.
template <int BITS, class T>
__device__ __forceinline__ void put_codes(T* to, u32x2 x, float scale) {
    st16(reinterpret_cast<uint8_t*>(to), widen8<BITS>(x, scale, (T*)nullptr));
}
template <int BITS>
__device__ __forceinline__ void put_codes(float* to, u32x2 x, float scale) {
    typedef float f32x2v __attribute__((ext_vector_type(2)));
    f32x2v f, g;
    if constexpr (BITS == 8) {
        f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x.x, scale, false);
        g = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x.x, scale, true);
    } else {
        f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x.x, scale, 0);
        g = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x.x, scale, 1);
    }
    st16(reinterpret_cast<uint8_t*>(to), u32x4{__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(g.x), __float_as_uint(g.y)});
}
template <int BITS, class T>
__device__ __forceinline__ u32x2 codes_of(const uint8_t* half, uint32_t at) {
    constexpr uint32_t N = kPiece<T> * BITS / 8;              // bytes
    const uint8_t* p = half + at * N;
    if constexpr (N == 8) return *as_global(reinterpret_cast<const u32x2*>(p));
    else if constexpr (N == 4) return u32x2{*as_global(reinterpret_cast<const uint32_t*>(p)), 0};
    else return u32x2{*as_global(reinterpret_cast<const uint16_t*>(p)), 0};
}

template <class T, int BITS>
__global__ __launch_bounds__(kBRB) void block_read_kernel(BrArgs a) {
    const uint32_t first = blockIdx.x * (kBRB * kBRIter) + threadIdx.x;
    uint32_t t[kBRIter], at[kBRIter];
    bool is_v[kBRIter];
    int32_t slot[kBRIter];
#pragma unroll
    for (int i = 0; i < kBRIter; ++i) {
        const uint32_t piece = min(first + i * kBRB, a.pieces - 1);
        t[i] = fdiv(piece, a.by_token);
        at[i] = piece - t[i] * a.by_token.d;
        is_v[i] = at[i] >= a.by_half.d;
        if (is_v[i]) at[i] -= a.by_half.d;
        slot[i] = a.slots[t[i]];
    }
    u32x2 x[kBRIter];
    uint32_t byte[kBRIter];
#pragma unroll
    for (int i = 0; i < kBRIter; ++i) {
        x[i] = u32x2{0, 0};
        byte[i] = 0;
        if (slot[i] >= 0 && int64_t(slot[i]) < a.n_slots) {
            const uint8_t* half = a.pool + (int64_t(slot[i]) * 2 + is_v[i]) * int64_t(a.half);
            x[i] = codes_of<BITS, T>(half, at[i]);
            byte[i] = *as_global(half + a.scales + at[i] / (kScaleBlock / kPiece<T>));
        }
    }
#pragma unroll
    for (int i = 0; i < kBRIter; ++i) {
        if (first + i * kBRB >= a.pieces) break;
        T* out = reinterpret_cast<T*>(is_v[i] ? a.v : a.k) + (uint64_t(t[i]) * a.by_half.d + at[i]) * kPiece<T>;
        put_codes<BITS>(out, x[i], scale_of(byte[i]));
    }
}

typedef void (*BrFn)(BrArgs);

template <class T>
BrFn pick_br(int bits) {
    return bits == 8 ? &block_read_kernel<T, 8> : &block_read_kernel<T, 4>;
}

}  // namespace kvec

using namespace kvec;

extern "C" int kvec_block_read_kv(const kvec_block_read* s, void* stream) {
    static const char* fn = "kvec_block_read_kv";
    if (!s) return set_error(KVEC_EINVAL, "%s: null descriptor", fn);
    if (s->tokens < 0 || s->kv_heads < 1 || s->dim < 1 || s->n_slots < 0) return set_error(KVEC_EINVAL, "%s: bad sizes", fn);
    const int bits = block_bits(s->pool_dtype);
    if (!bits) return set_error(KVEC_EINVAL, "%s: pool_dtype %d has no block scales", fn, s->pool_dtype);
    if (s->dim % kScaleBlock || s->dim > kMaxBlockDim)
        return set_error(KVEC_EUNSUPPORTED, "%s: dim=%d must be a multiple of %d up to %d", fn, s->dim, kScaleBlock, kMaxBlockDim);
    if (s->dtype != KVEC_F32 && s->dtype != KVEC_BF16 && s->dtype != KVEC_F16)
        return set_error(KVEC_EINVAL, "%s: dtype %d", fn, s->dtype);
    if (s->tokens == 0) return KVEC_OK;
    if (!s->slots || !s->k || !s->v || (s->n_slots && !s->pool)) return set_error(KVEC_EINVAL, "%s: null array", fn);
    if (!aligned16(s->pool) || !aligned16(s->k) || !aligned16(s->v))
        return set_error(KVEC_EINVAL, "%s: pool, k or v not 16-byte aligned", fn);
    const uint64_t half = half_bytes(s->kv_heads, s->dim, s->pool_dtype), n = uint64_t(s->kv_heads) * uint64_t(s->dim);
    const uint64_t piece = 16 / uint64_t(type_bytes(s->dtype));
    if (half >= kMaxBlockHalf || uint64_t(s->tokens) >= (uint64_t(1) << 32) ||
        uint64_t(s->tokens) * (2 * n / piece) >= (uint64_t(1) << 32) - kBRB * kBRIter)
        return set_error(KVEC_EUNSUPPORTED, "%s: too many values for one launch", fn);
    const uint64_t out = uint64_t(s->tokens) * n * uint64_t(type_bytes(s->dtype));
    {
        const Span w[2] = {{s->k, out, "k", -1}, {s->v, out, "v", -1}};
        const Span r[2] = {{s->pool, uint64_t(s->n_slots) * 2 * half, "pool", -1}, {s->slots, uint64_t(s->tokens) * 4, "slots", -1}};
        if (int rc = check_no_alias(w, 2, r, 2, fn)) return rc;
    }
    BrArgs a{};
    a.pool = (const uint8_t*)s->pool;
    a.slots = s->slots;
    a.k = (uint8_t*)s->k;
    a.v = (uint8_t*)s->v;
    a.n_slots = s->n_slots;
    a.by_half = make_fastdiv(uint32_t(n / piece));
    a.by_token = make_fastdiv(uint32_t(2 * n / piece));
    a.pieces = uint32_t(uint64_t(s->tokens) * (2 * n / piece));
    a.half = uint32_t(half);
    a.scales = uint32_t(n * uint64_t(bits) / 8);
    BrFn f = s->dtype == KVEC_F32 ? pick_br<float>(bits) : s->dtype == KVEC_BF16 ? pick_br<__bf16>(bits) : pick_br<_Float16>(bits);
    const unsigned blocks = unsigned((uint64_t(a.pieces) + kBRB * kBRIter - 1) / (kBRB * kBRIter));
    hipLaunchKernelGGL(f, dim3(blocks), dim3(kBRB), 0, as_stream(stream), a);
    return check_launch(fn);
}
