// norm_rotate.h -- arguments of the kernels that norm and turn heads and write the
// cache, and how a row is cut into units.
#pragma once

#include "lm_types.h"

namespace kvec {

constexpr int kNRB = 256;
constexpr int kMaxDim = 512;
constexpr int kMaxHalf = kMaxDim / 2;

struct NrArgs {
    const uint8_t *q, *k, *v;
    uint8_t* o;
    int64_t qs, qh, ks, kh, vs, vh, os, oh;   // elements
    const uint8_t *wq, *wk;
    const int32_t* pos;
    int64_t axis_stride;
    const uint8_t* axis_of;
    const double* freqs;
    uint8_t* pool;
    const int32_t* slots;
    const float *k_scale, *v_scale;
    const int32_t* n_tokens;
    int64_t n_slots;
    FastDiv div_chunks;                       // pieces of a token's rows, one wave each
    uint32_t items;                           // tokens * pieces
    uint32_t heads, kv_heads, dim, rot, axes;
    uint32_t lg;                              // log2 of the lanes of a row
    int norm, interleaved;
    float eps, factor;
};

// The two chunks of unit u: first values at a and b (b == dim: there is none).
template <int W>
__device__ __forceinline__ void unit_at(const NrArgs& p, uint32_t u, uint32_t& a, uint32_t& b, uint32_t& pair,
                                        bool& turned) {
    const uint32_t half = p.rot / 2, nu = half / W;
    turned = u < nu;
    if (turned) {
        pair = u * W;
        a = p.interleaved ? 2 * u * W : u * W;
        b = p.interleaved ? a + W : half + u * W;
    } else {
        pair = 0;
        a = min(p.rot + (u - nu) * 2 * W, p.dim);
        b = min(a + W, p.dim);
    }
}

// norm_rotate.hip's checks done: the kernel for a pool with block scales (block_write.hip).
int launch_block_write(const NrArgs& a, int64_t tokens, int dtype, int pool_dtype, bool wide, const char* fn, void* stream);

}  // namespace kvec
