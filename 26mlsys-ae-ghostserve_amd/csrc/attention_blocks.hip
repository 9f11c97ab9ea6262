// attention_blocks.hip -- the attention's kernels for pools with block scales.
#include "attention_kernels.h"

namespace kvec {

namespace {

template <class T, int POOL, int DP>
AttnFn pick_rows(bool flat_tile, bool own_tile, int heads) {
    if (own_tile) return &attn_kernel<T, POOL, DP, 0, 2>;
    if constexpr (POOL == kBlock4) {
        if (heads == 2) return flat_tile ? &attn_kernel<T, POOL, DP, 2, 1, 2> : &attn_kernel<T, POOL, DP, 1, 1, 2>;
    }
    return flat_tile ? &attn_kernel<T, POOL, DP, 2, 1, 1> : &attn_kernel<T, POOL, DP, 1, 1, 1>;
}
template <class T, int POOL>
AttnFn pick_block_dim(bool flat_tile, bool own_tile, int heads, int dim) {
    return dim <= 64    ? pick_rows<T, POOL, 64>(flat_tile, own_tile, heads)
           : dim <= 96  ? pick_rows<T, POOL, 96>(flat_tile, own_tile, heads)
           : dim <= 128 ? pick_rows<T, POOL, 128>(flat_tile, own_tile, heads)
                        : pick_rows<T, POOL, 256>(flat_tile, own_tile, heads);
}

}  // namespace

AttnFn pick_block_attn(bool bf16, int bits, bool flat_tile, bool own_tile, int heads, int dim) {
    if (bf16)
        return bits == 8 ? pick_block_dim<__bf16, kBlock8>(flat_tile, own_tile, heads, dim)
                         : pick_block_dim<__bf16, kBlock4>(flat_tile, own_tile, heads, dim);
    return bits == 8 ? pick_block_dim<_Float16, kBlock8>(flat_tile, own_tile, heads, dim)
                     : pick_block_dim<_Float16, kBlock4>(flat_tile, own_tile, heads, dim);
}

}  // namespace kvec
