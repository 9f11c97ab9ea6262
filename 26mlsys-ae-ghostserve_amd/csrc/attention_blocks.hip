// attention_blocks.hip -- the attention's kernels for pools with block scales.
#include "attention_kernels.h"

namespace kvec {

AttnFn pick_block_attn(bool bf16, int bits, bool flat_tile, bool own_tile, int dim) {
    if (bf16)
        return bits == 8 ? pick_attn<__bf16, kBlock8>(flat_tile, own_tile, dim) : pick_attn<__bf16, kBlock4>(flat_tile, own_tile, dim);
    return bits == 8 ? pick_attn<_Float16, kBlock8>(flat_tile, own_tile, dim) : pick_attn<_Float16, kBlock4>(flat_tile, own_tile, dim);
}

}  // namespace kvec
