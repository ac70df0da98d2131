// q3vl_kv_blocks.hpp -- the 8-bit blocks of a cache: where a block keeps its
// values, and what a sequence's lengths let be packed.
#pragma once

#include "q3vl_device.hpp"

namespace q3vl {

constexpr int BLOCK = 32;  // positions of a block

// Byte of position p, value d of a block. Keys lie as v_mfma_f32_16x16x32_f16
// takes them for K Q^T: a lane (i, g) of a 16-key tile has values 8 g + e of 32,
// two products' worth in 16 bytes, the 64 lanes' pieces in order. Values lie so
// for V^T P^T: a lane (i, g) has value i of 16 at positions 4 g + e and 16 + 4 g
// + e, the order in which the probabilities come out of the scores' product, and
// 16 values further on the same again. So a wave reads a block in whole KiB,
// straight into operand registers.
template <int D> __host__ __device__ __forceinline__ constexpr int key_at(int p, int d) {
    return (((p / 16 * (D / 64) + d / 64) * 4 + d % 32 / 8) * 16 + p % 16) * 16 + d % 64 / 32 * 8 + d % 8;
}
template <int D> __host__ __device__ __forceinline__ constexpr int value_at(int p, int d) {
    return ((d / 32 * 4 + p % 16 / 4) * 16 + d % 16) * 16 + d % 32 / 16 * 8 + p / 16 * 4 + p % 4;
}

// What of a sequence can be packed: all of its whole blocks or nothing.
struct Fill {
    int whole;  // blocks to pack
    int rest;   // rows behind them
    int first;  // the block that the first of them becomes
};
__host__ __device__ __forceinline__ Fill filled(int cached, int packed, int max_seq, int blocks) {
    Fill f{0, 0, 0};
    if (cached < 0 || cached > max_seq || packed < 0 || packed % BLOCK || packed / BLOCK > blocks) return f;
    if (cached / BLOCK > blocks - packed / BLOCK) return f;
    f.whole = cached / BLOCK;
    f.rest = cached % BLOCK;
    f.first = packed / BLOCK;
    return f;
}

}  // namespace q3vl
