// q3vl_kv_blocks.hpp -- the 8-bit blocks of a cache: where a block keeps its
// values, and what a sequence's lengths let be packed.
#pragma once

#include "q3vl_device.hpp"
#include "q3vl_mfma.hpp"

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

// Eight int8 as fp16, exactly: a byte u under the byte 0x64 is the half 1024 + u,
// so x ^ 0x80 gives 1152 + x. (No asm as in widen8: the compiler moves these
// instructions between the products and knows their waits.)
Q3VL_INLINE half8_t widen8_plain(uint32_t x, uint32_t y) {
    typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
    const half2_t off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    x ^= 0x80808080u;
    y ^= 0x80808080u;
    auto part = [&](uint32_t v, uint32_t sel) {
#if defined(__HIP_DEVICE_COMPILE__)
        return __builtin_bit_cast(uint32_t, (half2_t)(__builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, v, sel)) + off));
#else
        return v;
#endif
    };
    return __builtin_bit_cast(half8_t, (u32x4){part(x, 0x04010400u), part(x, 0x04030402u), part(y, 0x04010400u), part(y, 0x04030402u)});
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
