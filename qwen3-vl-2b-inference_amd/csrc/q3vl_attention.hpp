// q3vl_attention.hpp -- device pieces that the attentions over rows of tokens
// share: operand types, LDS places of cached rows, masks, the probabilities'
// range.
#pragma once

#include "q3vl_device.hpp"
#include "q3vl_mfma.hpp"

namespace q3vl {

// p is held as 2^(s sc + bias): a row's largest score gets 2^BASE, and one that
// passes it by up to GROW stays under fp16's 2^16 (tree_attention.hip).
constexpr float BASE = 6.0f, GROW = 9.0f;

// (rows of q and out may lie anywhere)
typedef _Float16 half8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t half4_bits __attribute__((ext_vector_type(4), aligned(2)));
typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ half4_t read_transposed(unsigned char *p) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)p));
#else
    return half4_t{};
#endif
}

// Where a row's 16-byte pieces lie: piece c at c ^ swizzle(row). The LDS serves
// 256 bytes a clock: a b64 read 32 lanes in order, a b128 read 16, of lanes 0 ..
// 31 first 0-3, 12-15, 20-27 (by the conflicts counted with other swizzles). So
// V is read by 8 consecutive rows at a time, two neighbouring pieces each: 8
// different pairs; K by rows 0-3 and 12-15 at piece c and rows 4-11 at c ^ 1, or
// the reverse: even and odd places. No conflicts are left (c ^ row: 2-way in V).
template <int D> __device__ __forceinline__ int swizzle(int r) { return D == 128 ? (r & 7) << 1 : r & 6; }

// Largest value of the four lanes i, i + 16, i + 32, i + 48, in each of them.
__device__ __forceinline__ float column_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// Their sum.
__device__ __forceinline__ float column_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// 32 bits of a row's mask line from bit i on (i may be negative: positions
// before the drafts, all seen); n rows exist.
__device__ __forceinline__ uint32_t mask_window(const uint64_t *line, int words, int n, int i) {
    const int at = max(i, 0), w = at >> 6, sh = at & 63;
    uint64_t v = w < words ? line[w] >> sh : 0;
    if (sh && w + 1 < words) v |= line[w + 1] << (64 - sh);
    const int left = n - at;
    if (left < 64) v &= left > 0 ? (1ull << left) - 1 : 0;
    if (i <= -32) return 0xFFFFFFFFu;
    return i < 0 ? (uint32_t)(v << -i) | ((1u << -i) - 1) : (uint32_t)v;
}

template <bool HALF> __device__ __forceinline__ void put(void *out, int64_t at, float v) {
    if (HALF) static_cast<uint16_t *>(out)[at] = f2h(v);
    else static_cast<float *>(out)[at] = v;
}

}  // namespace q3vl
