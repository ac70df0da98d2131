// kv_blocks.hip -- a cache's whole blocks of 32 positions in 8 bits: written
// from the fp16 rows, and read back. gfx950.
#include "q3vl_device.hpp"
#include "q3vl_kernels.hpp"
#include "q3vl_kv_blocks.hpp"

namespace q3vl {

namespace {

constexpr int THREADS = 256;

typedef _Float16 half8_row __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

}  // namespace

// Where a block's bytes lie in LDS: every 256 of them GAP further, so that a
// wave's accesses to pieces 256 bytes apart (the lane groups g) meet other banks.
constexpr int KGAP = 64, VGAP = 16;
template <int GAP> __device__ __forceinline__ int spread(int at) { return at + at / 256 * GAP; }

// Scale and integers of one block: s = max |x| / 127, n = rne(x / s), both
// quotients correctly rounded, so that the integers are those of their definition
// in fp32 and no value is further than s / 2 from its own. (x / s from r = 1 / s:
// q = x r, then q + (x - q s) r, both fused, is correctly rounded with a correctly
// rounded r, by Markstein's theorem; no step leaves the normal numbers, as x and s
// come from halves.)
//
// One workgroup a (sequence, kv head, block): two waves take the keys, two the
// values. The rows come in whole, 16 bytes a lane, PIECES rows of a value a thread
// for one 32-bit word of LDS each; the maximum of the fp16 bits without their sign
// tells infinities and NaN apart from the rest. The block is put into its order in
// LDS and leaves in pieces of 16 bytes.
//
// The workgroup of a sequence's first block also moves the rows behind the last
// whole one to the front: fewer than 32, which no other workgroup reads, to
// rows that this one alone reads, before it writes them.
//
// Bound by latency at a step's size (192 blocks 5.4 us); a prompt of 4099 rows, 25
// MB in and out, 8.4 us (with the block's bytes unspread in LDS, values a byte at a
// time, and the compiler's division 10.6). The grid is what the cache can hold, not
// what it does: 24 sequences with one whole block among them, 8 heads, us a call 5.0
// at 64 rows a sequence, 5.2 at 512, 14.0 at 4160, 26.5 at 8192.
template <int D> __global__ __launch_bounds__(THREADS) void kv_pack_kernel(KvPackArgs a, int most) {
    constexpr int HALF = THREADS / 2, PIECES = BLOCK * D / 8 / HALF;  // pieces of 8 values a thread
    __shared__ __align__(16) unsigned char tile[2][BLOCK * D / 256 * (256 + KGAP)];
    __shared__ int red[THREADS / 64];
    int x = blockIdx.x;
    const int j = x % most;
    x /= most;
    const int h = x % a.kv_heads, b = x / a.kv_heads;
    const Fill f = filled(a.cache_len[b], a.packed_len[b], a.max_seq, a.blocks);
    if (j >= f.whole) return;
    const int tid = threadIdx.x, part = tid / HALF, t = tid % HALF;  // part 0: keys, 1: values
    uint16_t *rows = (part ? a.v : a.k) + (size_t)b * a.seq_stride + (size_t)h * a.head_stride;
    const int r0 = t / (D / 8) * PIECES, c = t % (D / 8);  // rows r0 .. r0 + PIECES - 1, values 8 c .. 8 c + 7
    half8_row v[PIECES];
    int top = 0;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) v[p] = *reinterpret_cast<const half8_row *>(rows + (size_t)(j * BLOCK + r0 + p) * a.row_stride + c * 8);
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, (int)(__builtin_bit_cast(uint16_t, (_Float16)v[p][e]) & 0x7FFF));
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) top = max(top, __shfl_xor(top, k));
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = max(red[2 * part], red[2 * part + 1]);
    const bool fine = top < 0x7C00;
    const float s = fine ? h2f((uint16_t)top) / 127.0f : __builtin_nanf(""), inv = 1.0f / s;
    uint32_t n[PIECES][8];
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = (float)v[p][e], q = y * inv;
            n[p][e] = fine && top ? (uint32_t)(int)__builtin_rintf(fmaf(fmaf(-q, s, y), inv, q)) & 255 : 0;
        }
    if (part == 0) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            u32x2 w = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e >> 2] |= n[p][e] << (8 * (e & 3));
            *reinterpret_cast<u32x2 *>(tile[0] + spread<KGAP>(key_at<D>(r0 + p, 8 * c))) = w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // PIECES positions of one value
            unsigned char *to = tile[1] + spread<VGAP>(value_at<D>(r0, 8 * c + e));
            if constexpr (PIECES == 4) *reinterpret_cast<uint32_t *>(to) = n[0][e] | n[1][e] << 8 | n[2][e] << 16 | n[3][e] << 24;
            else *reinterpret_cast<uint16_t *>(to) = (uint16_t)(n[0][e] | n[1][e] << 8);
        }
    }
    const size_t to = ((size_t)b * a.kv_heads + h) * a.blocks + f.first + j;
    if (t == 0) (part ? a.v_scale : a.k_scale)[to] = s;
    __syncthreads();
    int8_t *out = (part ? a.v8 : a.k8) + to * (BLOCK * D);
#pragma unroll
    for (int p = 0; p < PIECES / 2; ++p) {
        const int at = (t + p * HALF) * 16;
        *reinterpret_cast<u32x4 *>(out + at) = *reinterpret_cast<const u32x4 *>(tile[part] + (part ? spread<VGAP>(at) : spread<KGAP>(at)));
    }
    if (j) return;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int at = t + p * HALF, r = at / (D / 8), c = at % (D / 8);
        if (r >= f.rest) continue;
        const half8_row y = *reinterpret_cast<const half8_row *>(rows + (size_t)(f.whole * BLOCK + r) * a.row_stride + c * 8);
        *reinterpret_cast<half8_row *>(rows + (size_t)r * a.row_stride + c * 8) = y;
    }
}

__global__ __launch_bounds__(THREADS) void kv_advance_kernel(int32_t *cache_len, int32_t *packed_len, int batch, int max_seq, int blocks) {
    for (int b = blockIdx.x * THREADS + threadIdx.x; b < batch; b += gridDim.x * THREADS) {
        const Fill f = filled(cache_len[b], packed_len[b], max_seq, blocks);
        if (!f.whole) continue;
        packed_len[b] += f.whole * BLOCK;
        cache_len[b] = f.rest;
    }
}

// One workgroup a (sequence, kv head, block that holds a wanted position): the
// block's bytes to LDS as they are, and rows of 8 values from there: a key's are
// eight bytes in a row, a thread takes four positions of eight values, a 32-bit
// word each.
//
// Bound by HBM: 4 sequences of up to 16000 positions, 294 MB in and out, 60 us, 4.9
// TB/s, the rate of a large copy here; 4096 positions 7.2 us (with a byte a read for
// the values 9.8).
template <int D> __global__ __launch_bounds__(THREADS) void kv_unpack_kernel(KvUnpackArgs a, int most) {
    __shared__ __align__(16) unsigned char tile[2][BLOCK * D / 256 * (256 + KGAP)];
    int x = blockIdx.x;
    const int j = x % most;
    x /= most;
    const int h = x % a.kv_heads, b = x / a.kv_heads, tid = threadIdx.x;
    const int first = a.first ? a.first[b] : 0;
    if (first < 0) return;
    const int64_t have = min((int64_t)a.packed_len[b], (int64_t)a.blocks * BLOCK);
    const int64_t end = min((int64_t)first + a.count, have);  // of the positions wanted
    const int64_t blk = first / BLOCK + j, p0 = blk * BLOCK;
    if (p0 >= end) return;
    const size_t from = ((size_t)b * a.kv_heads + h) * a.blocks + blk;
    constexpr int LOADS = BLOCK * D / 16;  // pieces of 16 bytes of one part
#pragma unroll
    for (int i = tid; i < 2 * LOADS; i += THREADS) {
        const int part = i / LOADS, at = i % LOADS * 16;
        *reinterpret_cast<u32x4 *>(tile[part] + (part ? spread<VGAP>(at) : spread<KGAP>(at))) =
            *reinterpret_cast<const u32x4 *>((part ? a.v8 : a.k8) + from * (BLOCK * D) + at);
    }
    const float ks = a.k_scale[from], vs = a.v_scale[from];
    __syncthreads();
    const size_t base = (size_t)b * a.seq_stride + (size_t)h * a.head_stride;
    auto store = [&](uint16_t *rows, int r, int c, const float (&y)[8]) {
        const int64_t p = p0 + r;
        if (p < first || p >= end) return;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = f2h(y[2 * e]) | (uint32_t)f2h(y[2 * e + 1]) << 16;
        *reinterpret_cast<u32x4 *>(rows + base + (size_t)(p - first) * a.row_stride + 8 * c) = w;
    };
    // (the first half of the workgroup keys, the second values)
    constexpr int HALF = THREADS / 2, QUADS = BLOCK / 4 * (D / 8);  // (four positions, eight values)
    const int part = tid / HALF;
    for (int i = tid % HALF; i < QUADS; i += HALF) {
        const int r = i / (D / 8) * 4, c = i % (D / 8);
        float y[4][8];
        if (part == 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(tile[0] + spread<KGAP>(key_at<D>(r + k, 8 * c)));
#pragma unroll
                for (int e = 0; e < 8; ++e) y[k][e] = (float)(int8_t)(w[e >> 2] >> (8 * (e & 3))) * ks;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(tile[1] + spread<VGAP>(value_at<D>(r, 8 * c + e)));
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k][e] = (float)(int8_t)(w >> (8 * k)) * vs;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) store(part ? a.v : a.k, r + k, c, y[k]);
    }
}

hipError_t launch_kv_pack(const KvPackArgs &a, int head_dim, hipStream_t st) {
    const int64_t most = a.max_seq / BLOCK;
    if (most == 0) return hipSuccess;  // no whole block fits the cache
    const unsigned grid = (unsigned)(most * a.kv_heads * a.batch);
    if (head_dim == 128) kv_pack_kernel<128><<<grid, THREADS, 0, st>>>(a, (int)most);
    else kv_pack_kernel<64><<<grid, THREADS, 0, st>>>(a, (int)most);
    return hipGetLastError();
}

hipError_t launch_kv_advance(int32_t *cache_len, int32_t *packed_len, int batch, int max_seq, int blocks, hipStream_t st) {
    const int grid = (batch + THREADS - 1) / THREADS;
    kv_advance_kernel<<<grid < 1024 ? grid : 1024, THREADS, 0, st>>>(cache_len, packed_len, batch, max_seq, blocks);
    return hipGetLastError();
}

hipError_t launch_kv_unpack(const KvUnpackArgs &a, int head_dim, hipStream_t st) {
    // blocks that `count` positions from anywhere on can touch
    const int64_t touched = ((int64_t)a.count + BLOCK - 1) / BLOCK + (a.first ? 1 : 0);
    const int64_t most = touched < a.blocks ? touched : a.blocks;
    const unsigned grid = (unsigned)(most * a.kv_heads * a.batch);
    if (head_dim == 128) kv_unpack_kernel<128><<<grid, THREADS, 0, st>>>(a, (int)most);
    else kv_unpack_kernel<64><<<grid, THREADS, 0, st>>>(a, (int)most);
    return hipGetLastError();
}

}  // namespace q3vl
