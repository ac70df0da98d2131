// long_attention.hip -- attention over long contexts: positions in 8-bit blocks
// and the fp16 rows behind them, all of them or a window of them with a few
// first ones. gfx950.
#include "q3vl_attention.hpp"
#include "q3vl_device.hpp"
#include "q3vl_kernels.hpp"
#include "q3vl_kv_blocks.hpp"
#include "q3vl_mfma.hpp"

#include <type_traits>
#include <utility>

namespace q3vl {

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;

// Weights p |vs| of packed positions: set to 2^BASE .. 2^(BASE + 2), they may grow
// by 2^MORE before they are set anew, and stay under 2^15.
constexpr float MORE = 7.0f;

// What a block knows of its sequence.
struct LongSeq {
    int start, n;  // its rows of q
    int packed;    // positions in 8-bit blocks
    int len;       // fp16 rows before the step's own
    bool ok;       // all of them fit
};
__device__ __forceinline__ LongSeq long_sequence(const LongAttnArgs &a, int b) {
    LongSeq s;
    s.start = min(max(a.row_start[b], 0), a.rows);
    s.n = min(max(a.row_start[b + 1], s.start), a.rows) - s.start;
    s.len = a.cache_len[b];
    s.ok = s.len >= 0 && (int64_t)s.len + s.n <= a.max_seq;
    s.packed = 0;
    if (a.packed_len) {
        s.packed = a.packed_len[b];
        s.ok = s.ok && s.packed >= 0 && s.packed % BLOCK == 0 && s.packed / BLOCK <= a.blocks;
    }
    return s;
}

// Positions in order: the packed ones, the fp16 rows before the step's, the
// step's own. Row t sees those before the step's, and of the step's rows t and
// earlier ones, or its mask's; of what it sees the first `sinks` and the last
// `window`. `from`: the first of the latter among the positions before the
// step's own and, without a mask, among those too (with one, every row of the
// mask is within the window).
__device__ __forceinline__ int64_t window_from(const LongAttnArgs &a, const LongSeq &s, int t) {
    if (!a.window) return 0;
    int64_t seen = (int64_t)s.packed + s.len;
    if (a.mask) {
        const uint64_t *line = a.mask + (size_t)(s.start + t) * a.words;
        for (int w = 0; w < a.words && w * 64 < s.n; ++w) {
            uint64_t v = line[w];
            if (s.n - w * 64 < 64) v &= (1ull << (s.n - w * 64)) - 1;
            seen += __popcll(v);
        }
        return min(seen - a.window, (int64_t)s.packed + s.len);
    }
    return seen + t + 1 - a.window;
}
__device__ __forceinline__ bool long_sees(const LongAttnArgs &a, const LongSeq &s, int t, int64_t from, int64_t j) {
    const int64_t i = j - s.packed - s.len;
    if (i >= 0 && a.mask) return i < s.n && i < 64 * (int64_t)a.words && (a.mask[(size_t)(s.start + t) * a.words + (i >> 6)] >> (i & 63) & 1);
    if (i > t) return false;
    return j >= from || j < a.sinks;
}

// Turns of UNIT positions: those of the packed ones, then those of the fp16
// rows; of them the ones with a first position, and the ones from the window's
// first position on.
template <int UNIT> struct Turns {
    int packed;     // turns of packed positions
    int first;      // turns [0, first) hold first positions
    int skip;       // the next one after them is first + skip
    int count;      // turns in all
    __device__ __forceinline__ int at(int i) const { return i < first ? i : i + skip; }
};
template <int UNIT> __device__ __forceinline__ Turns<UNIT> turns_of(const LongAttnArgs &a, const LongSeq &s, int rows, int64_t from) {
    Turns<UNIT> u;
    u.packed = (s.packed + UNIT - 1) / UNIT;
    const int all = u.packed + (int)(((int64_t)rows + UNIT - 1) / UNIT);
    u.first = all;
    u.skip = 0;
    if (a.window) {
        auto turn = [&](int64_t j) {  // that holds position j
            return (int)(j < s.packed ? j / UNIT : u.packed + (j - s.packed) / UNIT);
        };
        const int end = a.sinks > 0 ? turn(a.sinks - 1) + 1 : 0;
        u.first = min(end, all);
        u.skip = max(0, min(from > 0 ? turn(from) : 0, all) - u.first);
    }
    u.count = all - u.skip;
    return u;
}

struct LongScratch {
    float q[128];
    float p[THREADS];
    uint64_t seen[WAVES];
    float red[WAVES];
};

// One row and head over turns [i0, i1), plainly and in fp32, by a whole block: o
// (threads 0 .. D-1) = sum p v, p = 2^(s - m), l = sum p, with s the scores times
// log2 e. m is -inf where nothing is seen (then o = l = 0), else at least
// -FLT_MAX. Products of what the row does not see are never formed.
template <int D, bool HALF, int UNIT>
__device__ void long_row(const LongAttnArgs &a, const LongSeq &s, int b, int t, int head, const Turns<UNIT> &turns, int i0, int i1,
                         LongScratch &sh, float &o, float &m, float &l) {
    const int tid = threadIdx.x, lane = tid & 63, h = head / (a.heads / a.kv_heads);
    const size_t base = (size_t)b * a.seq_stride + (size_t)h * a.head_stride;
    const size_t blocks = ((size_t)b * a.kv_heads + h) * a.blocks;
    const int64_t qat = (int64_t)(s.start + t) * a.ldq + (int64_t)head * D;
    const int64_t from = window_from(a, s, t);
    __syncthreads();
    if (tid < D) sh.q[tid] = HALF ? h2f(static_cast<const uint16_t *>(a.q)[qat + tid]) : static_cast<const float *>(a.q)[qat + tid];
    o = l = 0.0f;
    m = -INFINITY;
    for (int i = i0; i < i1; ++i) {
        const int u = turns.at(i);
        const bool packed = u < turns.packed;
        const int first = (packed ? u : u - turns.packed) * UNIT, j = first + tid;  // among their own kind
        const int count = min(UNIT, (packed ? s.packed : s.len + s.n) - first);
        const bool seen = tid < count && long_sees(a, s, t, from, (packed ? 0 : (int64_t)s.packed) + j);
        float sc = -INFINITY;
        __syncthreads();  // the scratch of the last turn is read
        if (seen) {
            float acc = 0.0f;
            if (packed) {
                const size_t blk = blocks + j / BLOCK;
                const int8_t *k = a.k8 + blk * (BLOCK * D);
                for (int d = 0; d < D; ++d) acc = fmaf(sh.q[d], (float)k[key_at<D>(j % BLOCK, d)], acc);
                acc *= a.k_scale[blk];
            } else {
                const uint16_t *k = a.k_cache + base + (size_t)j * a.row_stride;
                for (int d = 0; d < D; ++d) acc = fmaf(sh.q[d], h2f(k[d]), acc);
            }
            sc = acc * a.scale_log2e;
        }
        float top = sc;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
        const uint64_t any = __ballot(seen);
        if (lane == 0) {
            sh.red[tid >> 6] = top;
            sh.seen[tid >> 6] = any;
        }
        __syncthreads();
        uint64_t some = 0;
        for (int w = 0; w < WAVES; ++w) {
            top = fmaxf(top, sh.red[w]);
            some |= sh.seen[w];
        }
        if (!some) continue;
        const float ref = fmaxf(fmaxf(m, top), -FLT_MAX);
        const float shrink = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - ref);
        m = ref;
        const float p = seen ? __builtin_amdgcn_exp2f(sc - ref) : 0.0f;
        sh.p[tid] = p;
        float sum = p;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
        __syncthreads();
        if (lane == 0) sh.red[tid >> 6] = sum;
        __syncthreads();
        l = l * shrink;
        for (int w = 0; w < WAVES; ++w) l += sh.red[w];
        o *= shrink;
        if (tid < D)
            for (int k = 0; k < count; ++k)
                if (sh.seen[k >> 6] >> (k & 63) & 1) {
                    float v;
                    if (packed) {
                        const size_t blk = blocks + (first + k) / BLOCK;
                        v = (float)a.v8[blk * (BLOCK * D) + value_at<D>((first + k) % BLOCK, tid)] * a.v_scale[blk];
                    } else {
                        v = h2f(a.v_cache[base + (size_t)(first + k) * a.row_stride + tid]);
                    }
                    o = fmaf(sh.p[k], v, o);
                }
    }
}

}  // namespace

// ------------------------------------------------------------ the kernel
// Scores, softmax and values of 32 positions a step as in tree_attention_kernel,
// which tells the layout: S^T = K Q^T and O^T = V^T P^T by v_mfma_f32_16x16x32_f16,
// a query row in a lane, p held as 2^(s sc + bias). fp16 rows come as they do there.
// What differs:
//
// Packed blocks. int8 are exact in fp16, so a block's integers are operands as they
// are, and its scales are factors: the keys' of the score (sc ks), the values' of
// the probability, p vs. These weights have a reference of their own: each row's are
// in units of a power of two that puts the largest p |vs| which the row has seen so
// far at 2^BASE or a little more, whatever the scales of blocks that it does not see
// or that weigh nothing in it; O is in those units until the packed positions are
// done. l sums p itself, in fp32 and in the lane: a key with much weight and tiny
// values must count in it. So no p vs is held finer than 2^-31 of the row's largest
// p |vs|, as no p of a fp16 row finer than 2^-31 of its largest.
//
// Few rows: a wave takes a block of every four, 16 bytes a lane and load, straight
// from memory into operand registers (the block's order is theirs) and widens them
// there; a block's registers are filled again as soon as they are read, the next
// block is on its way meanwhile. No LDS, no barrier. Bound by the reads: one token
// each of 24 sequences of up to 12000, 472 MB, 81 us, 5.8 TB/s, 32 of 16384 all
// alike 6.5 (a plain read here: 6.46); the rest is sequences of different length.
// Of the busy cycles the matrix cores work in 16 of 100 and other vector
// instructions run in 42.
//
// Many rows: the four waves each widen a quarter of the next 64 positions into LDS,
// in the operands' order, read ahead by a turn (each wave widening all of them for
// itself: three trees of 61 rows over 16000 128 us for 63). Trees 60 us, 1000 rows
// behind 8000 in fp16 89; matrix cores 36 of 100, other vector instructions 40 and
// 49, two waves a SIMD. (One unit for all rows of a wave, which loses bits: 59 and
// 87.) In fp32 and heads of 128 the tiles of 128 rows take all 256 registers, with 6
// spilled over blocks and 8 without.
//
// A window. The turns that no row of the workgroup sees are left out: the ones of
// the first positions come first, then from the earliest window's start on. Within
// the others a lane masks what its row does not see, where some row does not see
// all. One token of 16 sequences through 4096 positions 45 us, 6.0 TB/s; a prompt
// of 4000 through 1024 in fp16 49 us.
template <int D, int NR, bool SHARED, bool PACKED> struct LongTile {
    static constexpr int RB = 2 * D;                           // bytes of an fp16 row
    static constexpr int NS = SHARED ? 2 : PACKED ? 128 / D : 256 / D;  // stages of fp16 rows
    static constexpr int STAGE = (SHARED ? 64 : 32) * RB * 2;  // K, then V
    static constexpr int RING = (SHARED ? 1 : WAVES) * NS * STAGE;
    static constexpr int BM = 16 * NR * (SHARED ? WAVES : 1);  // query rows of a workgroup
    static constexpr int OS = D + 4;                           // floats of a joined row (spread over the banks)
    static constexpr int JOIN = SHARED ? 0 : WAVES * BM * OS * 4;
    static constexpr int ML = RING > JOIN ? RING : JOIN;       // (M, l) of each wave's rows
    static constexpr int FLAG = ML + (SHARED ? 0 : WAVES * BM * 8);
    static constexpr int LDS = FLAG + (BM + 1) * 4;
    static constexpr int UNIT = SHARED ? 64 : 32 * WAVES;      // positions of a turn
    static_assert(LDS <= 160 * 1024 && sizeof(LongScratch) <= (size_t)RING, "LDS");
};

// A block of 32 packed positions on its way to the operands.
template <int D> struct PackedBlock {
    u32x4 k[2 * D / 64], v[D / 32];
    float ks, vs;
};

// ONCE: no other workgroup reads this one's keys and values; they go past the caches.
template <int D, bool HALF, int NR, bool SHARED, bool PACKED, bool ONCE>
__global__ __launch_bounds__(THREADS, SHARED || PACKED ? 2 : 1) void long_attention_kernel(
    const int32_t *row_start_p, const int32_t *cache_len_p, const void *q_p, const int32_t *packed_len_p, int kv_heads_p, int heads_p,
    int splits_p, int rows_p, int max_rows_p, int max_seq_p, int tiles, int paired, LongAttnArgs args) {
    LongAttnArgs a = args;  // (the leading arguments arrive in registers)
    a.row_start = row_start_p;
    a.cache_len = cache_len_p;
    a.q = q_p;
    a.packed_len = PACKED ? packed_len_p : nullptr;
    a.kv_heads = kv_heads_p;
    a.heads = heads_p;
    a.splits = splits_p;
    a.rows = rows_p;
    a.max_rows = max_rows_p;
    a.max_seq = max_seq_p;
    using T = LongTile<D, NR, SHARED, PACKED>;
    constexpr int KS = D / 32, NT = D / 16, NQ = HALF ? 1 : 2, UNIT = T::UNIT;
    constexpr int NT_BIT = ONCE ? 2 : 0;  // (a buffer load's non-temporal bit)
    extern __shared__ __align__(16) unsigned char smem[];
    // (loads with an LDS destination take its offset: 0, as the kernel has no other LDS)
    const int tid = threadIdx.x, wid = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, i = lane & 15, g = lane >> 4;
    int x = blockIdx.x;  // kv head, split, tile, sequence
    const int h = x % a.kv_heads;
    x /= a.kv_heads;
    const int split = x % a.splits;
    x /= a.splits;
    const int b = x / tiles;
    x -= b * tiles;
    // a chain's last rows see most: they go first, and where every workgroup has
    // a place at once, the second half goes the other way round
    const int tile = paired && 2 * x >= tiles ? x - (tiles + 1) / 2 : tiles - 1 - x;
    const LongSeq s = long_sequence(a, b);
    const int group = a.heads / a.kv_heads;
    const int n = min(s.n, a.max_rows), nrows = n * group, r0 = tile * T::BM;
    if (r0 >= nrows) return;

    int row[NR], tok[NR], head[NR];  // of column i: its row, token, query head
    bool live[NR];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        row[nr] = r0 + (SHARED ? wid * 16 * NR : 0) + nr * 16 + i;
        live[nr] = row[nr] < nrows;
        tok[nr] = live[nr] ? row[nr] / group : 0;
        head[nr] = h * group + (live[nr] ? row[nr] - tok[nr] * group : 0);
    }
    if (!s.ok) {
        if (a.splits == 1)
            for (int e = tid; e < min(T::BM, nrows - r0) * D; e += THREADS) {
                const int r = r0 + e / D, t = r / group;
                put<HALF>(a.out, (int64_t)(s.start + t) * a.ldo + (int64_t)(h * group + r - t * group) * D + e % D, __builtin_nanf(""));
            }
        return;
    }

    // ---- this workgroup's turns
    const int before = s.packed + s.len;  // positions before the step's
    const int first_tok = (r0 + (SHARED ? wid * 16 * NR : 0)) / group;  // of this wave's rows
    const int tile_tok = r0 / group, last_tok = min((r0 + T::BM - 1) / group, n - 1);
    const int total = s.len + (a.mask ? s.n : last_tok + 1);  // fp16 rows that some row sees
    const Turns<UNIT> turns = turns_of<UNIT>(a, s, total, (int64_t)before + (a.mask ? 0 : tile_tok + 1) - a.window);
    const int u0 = (int)((int64_t)turns.count * split / a.splits), u1 = (int)((int64_t)turns.count * (split + 1) / a.splits);

    int tp = u0;  // turns [u0, tp) are of packed positions (turns.at rises: they come first)
    if constexpr (PACKED) {
        const int end = turns.first < turns.packed ? max(turns.first, turns.packed - turns.skip) : turns.packed;
        tp = min(max(end, u0), u1);
    }

    // ---- queries (the first tiles' loads go out behind theirs, before they are used)
    half8_any qh[NR][KS];
    float4_any qs[NR][KS][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        const int64_t at = (int64_t)(s.start + tok[nr]) * a.ldq + (int64_t)head[nr] * D + 8 * g;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if constexpr (HALF) {
                qh[nr][ks] = *reinterpret_cast<const half8_any *>(static_cast<const _Float16 *>(a.q) + at + 32 * ks);
            } else {
                const float *p = static_cast<const float *>(a.q) + at + 32 * ks;
                qs[nr][ks][0] = *reinterpret_cast<const float4_any *>(p);
                qs[nr][ks][1] = *reinterpret_cast<const float4_any *>(p + 4);
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);

    // ---- loads of fp16 rows: a lane's place in 16 rows of the cache, and of LDS
    const size_t head_at = (size_t)b * a.seq_stride + (size_t)h * a.head_stride;
    const int rsb = (int)(a.row_stride * 2);
    constexpr int NL = (SHARED ? 1 : 2) * (D / 32);  // loads of a K or V part
    int voff[NL];
#pragma unroll
    for (int t = 0; t < NL; ++t) {
        const int r = (t * 64 + lane) / (D / 8), c = lane % (D / 8);
        voff[t] = (r + (SHARED ? wid * 16 : 0)) * rsb + (c ^ swizzle<D>(r)) * 16;
    }
    // rows from p on, `left` of them there: 32 to this wave's own stage, or its
    // 16 of a tile's 64. Rows past the end read as zeros by the buffer's bounds.
    auto load_rows = [&](const uint16_t *p, int left, int lds) {
        left = min(left, SHARED ? 64 : 32);
        const rsrc_t r = make_rsrc(p, left > 0 ? (uint32_t)((left - 1) * rsb + 2 * D) : 0);
#pragma unroll
        for (int t = 0; t < NL; ++t) {
            const int at = lds + ((SHARED ? wid * NL : 0) + t) * 1024;
            if constexpr (ONCE) dma16_nt(r, voff[t], 0, at);
            else dma16(r, voff[t], 0, at);
        }
    };
    const size_t head_blocks = ((size_t)b * a.kv_heads + h) * a.blocks;
    const int held = s.packed / BLOCK;
    // (SHARED) turn u's fp16 rows to LDS at `lds`
    auto load_tile = [&](int u, int lds) {
        const int first = (u - turns.packed) * UNIT;
        const size_t at = head_at + (size_t)first * a.row_stride;
        load_rows(a.k_cache + at, total - first, lds);
        load_rows(a.v_cache + at, total - first, lds + 64 * T::RB);
    };
    // ... its two packed blocks: this wave's quarter of the keys and of the values
    // to registers, and from there, widened, to LDS, in the operands' order
    constexpr int PER = SHARED && PACKED ? 2 * BLOCK * D / 1024 / WAVES : 1;  // KiB of int8
    u32x4 nk[PER], nv[PER];
    auto fetch_tile = [&](int u) {
        const int left = min(held - u * 2, 2) * (BLOCK * D);  // bytes of a part
        const size_t at = (head_blocks + u * 2) * (BLOCK * D);
        const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(a.k8 + at), 0, left, 0x00020000);
        const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(a.v8 + at), 0, left, 0x00020000);
#pragma unroll
        for (int k = 0; k < PER; ++k) nk[k] = __builtin_amdgcn_raw_buffer_load_b128(rk, (wid * PER + k) * 1024 + lane * 16, 0, NT_BIT);
#pragma unroll
        for (int k = 0; k < PER; ++k) nv[k] = __builtin_amdgcn_raw_buffer_load_b128(rv, (wid * PER + k) * 1024 + lane * 16, 0, NT_BIT);
    };
    // ... their scales, a turn ahead too (keys', then values'; of the last block twice)
    float scale[4];
    auto fetch_scales = [&](int u) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const size_t at = head_blocks + min(u * 2 + k, held - 1);
            scale[k] = a.k_scale[at];
            scale[2 + k] = a.v_scale[at];
        }
    };
    auto widen_tile = [&](int lds) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            unsigned char *p = smem + lds + (wid * PER + k) * 2048 + lane * 16;
            *reinterpret_cast<half8_t *>(p) = widen8_plain(nk[k][0], nk[k][1]);
            *reinterpret_cast<half8_t *>(p + 1024) = widen8_plain(nk[k][2], nk[k][3]);
            *reinterpret_cast<half8_t *>(p + 64 * T::RB) = widen8_plain(nv[k][0], nv[k][1]);
            *reinterpret_cast<half8_t *>(p + 64 * T::RB + 1024) = widen8_plain(nv[k][2], nv[k][3]);
        }
    };

    // ---- operand registers, the score's factor
    half8_t qf[NR][NQ][KS];
    float sc[NR];
    auto queries = [&] {
        const float sign = a.scale_log2e < 0.0f ? -1.0f : a.scale_log2e == 0.0f ? 0.0f : 1.0f;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            sc[nr] = sign == 0.0f ? 1.0f : fabsf(a.scale_log2e);
            if constexpr (HALF) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < 8; ++e) qf[nr][0][ks][e] = live[nr] ? (_Float16)(qh[nr][ks][e] * (_Float16)sign) : (_Float16)0.0f;
            } else {
                float v[KS][8], top = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[ks][e] = live[nr] ? qs[nr][ks][e >> 2][e & 3] * sign : 0.0f;
                        top = fmaxf(top, fabsf(v[ks][e]));
                    }
                top = column_max(top);
                // the largest value to [2^13, 2^14)
                const int shift = top > 0.0f && top < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
                sc[nr] = ldexpf(sc[nr], -shift);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float y = ldexpf(v[ks][e], shift);
                        qf[nr][0][ks][e] = (_Float16)y;
                        qf[nr][1][ks][e] = (_Float16)(y - (float)qf[nr][0][ks][e]);
                    }
            }
        }
    };

    // ---- what a row's window holds: positions from lo[] on, and below `sinks`
    int lo[NR], lo_most = 0;  // (lo_most: of this wave's rows)
    const bool windowed = a.window != 0;
    if (windowed) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) lo[nr] = (int)max(window_from(a, s, tok[nr]), (int64_t)0);
        const int last = min((r0 + (SHARED ? (wid + 1) * 16 * NR : T::BM) - 1) / group, n - 1);
        const int64_t most = (int64_t)before + (a.mask ? min((int64_t)0, (int64_t)s.n - a.window) : (int64_t)last + 1 - a.window);
        lo_most = (int)max(most, (int64_t)0);
    }
    // whether all of this wave's rows see positions j .. j + 31, as far as the window goes
    auto inside = [&](int j) { return !windowed || j >= lo_most || j + 32 <= a.sinks; };
    auto window_bits = [&](int nr, int j) {
        auto from = [](int k) { return k <= 0 ? 0xFFFFFFFFu : k >= 32 ? 0u : 0xFFFFFFFFu << k; };  // bits from k on
        return from(lo[nr] - j) | ~from(a.sinks - j);
    };
    // fp16 rows below this are seen by all of this wave's rows, as far as the mask goes
    const int clear = min(s.len + (a.mask ? 0 : min(first_tok, n - 1) + 1), total);

    // ---- one step: 32 positions
    int kaddr[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kaddr[ks] = i * T::RB + ((ks * 4 + g) ^ swizzle<D>(i)) * 16;
    const int vr = 4 * g + (i >> 2);  // row of a 16-position tile this lane's transposing read starts from
    const int vaddr = vr * T::RB + (((i & 3) >> 1) ^ swizzle<D>(vr)) * 16 + (i & 1) * 8;
    float M[NR], bias[NR];
    float limit[NR];  // of fp16 rows: the score from which M is set anew
    float4_t O[NT][NR], L[NR];  // L: the sum of p, in each register and lane of the column,
    float lsum[NR];             // and of packed positions, this lane's share
    bool any[NR];
    float most[NR];  // of packed positions: log2 of p |vs|, and 126, from which O's units are set anew
    int units[NR];   // those units, a power of two
    auto clear_rows = [&] {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            M[nr] = limit[nr] = most[nr] = -INFINITY;
            bias[nr] = lsum[nr] = 0.0f;
            units[nr] = 0;
            any[nr] = false;
            if constexpr (!PACKED) L[nr] = float4_t{0, 0, 0, 0};
#pragma unroll
            for (int dt = 0; dt < NT; ++dt) O[dt][nr] = float4_t{0, 0, 0, 0};
        }
    };
    float4_t S[2][NR];
    half8_t P[NR][NQ];
    auto zero_scores = [&](int kb) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) S[kb][nr] = float4_t{0, 0, 0, 0};
    };
    auto score = [&](half8_t f, int kb, int ks) {
#pragma unroll
        for (int q = NQ - 1; q >= 0; --q)
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) S[kb][nr] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, qf[nr][q][ks], S[kb][nr], 0, 0, 0);
    };
    auto value = [&](half8_t f, int dt) {
#pragma unroll
        for (int q = NQ - 1; q >= 0; --q)
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) O[dt][nr] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, P[nr][q], O[dt][nr], 0, 0, 0);
    };
    auto masked = [&](int nr, uint32_t w) {  // scores of positions whose bit is not set
        any[nr] = any[nr] || w;
        w >>= 4 * g;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!(w >> (16 * kb + e) & 1)) S[kb][nr][e] = -INFINITY;
    };
    // probabilities of scores ks S; those of packed positions times the values' scale
    auto softmax = [&](float ks, float vs, auto packed) {
        float top[NR];  // of this lane's positions
        bool grow = false;
        const float by = (float)(__float_as_uint(vs) >> 23 & 255);  // |vs| is in [2^(by - 127), 2^(by - 126)), or less for by = 0
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            top[nr] = S[0][nr][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top[nr] = fmaxf(top[nr], S[e >> 2][nr][e & 3]);
            if constexpr (packed) {
                top[nr] *= ks;
                grow = grow || fmaf(top[nr], sc[nr], bias[nr]) > fminf(BASE + GROW, most[nr] - by);
            } else {
                grow = grow || top[nr] > limit[nr];
            }
        }
        if (__any(grow)) {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                const float t = column_max(top[nr]), m = fmaxf(M[nr], t);
                const float nb = m == -INFINITY ? 0.0f : fmaf(-m, sc[nr], BASE);
                const float f = M[nr] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(nb - bias[nr]);
                float fo = f;
                if constexpr (packed) {  // the largest weight to [2^BASE, 2^(BASE + 2)), or up to that from below
                    const float w = fmaxf(M[nr] == -INFINITY ? M[nr] : most[nr] - MORE + (nb - bias[nr]), fmaf(t, sc[nr], nb) + by);
                    const int to = (int)fminf(fmaxf(floorf(w - (BASE + 127.0f)), -999.0f), 999.0f);
                    fo = ldexpf(f, units[nr] - to);
                    units[nr] = to;
                    most[nr] = m == -INFINITY ? m : (float)to + (BASE + 127.0f + MORE);
                } else {
                    limit[nr] = m == -INFINITY ? m : m + GROW / sc[nr];  // (the quotient is infinite for the smallest queries)
                    L[nr] *= f;
                }
                M[nr] = m;
                bias[nr] = nb;
                if constexpr (PACKED) lsum[nr] *= f;
#pragma unroll
                for (int dt = 0; dt < NT; ++dt) O[dt][nr] *= fo;
            }
        }
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const float c = packed ? sc[nr] * ks : sc[nr];
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(S[e >> 2][nr][e & 3], c, bias[nr]));
            if constexpr (packed) {
                const float v = ldexpf(vs, -units[nr]);
#pragma unroll
                for (int e = 0; e < 8; ++e) lsum[nr] += p[e];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] *= v;
                    // (the product as it is rounded here: fused into the conversion below, the
                    // first term would now and then be another than the one the rest is of)
                    asm("" : "+v"(p[e]));
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                P[nr][0][e] = (_Float16)p[e];
                if constexpr (!HALF) P[nr][1][e] = (_Float16)(p[e] - (float)P[nr][0][e]);
            }
        }
    };
    constexpr std::integral_constant<bool, true> kPacked{};
    constexpr std::integral_constant<bool, false> kRows{};

    auto packed_softmax = [&](float ks, float vs, int j, bool there = true) {
        if (there && inside(j)) {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) any[nr] = true;
        } else {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) masked(nr, there ? windowed ? window_bits(nr, j) : 0xFFFFFFFFu : 0u);
        }
        softmax(ks, vs, kPacked);
    };
    // 32 packed positions from j on, out of registers; more_k and more_v: the keys'
    // and the values' registers are free
    auto packed_step = [&](const PackedBlock<D> &f, int j, auto more_k, auto more_v) {
        const float ks = f.ks, vs = f.vs;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            zero_scores(kb);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                const u32x4 w = f.k[kb * (D / 64) + c];
                score(widen8_plain(w[0], w[1]), kb, 2 * c);
                score(widen8_plain(w[2], w[3]), kb, 2 * c + 1);
            }
        }
        more_k();
        packed_softmax(ks, vs, j);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            const u32x4 w = f.v[c];
            value(widen8_plain(w[0], w[1]), 2 * c);
            value(widen8_plain(w[2], w[3]), 2 * c + 1);
        }
        more_v();
    };
    auto leave_packed = [&] {  // to fp16 rows: O in the values' own units
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
            for (int dt = 0; dt < NT; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e) O[dt][nr][e] = ldexpf(O[dt][nr][e], units[nr]);
            L[nr] = float4_t{0, 0, 0, 0};
            limit[nr] = M[nr] == -INFINITY ? M[nr] : M[nr] + GROW / sc[nr];
        }
    };

    // 32 fp16 rows from row j on, K and V at LDS offsets. Operand reads, half a
    // step's at a time: the next half is on its way while the matrix cores work on
    // this one.
    const half8_t ones = {(_Float16)1, (_Float16)1, (_Float16)1, (_Float16)1, (_Float16)1, (_Float16)1, (_Float16)1, (_Float16)1};
    half8_t ka[KS], kb[KS], va[NT / 2], vb[NT / 2];
    auto read_k = [&](half8_t (&f)[KS], int klds, int t) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) f[ks] = *reinterpret_cast<const half8_t *>(smem + klds + kaddr[ks] + t * 16 * T::RB);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto read_v = [&](half8_t (&f)[NT / 2], int vlds, int part) {
#pragma unroll
        for (int t = 0; t < NT / 2; ++t) {
            const int dt = part * (NT / 2) + t;
            const half4_t low = read_transposed(smem + vlds + (vaddr ^ (dt * 32)));
            const half4_t high = read_transposed(smem + vlds + (vaddr ^ (dt * 32)) + 16 * T::RB);
            f[t] = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto scores = [&](const half8_t (&f)[KS], int t) {
        zero_scores(t);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) score(f[ks], t, ks);
    };
    auto values = [&](const half8_t (&f)[NT / 2], int part) {
#pragma unroll
        for (int t = 0; t < NT / 2; ++t) value(f[t], part * (NT / 2) + t);
    };
    auto rows_softmax = [&](int j) {
        const bool in = inside(s.packed + j);
        if (j + 32 > clear || !in) {  // some positions are not for every row
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                uint32_t w;
                if (a.mask) {
                    w = mask_window(a.mask + (size_t)(s.start + tok[nr]) * a.words, a.words, s.n, j - s.len);
                } else {
                    const int left = s.len + tok[nr] + 1 - j;
                    w = left >= 32 ? 0xFFFFFFFFu : left > 0 ? (1u << left) - 1 : 0;
                }
                if (total - j < 32) w &= total > j ? (1u << (total - j)) - 1 : 0;
                if (!in) {
                    uint32_t win = window_bits(nr, s.packed + j);
                    if (a.mask && j + 32 > s.len) win |= j >= s.len ? 0xFFFFFFFFu : 0xFFFFFFFFu << (s.len - j);  // (the step's own rows)
                    w &= win;
                }
                masked(nr, w);
            }
        } else {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) any[nr] = true;
        }
        softmax(1.0f, 1.0f, kRows);
    };
    auto sums = [&] {
#pragma unroll
        for (int q = NQ - 1; q >= 0; --q)
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) L[nr] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, P[nr][q], L[nr], 0, 0, 0);
    };

    if constexpr (SHARED) {
        int lds = 0;
        if constexpr (PACKED) {
            if (u0 < tp) {
                fetch_tile(turns.at(u0));
                fetch_scales(turns.at(u0));
                widen_tile(0);
                if (u0 + 1 < tp) fetch_tile(turns.at(u0 + 1));
            }
        }
        if (u0 >= tp && u0 < u1) load_tile(turns.at(u0), 0);
        queries();
        clear_rows();
        if constexpr (PACKED) {
            for (int t = u0; t < tp; ++t, lds = T::STAGE - lds) {
                const int u = turns.at(t);
                lds_barrier();  // the tile is there, and every wave is done with the other buffer
                if (t + 1 < tp) {
                    widen_tile(T::STAGE - lds);
                    if (t + 2 < tp) fetch_tile(turns.at(t + 2));
                } else if (t + 1 < u1) {
                    load_tile(turns.at(t + 1), T::STAGE - lds);
                }
                const bool two = u * 2 + 1 < held;  // (else the second block's bytes are zeros, and no row sees it)
                const float k0 = scale[0], k1 = two ? scale[1] : 1.0f, v0 = scale[2], v1 = scale[3];
                if (t + 1 < tp) fetch_scales(turns.at(t + 1));
                const unsigned char *at = smem + lds + lane * 16;
                auto keys = [&](half8_t (&f)[KS], const unsigned char *p, int kb) {
#pragma unroll
                    for (int i = 0; i < KS; ++i) f[i] = *reinterpret_cast<const half8_t *>(p + (kb * KS + i) * 1024);
                    __builtin_amdgcn_sched_barrier(0);
                };
                auto vals = [&](half8_t (&f)[NT / 2], const unsigned char *p, int part) {
#pragma unroll
                    for (int i = 0; i < NT / 2; ++i) f[i] = *reinterpret_cast<const half8_t *>(p + 64 * T::RB + (part * (NT / 2) + i) * 1024);
                    __builtin_amdgcn_sched_barrier(0);
                };
                // (us a call when all rows shared their units, scales loaded where they are needed
                // and a loop over the blocks: trees in fp32 69, a prompt in fp16 100. Scales a turn
                // ahead: 61 and 101; both blocks in a row, the second's keys read under the first's
                // last products: 68 and 94.)
                if constexpr (HALF) {
                    keys(ka, at, 0);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const unsigned char *p = at + k * 64 * D;
                        keys(kb, p, 1);
                        scores(ka, 0);
                        scores(kb, 1);
                        vals(va, p, 0);
                        packed_softmax(k ? k1 : k0, k ? v1 : v0, (u * 2 + k) * BLOCK, k == 0 || two);
                        vals(vb, p, 1);
                        values(va, 0);
                        if (k == 0) keys(ka, p + 64 * D, 0);
                        values(vb, 1);
                    }
                } else {
                    const int end = two ? 2 : 1;
#pragma unroll 1
                    for (int k = 0; k < end; ++k) {
                        const unsigned char *p = at + k * 64 * D;
                        const float ks = k ? k1 : k0, vs = k ? v1 : v0;
                        keys(ka, p, 0);
                        keys(kb, p, 1);
                        scores(ka, 0);
                        scores(kb, 1);
                        vals(va, p, 0);
                        packed_softmax(ks, vs, (u * 2 + k) * BLOCK, true);
                        vals(vb, p, 1);
                        values(va, 0);
                        values(vb, 1);
                    }
                }
            }
            leave_packed();
        }
        for (int t = tp; t < u1; ++t, lds = T::STAGE - lds) {
            const int j = (turns.at(t) - turns.packed) * UNIT;
            dma_wait<0>();
            lds_barrier();
            if (t + 1 < u1) load_tile(turns.at(t + 1), T::STAGE - lds);
            read_k(ka, lds, 0);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int klds = lds + k * 32 * T::RB, vlds = klds + 64 * T::RB;
                read_k(kb, klds, 1);
                scores(ka, 0);
                scores(kb, 1);
                read_v(va, vlds, 0);
                rows_softmax(j + k * 32);
                read_v(vb, vlds, 1);
                sums();
                values(va, 0);
                if (k == 0) read_k(ka, klds + 32 * T::RB, 0);
                values(vb, 1);
            }
        }
    } else {
        const int mine = wid * T::NS * T::STAGE;  // this wave's ring
        // fp16 rows, a wave's 32 of each turn
        int ahead = tp;  // the next turn to load
        auto load_turn = [&](int slot) {
            const int first = ahead < u1 ? (turns.at(ahead) - turns.packed) * UNIT + wid * 32 : 0;
            const size_t at = head_at + (size_t)first * a.row_stride;
            return std::pair<size_t, int>{at, ahead < u1 ? total - first : 0};
        };
#pragma unroll
        for (int k = 0; k < T::NS; ++k) {
            const auto [at, left] = load_turn(k);
            load_rows(a.k_cache + at, left, mine + k * T::STAGE);
            load_rows(a.v_cache + at, left, mine + k * T::STAGE + 32 * T::RB);
            ++ahead;
        }
        if constexpr (PACKED) {
            PackedBlock<D> f[2];  // on their way
            auto block_of = [&](int t) {  // this wave's of turn t; past the last: -1
                if (t >= tp) return -1;
                const int blk = turns.at(t) * WAVES + wid;
                return blk < held ? blk : -1;
            };
            auto fetch = [&](PackedBlock<D> &to, int t, bool keys) {
                const int blk = block_of(t);
                const bool there = blk >= 0;
                const size_t at = head_blocks + (there ? blk : 0);
                const int bytes = there ? BLOCK * D : 0;
                const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>((keys ? a.k8 : a.v8) + at * (BLOCK * D)), 0, bytes, 0x00020000);
                if (keys) {
#pragma unroll
                    for (int c = 0; c < 2 * D / 64; ++c) to.k[c] = __builtin_amdgcn_raw_buffer_load_b128(r, lane * 16 + c * 1024, 0, NT_BIT);
                    to.ks = a.k_scale[at];
                    to.vs = a.v_scale[at];
                } else {
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) to.v[c] = __builtin_amdgcn_raw_buffer_load_b128(r, lane * 16 + c * 1024, 0, NT_BIT);
                }
            };
            if (u0 < tp) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    fetch(f[k], u0 + k, true);
                    fetch(f[k], u0 + k, false);
                }
            }
            queries();
            clear_rows();
            auto step = [&](PackedBlock<D> &now, int t) {
                const int blk = block_of(t);
                if (blk < 0) {
                    fetch(now, t + 2, true);
                    fetch(now, t + 2, false);
                    return;
                }
                packed_step(now, blk * BLOCK, [&] { fetch(now, t + 2, true); }, [&] { fetch(now, t + 2, false); });
            };
            for (int t = u0; t < tp; t += 2) {
                step(f[0], t);
                if (t + 1 < tp) step(f[1], t + 1);
            }
            leave_packed();
        } else {
            queries();
            clear_rows();
        }
        // loads younger than the K or V part waited for
        constexpr int YOUNGER = NL + (T::NS - 1) * 2 * NL;
        int lds = mine;
        for (int t = tp; t < u1; ++t) {
            const int j = (turns.at(t) - turns.packed) * UNIT + wid * 32;
            const auto [at, left] = load_turn(0);
            dma_wait<YOUNGER>();
            read_k(ka, lds, 0);
            read_k(kb, lds, 1);
            scores(ka, 0);
            scores(kb, 1);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the slot is refilled
            load_rows(a.k_cache + at, left, lds);
            rows_softmax(j);
            dma_wait<YOUNGER>();
            read_v(va, lds + 32 * T::RB, 0);
            read_v(vb, lds + 32 * T::RB, 1);
            sums();
            values(va, 0);
            values(vb, 1);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            load_rows(a.v_cache + at, left, lds + 32 * T::RB);
            ++ahead;
            lds += T::STAGE;
            if (lds == mine + T::NS * T::STAGE) lds = mine;
        }
    }
    dma_wait<0>();
    lds_barrier();  // the ring is free

    // ---- results: whole rows, what is not finite again
    int *flag = reinterpret_cast<int *>(smem + T::FLAG);
    for (int e = tid; e <= T::BM; e += THREADS) flag[e] = 0;
    lds_barrier();
    bool redo[NR];
    float l[NR];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        l[nr] = L[nr][0];
        if constexpr (PACKED) l[nr] += column_sum(lsum[nr]);
        float z = l[nr] * 0.0f;
#pragma unroll
        for (int dt = 0; dt < NT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) z = fmaf(O[dt][nr][e], 0.0f, z);
        // (the largest score's p is 2^BASE at least if its product with sc rounds to within a bit)
        redo[nr] = live[nr] && (z != 0.0f || (any[nr] && !(l[nr] >= 32.0f)));
        if (redo[nr]) flag[row[nr] - r0] = flag[T::BM] = 1;
    }
    auto emit = [&](int t, int hd, int d, float4_t o, float m, float sum) {
        const int64_t r = s.start + t;
        if (a.splits == 1) {
            const float inv = m == -INFINITY ? 0.0f : 1.0f / sum;
            o *= inv;
            const int64_t at = r * a.ldo + (int64_t)hd * D + d;
            if constexpr (HALF)
                *reinterpret_cast<half4_bits *>(static_cast<uint16_t *>(a.out) + at) = half4_bits{f2h(o[0]), f2h(o[1]), f2h(o[2]), f2h(o[3])};
            else
                *reinterpret_cast<float4_any *>(static_cast<float *>(a.out) + at) = o;
        } else {
            const int64_t part = (r * a.heads + hd) * a.splits + split;
            *reinterpret_cast<float4_t *>(a.part_o + part * D + d) = o;
            if (d == 0) {
                a.part_ml[part * 2] = m;
                a.part_ml[part * 2 + 1] = sum;
            }
        }
    };
    if constexpr (SHARED) {
        lds_barrier();  // one lane alone may have set a row's flag, and its other three read it
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
            if (live[nr] && !flag[row[nr] - r0])
#pragma unroll
                for (int dt = 0; dt < NT; ++dt)
                    emit(tok[nr], head[nr], dt * 16 + 4 * g, O[dt][nr], M[nr] == -INFINITY ? -INFINITY : -bias[nr], l[nr]);
        lds_barrier();
    } else {
        float *join = reinterpret_cast<float *>(smem);
        float *ml = reinterpret_cast<float *>(smem + T::ML);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const int at = wid * T::BM + nr * 16 + i;
#pragma unroll
            for (int dt = 0; dt < NT; ++dt) *reinterpret_cast<float4_t *>(join + at * T::OS + dt * 16 + 4 * g) = O[dt][nr];
            if (g == 0) {
                ml[at * 2] = M[nr] == -INFINITY ? -INFINITY : -bias[nr];
                ml[at * 2 + 1] = l[nr];
            }
        }
        lds_barrier();
        for (int e = tid; e < T::BM * (D / 4); e += THREADS) {
            const int k = e / (D / 4), d = e % (D / 4) * 4, r = r0 + k;
            if (r >= nrows || flag[k]) continue;
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) m = fmaxf(m, ml[(w * T::BM + k) * 2]);
            float4_t o = {0, 0, 0, 0};
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float mw = ml[(w * T::BM + k) * 2];
                const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - m);
                sum = fmaf(ml[(w * T::BM + k) * 2 + 1], f, sum);
                o += *reinterpret_cast<const float4_t *>(join + (w * T::BM + k) * T::OS + d) * f;
            }
            const int t = r / group;
            emit(t, h * group + r - t * group, d, o, m, sum);
        }
        lds_barrier();
    }
    if (!flag[T::BM]) return;
    LongScratch &sh = *reinterpret_cast<LongScratch *>(smem);
    for (int k = 0; k < T::BM; ++k) {
        if (!flag[k]) continue;  // (uniform)
        const int t = (r0 + k) / group, hd = h * group + r0 + k - t * group;
        float o, m, sum;
        long_row<D, HALF, UNIT>(a, s, b, t, hd, turns, u0, u1, sh, o, m, sum);
        if (tid < D) {
            const int64_t r = s.start + t;
            if (a.splits == 1) {
                put<HALF>(a.out, r * a.ldo + (int64_t)hd * D + tid, m == -INFINITY ? 0.0f : o / sum);
            } else {
                const int64_t part = (r * a.heads + hd) * a.splits + split;
                a.part_o[part * D + tid] = o;
                if (tid == 0) {
                    a.part_ml[part * 2] = m;
                    a.part_ml[part * 2 + 1] = sum;
                }
            }
        }
    }
}

// Joins a row's splits: one wave a (row, query head), four values a lane, 64 /
// (D / 4) splits side by side and four such loads under way.
template <int D, bool HALF>
__global__ __launch_bounds__(THREADS) void long_join_kernel(const int32_t *row_start_p, const int32_t *cache_len_p, const float *part_ml_p,
                                                            const float *part_o_p, int heads_p, int splits_p, int rows_p, int max_rows_p,
                                                            LongAttnArgs args) {
    LongAttnArgs a = args;
    a.row_start = row_start_p;
    a.cache_len = cache_len_p;
    a.heads = heads_p;
    a.splits = splits_p;
    a.rows = rows_p;
    a.max_rows = max_rows_p;
    constexpr int LANES = D / 4, SIDE = 64 / LANES;
    const int lane = threadIdx.x & 63, d = lane % LANES * 4, side = lane / LANES;
    const int x = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hd = x % a.heads, bt = x / a.heads, t = bt % a.max_rows, b = bt / a.max_rows;
    if (b >= a.batch) return;
    const LongSeq s = long_sequence(a, b);
    if (t >= s.n) return;
    const int64_t r = s.start + t, part = (r * a.heads + hd) * a.splits;
    float4_t o = {0, 0, 0, 0};
    if (s.ok) {
        float m = -INFINITY, lw = 0.0f;
        if (lane < a.splits) {
            m = part_ml_p[(part + lane) * 2];
            lw = part_ml_p[(part + lane) * 2 + 1];
        }
        const float *p = part_o_p + part * D + d;
        float4_t v[4];
        auto load = [&](int k) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int at = k + u * SIDE + side;
                v[u] = at < a.splits ? *reinterpret_cast<const float4_t *>(p + (size_t)at * D) : float4_t{0, 0, 0, 0};
            }
        };
        load(0);
        const float top = column_max(row16_max(m));
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);  // (nothing seen there: o = l = 0)
        lw *= f;
        lw += dpp_f(lw, dpp_xor1);
        lw += dpp_f(lw, dpp_xor2);
        lw += dpp_f(lw, dpp_half_mirror);
        lw += dpp_f(lw, dpp_mirror);
        lw = column_sum(lw);
        for (int k = 0; k < a.splits; k += 4 * SIDE) {
            if (k) load(k);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float fk = 0.0f;
#pragma unroll
                for (int z = 0; z < SIDE; ++z) {
                    const float fz = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), min(k + u * SIDE + z, 63)));
                    fk = side == z ? fz : fk;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(v[u][e], fk, o[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (SIDE == 4) {
                o[e] = column_sum(o[e]);
            } else {
                auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(o[e]), __float_as_uint(o[e]), false, false);
                o[e] = __uint_as_float(y[0]) + __uint_as_float(y[1]);
            }
        }
        const float inv = top == -INFINITY ? 0.0f : 1.0f / lw;
        o *= inv;
    } else {
        const float nan = __builtin_nanf("");
        o = float4_t{nan, nan, nan, nan};
    }
    if (side) return;
    const int64_t at = r * a.ldo + (int64_t)hd * D + d;
    if constexpr (HALF)
        *reinterpret_cast<half4_bits *>(static_cast<uint16_t *>(a.out) + at) = half4_bits{f2h(o[0]), f2h(o[1]), f2h(o[2]), f2h(o[3])};
    else
        *reinterpret_cast<float4_any *>(static_cast<float *>(a.out) + at) = o;
}

// Rows of a workgroup and splits.
//
// Over packed blocks up to 64 rows of a kv head go in tiles of 16, each of which
// reads and widens for itself what its neighbours read too (out of the caches):
// two workgroups fit a CU, where 32 rows' registers leave room for one. us
// (16 / 8 heads of 128, fp32, lengths from half to all, each at its best split):
// 24 trees of 12 rows over 8000 75 in tiles of 16, 103 with 32 rows a workgroup,
// 119 in shared tiles of 64; of 20 rows 94 and 131 shared; of 32 139 and 140; of
// 40 146 and 146, 6 of 40 53 and 51.
// As many splits as fill whole rounds of 512 workgroups to nine tenths (the rule's
// choice first): one token of 4 sequences of 16000 25.2 at 15, 24.9 at 16, 26.9 at
// 8; of 8 of 12000 31.7 at 8, 34.9 at 4; of 12 47.0 at 5, 55.4 at 2; of 24 84.7 at
// 5, 90.6 at 2, 83.8 at 8; of 40 of 3000 43.7 at 3, 44.6 at 1. Below 512 positions
// a split one round of 256: one token of 8 of 3000 16.9 at 4, 17.8 at 8; of 2 of
// 8000 14.9 at 16, 16.5 at 32; 6 trees of 20 over 1000 15.1 at 1, 16.2 at 4. (All of
// one length: 32 of 8192 90.8 at 2, 87.6 at 1, which the host cannot tell apart.)
//
// Else as tree_attention_plan says, whose kernels these are.
TreePlan long_attention_plan(int64_t rows, int heads, int kv_heads, int batch, int max_rows, int max_len, int head_dim, bool half,
                             bool chain, bool packed) {
    const int64_t kv_rows = (int64_t)max_rows * (heads / kv_heads), tiles = (kv_rows + 15) / 16;
    if (!packed || tiles > 4) return tree_attention_plan(rows, heads, kv_heads, batch, max_rows, max_len, head_dim, half, chain);
    const int64_t base = (int64_t)batch * kv_heads * tiles, most = ((int64_t)max_len + 127) / 128;
    if (base < 1) return {16, 1};
    int64_t k = 256 / base;
    for (int i = 1; i <= 16 && base <= 4096; ++i) {
        const int64_t blocks = base * i, rounds = (blocks + 511) / 512;
        if (blocks * 10 < rounds * 512 * 9) continue;
        if (max_len / i >= 512) k = i;
        break;
    }
    k = k < most ? k : most;
    return {16, (int)(k < 1 ? 1 : k < kLongSplits ? k : kLongSplits)};
}

template <int D, bool HALF, int NR, bool SHARED, bool PACKED, bool ONCE>
static hipError_t launch_tile(const LongAttnArgs &a, int tiles, hipStream_t st) {
    using T = LongTile<D, NR, SHARED, PACKED>;
    const unsigned grid = (unsigned)tiles * a.splits * a.batch * a.kv_heads;
    const hipError_t e = allow_lds<&long_attention_kernel<D, HALF, NR, SHARED, PACKED, ONCE>>(T::LDS);
    if (e != hipSuccess) return e;
    long_attention_kernel<D, HALF, NR, SHARED, PACKED, ONCE><<<grid, THREADS, T::LDS, st>>>(
        a.row_start, a.cache_len, a.q, a.packed_len, a.kv_heads, a.heads, a.splits, a.rows, a.max_rows, a.max_seq, tiles, grid <= 512, a);
    return hipGetLastError();
}

template <int D, bool HALF, bool PACKED> static hipError_t launch_d(const LongAttnArgs &a, int bm, hipStream_t st) {
    const int tiles = (int)(((int64_t)a.max_rows * (a.heads / a.kv_heads) + bm - 1) / bm);
    // Keys and values that one workgroup reads go past the caches: always with up to
    // 32 rows in one tile (us past the caches and through them, packed, three calls'
    // blocks in turn: one token of 16 sequences of 8000 41.9 and 47.0, of 8 27.0 and
    // 29.3, of one 13.4 and 14.2; one of 1024 13.1 both; but trees of 32 rows in four
    // tiles 141 and 132), of shared tiles where together they are more than the caches
    // keep.
    const bool one = tiles == 1, once = one && (double)a.batch * a.kv_heads * a.max_len * D * (PACKED ? 2 : 4) > 192e6;
    hipError_t e;
    if (PACKED && bm == 16 && !one) e = launch_tile<D, HALF, 1, false, true, false>(a, tiles, st);
    else if (bm == 16) e = launch_tile<D, HALF, 1, false, PACKED, true>(a, tiles, st);
    else if (!PACKED && bm == 32) e = launch_tile<D, HALF, 2, false, false, true>(a, tiles, st);
    else if (bm == 64) e = once ? launch_tile<D, HALF, 1, true, PACKED, true>(a, tiles, st) : launch_tile<D, HALF, 1, true, PACKED, false>(a, tiles, st);
    else e = once ? launch_tile<D, HALF, 2, true, PACKED, true>(a, tiles, st) : launch_tile<D, HALF, 2, true, PACKED, false>(a, tiles, st);
    if (e != hipSuccess || a.splits == 1) return e;
    const unsigned waves = (unsigned)a.batch * a.max_rows * a.heads;
    long_join_kernel<D, HALF><<<(waves + WAVES - 1) / WAVES, THREADS, 0, st>>>(a.row_start, a.cache_len, a.part_ml, a.part_o, a.heads,
                                                                             a.splits, a.rows, a.max_rows, a);
    return hipGetLastError();
}

hipError_t launch_long_attention(const LongAttnArgs &a, int head_dim, bool half, int block_rows, hipStream_t st) {
    const bool packed = a.packed_len != nullptr;
    auto go = [&](auto d, auto h) {
        return packed ? launch_d<d, h, true>(a, block_rows, st) : launch_d<d, h, false>(a, block_rows, st);
    };
    using std::integral_constant;
    if (head_dim == 128)
        return half ? go(integral_constant<int, 128>{}, std::true_type{}) : go(integral_constant<int, 128>{}, std::false_type{});
    return half ? go(integral_constant<int, 64>{}, std::true_type{}) : go(integral_constant<int, 64>{}, std::false_type{});
}

}  // namespace q3vl
