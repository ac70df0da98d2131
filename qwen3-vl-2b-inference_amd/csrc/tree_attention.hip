// tree_attention.hip -- attention of several rows a sequence over its cache:
// one token of each sequence of a batch, a prompt's chunk, or a tree of
// drafted tokens. gfx950.
#include "q3vl_device.hpp"
#include "q3vl_kernels.hpp"
#include "q3vl_mfma.hpp"

namespace q3vl {

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;

// What a block knows of its sequence.
struct Seq {
    int start, n;  // its rows of q
    int len;       // cached positions before them
    bool ok;       // cached positions and rows fit the cache
};
__device__ __forceinline__ Seq sequence(const TreeAttnArgs &a, int b) {
    Seq s;
    s.start = min(max(a.row_start[b], 0), a.rows);
    s.n = min(max(a.row_start[b + 1], s.start), a.rows) - s.start;
    s.len = a.cache_len[b];
    s.ok = s.len >= 0 && (int64_t)s.len + s.n <= a.max_seq;
    return s;
}

// Whether row t of the sequence sees position j of its cache (j < len + n).
__device__ __forceinline__ bool sees(const TreeAttnArgs &a, const Seq &s, int t, int j) {
    const int i = j - s.len;
    if (i < 0) return true;
    if (!a.mask) return i <= t;
    return i < 64 * a.words && (a.mask[(size_t)(s.start + t) * a.words + (i >> 6)] >> (i & 63) & 1);
}

struct RowScratch {
    float q[128];
    float p[THREADS];
    uint64_t seen[WAVES];
    float red[WAVES];
};

// One row and head over positions [j0, j1), plainly and in fp32, by a whole
// block: o (threads 0 .. D-1) = sum p v, p = 2^(s - m), l = sum p, with s the
// scores times log2 e. m is -inf where nothing is seen (then o = l = 0), else
// at least -FLT_MAX. Products of what the row does not see are never formed.
template <int D, bool HALF>
__device__ void row_attention(const TreeAttnArgs &a, const Seq &s, int b, int t, int head, int j0, int j1,
                              RowScratch &sh, float &o, float &m, float &l) {
    const int tid = threadIdx.x, lane = tid & 63;
    const size_t base = (size_t)b * a.seq_stride + (size_t)(head / (a.heads / a.kv_heads)) * a.head_stride;
    const int64_t qat = (int64_t)(s.start + t) * a.ldq + (int64_t)head * D;
    __syncthreads();
    if (tid < D) sh.q[tid] = HALF ? h2f(static_cast<const uint16_t *>(a.q)[qat + tid]) : static_cast<const float *>(a.q)[qat + tid];
    o = l = 0.0f;
    m = -INFINITY;
    for (int c = j0; c < j1; c += THREADS) {
        const int j = c + tid;
        const bool seen = j < j1 && sees(a, s, t, j);
        float sc = -INFINITY;
        __syncthreads();  // the scratch of the last chunk is read
        if (seen) {
            const uint16_t *k = a.k_cache + base + (size_t)j * a.row_stride;
            float acc = 0.0f;
            for (int d = 0; d < D; ++d) acc = fmaf(sh.q[d], h2f(k[d]), acc);
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
            for (int i = 0; i < min(THREADS, j1 - c); ++i)
                if (sh.seen[i >> 6] >> (i & 63) & 1)
                    o = fmaf(sh.p[i], h2f(a.v_cache[base + (size_t)(c + i) * a.row_stride + tid]), o);
    }
}

template <bool HALF> __device__ __forceinline__ void put(void *out, int64_t at, float v) {
    if (HALF) static_cast<uint16_t *>(out)[at] = f2h(v);
    else static_cast<float *>(out)[at] = v;
}

}  // namespace

// ------------------------------------------------------------ the kernel
// Scores transposed, S^T = K Q^T, by v_mfma_f32_16x16x32_f16: a lane then holds
// four keys of one query row (column i = lane & 15, keys 4 g + e with g = lane
// >> 4), so a row's running maximum, its bias and its sum stay in the lane, and
// only the maximum of a step crosses lanes. The same registers, two 16-key
// tiles side by side, are the B operand of O^T += V^T P^T: operand slot (g, e)
// holds key 4 g + e of the first tile, slot (g, 4 + e) of the second, and V^T is
// read in that order by the transposing LDS read. O^T's column is the same
// query row, so its rescaling needs no exchange either.
//
// Query row r of a (sequence, kv head): token r / group, head r % group of the
// group of query heads that share the kv head.
//
// K and V go to LDS by loads with an LDS destination (no registers, any number
// in flight), 16-byte pieces swizzled by the row so that both reads spread over
// the banks. Rows past the end read as zeros by the buffer's bounds.
//
// Two forms. Few rows (at most 32 of a kv head's): each wave walks its own 32
// keys of every 128 with all rows, in a private ring of two stages, no barrier;
// the four waves' results are joined in LDS at the end. Bound by the cache's
// reads: one token each of 24 sequences of up to 6000, 67.1 us, 6.5 TB/s, the
// rate of a plain read here. Many rows: a wave has 16 or 32 rows of its own, the
// block shares 64-key tiles in two buffers, one barrier a tile. Two waves a SIMD,
// each a chain of scores, softmax and values: three trees of up to 61 rows over
// 16000 in fp32 55.2 us, 2000 rows behind 1200 in fp16 51.8. Of the shader
// engines' busy cycles the matrix cores work in 45 and 35 of 100 and other vector
// instructions run in 31 and 27, a SIMD's mean; even laid end to end they leave 24
// and 38 to waits (for the chain's own results, LDS reads, the next tile and its
// barrier) and to SIMDs without a block.
//
// fp32 queries are two fp16 terms, hi + lo, relative to the row's largest value
// (a power of two, undone in the score's factor sc), and so are their
// probabilities; products of fp16 are exact in fp32, so the scores keep 2^-21 of
// sum |q k|. fp16 queries and their probabilities are one term each: half a
// step of fp16 in each p, as the output's own rounding. (With two terms of p the
// 2000 rows' error against 64 bits is the output's rounding alone, 2.1e-4 for
// 2.7e-4 of its norm, at 68.6 us a call for 51.4; few rows, bound by reads, would
// pay nothing.)
//
// p is held as 2^(s sc + bias), bias = BASE - M sc, M a row's largest raw score
// when the bias was last set: a score that passes it by up to GROW stays under
// fp16's 2^16, so the accumulators are rescaled in the first step and seldom
// after (with every new maximum, some row of 32 had one in most steps: 267 VALU
// instructions a step). 2^-20 of the largest p is still a normal number; no p
// is held finer than 2^-31 of it, of two terms either, and below that it counts
// for nothing (BASE 12 and GROW 3 would hold 2^-37: the tree's case below 62.8
// us a call for 61.2, the prompt's 52.3 for 51.4). A row's results are its O and
// l with weights 2^(-bias). l is summed by the matrix cores too, as V's column
// of ones: a product a step instead of an addition a score.
//
// What no row sees never enters: rows past the end are zeros, scores of unseen
// keys are replaced by -inf before the maximum. An unseen V row of another
// row's draft can still hold an infinity or NaN, and 0 times it is NaN: a row
// whose O or l is not finite is done again by row_attention; so is one whose
// scores pass 2^23, where the rounding of M sc alone moves p by bits. Such rows
// go one after the other through their block's part of the cache, and a NaN in
// a draft that no row sees brings every row of the sequence there: 8 drafts
// over 1000 in fp32 370 us for 10.3, three trees of up to 61 over 16000 17.2 ms
// for 57 us.
template <int D, int NR, bool SHARED> struct Tile {
    static constexpr int RB = 2 * D;             // bytes of a cached row
    static constexpr int RI = D / 32;            // loads of 1 KiB for 16 rows
    static constexpr int NS = SHARED ? 2 : 256 / D;
    static constexpr int STAGE = (SHARED ? 64 : 32) * RB * 2;  // K, then V
    static constexpr int RING = (SHARED ? 1 : WAVES) * NS * STAGE;
    static constexpr int BM = 16 * NR * (SHARED ? WAVES : 1);  // query rows of a block
    static constexpr int OS = D + 4;             // floats of a joined row (spread over the banks)
    static constexpr int JOIN = SHARED ? 0 : WAVES * BM * OS * 4;
    static constexpr int ML = RING > JOIN ? RING : JOIN;       // (M, l) of each wave's rows
    static constexpr int FLAG = ML + (SHARED ? 0 : WAVES * BM * 8);
    static constexpr int LDS = FLAG + (BM + 1) * 4;
    static constexpr int UNIT = SHARED ? 64 : 32 * WAVES;      // keys of a turn
    static_assert(LDS <= 160 * 1024 && sizeof(RowScratch) <= (size_t)RING, "LDS");
};

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

// ONCE: no other block reads this one's keys and values; they go past the caches.
// (What the first loads need comes as plain leading arguments, which arrive in
// registers; the rest is read from the struct beside those loads.)
template <int D, bool HALF, int NR, bool SHARED, bool ONCE>
__global__ __launch_bounds__(THREADS, SHARED ? 2 : 1) void tree_attention_kernel(
    const int32_t *row_start_p, const int32_t *cache_len_p, const void *q_p, int kv_heads_p, int heads_p, int splits_p, int rows_p,
    int max_rows_p, int max_seq_p, int tiles, int paired, TreeAttnArgs args) {
    TreeAttnArgs a = args;
    a.row_start = row_start_p;
    a.cache_len = cache_len_p;
    a.q = q_p;
    a.kv_heads = kv_heads_p;
    a.heads = heads_p;
    a.splits = splits_p;
    a.rows = rows_p;
    a.max_rows = max_rows_p;
    a.max_seq = max_seq_p;
    using T = Tile<D, NR, SHARED>;
    constexpr int KS = D / 32, NT = D / 16, NQ = HALF ? 1 : 2;
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
    // a chain's last rows see most: they go first, and where every block has a
    // place at once (two a CU, the second half of them beside the first), the
    // second half goes the other way round
    const int tile = paired && 2 * x >= tiles ? x - (tiles + 1) / 2 : tiles - 1 - x;
    const Seq s = sequence(a, b);
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

    // ---- this block's positions: units of T::UNIT keys, a chain's up to the
    // last one that the tile's rows see
    const int last_tok = min((r0 + T::BM - 1) / group, n - 1);
    const int total = s.len + (a.mask ? s.n : last_tok + 1);
    const int units = (total + T::UNIT - 1) / T::UNIT;
    const int u0 = (int)((int64_t)units * split / a.splits), u1 = (int)((int64_t)units * (split + 1) / a.splits);
    const int j0 = u0 * T::UNIT, j1 = min(u1 * T::UNIT, total);

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

    // ---- loads: lane's place in 16 rows of the cache, and of LDS
    const size_t head_at = (size_t)b * a.seq_stride + (size_t)h * a.head_stride;
    const int rsb = (int)(a.row_stride * 2);
    constexpr int NL = (SHARED ? 1 : 2) * T::RI;  // loads of a K or V part
    int voff[NL];
#pragma unroll
    for (int t = 0; t < NL; ++t) {
        const int r = (t * 64 + lane) / (D / 8), c = lane % (D / 8);
        voff[t] = (r + (SHARED ? wid * 16 : 0)) * rsb + (c ^ swizzle<D>(r)) * 16;
    }
    // rows from p on, `left` of them there: 32 to this wave's own stage, or its
    // 16 of a block's 64
    auto load = [&](const uint16_t *p, int left, int lds) {
        left = min(left, SHARED ? 64 : 32);
        const rsrc_t r = make_rsrc(p, left > 0 ? (uint32_t)((left - 1) * rsb + 2 * D) : 0);
#pragma unroll
        for (int t = 0; t < NL; ++t) {
            const int at = lds + ((SHARED ? wid * NL : 0) + t) * 1024;
            if constexpr (ONCE) dma16_nt(r, voff[t], 0, at);
            else dma16(r, voff[t], 0, at);
        }
    };
    const size_t first_at = head_at + (size_t)(j0 + (SHARED ? 0 : wid * 32)) * a.row_stride, turn = (size_t)T::UNIT * a.row_stride;
    const uint16_t *kp = a.k_cache + first_at, *vp = a.v_cache + first_at;  // of the next loads
    auto load_tile = [&](int u) {  // (SHARED)
        const int lds = (u & 1) * T::STAGE;
        load(kp, j1 - u * 64, lds);
        load(vp, j1 - u * 64, lds + 64 * T::RB);
        kp += turn;
        vp += turn;
    };
    const int mine = wid * T::NS * T::STAGE;  // (else: this wave's ring,
    int left = j1 - j0 - wid * 32;            // positions from the next loads' first on)
    if (u0 < u1) {
        if constexpr (SHARED) {
            load_tile(u0);
        } else {
#pragma unroll
            for (int k = 0; k < T::NS; ++k) {
                load(kp, left, mine + k * T::STAGE);
                load(vp, left, mine + k * T::STAGE + 32 * T::RB);
                kp += turn;
                vp += turn;
                left -= T::UNIT;
            }
        }
    }

    // ---- operand registers, the score's factor
    half8_t qf[NR][NQ][KS];
    float sc[NR];
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

    // positions below this are seen by all of this wave's rows
    const int first_tok = (r0 + (SHARED ? wid * 16 * NR : 0)) / group;
    const int clear = min(s.len + (a.mask ? 0 : min(first_tok, n - 1) + 1), j1);

    // ---- one step: 32 keys from position j, K and V rows at LDS offsets
    int kaddr[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kaddr[ks] = i * T::RB + ((ks * 4 + g) ^ swizzle<D>(i)) * 16;
    const int vr = 4 * g + (i >> 2);  // row of a 16-key tile this lane's transposing read starts from
    const int vaddr = vr * T::RB + (((i & 3) >> 1) ^ swizzle<D>(vr)) * 16 + (i & 1) * 8;
    const half8_t ones = {(_Float16)1, (_Float16)1, (_Float16)1, (_Float16)1, (_Float16)1, (_Float16)1, (_Float16)1, (_Float16)1};
    float M[NR], bias[NR], limit[NR], room[NR];  // limit: the score from which M is set anew, M + room
    float4_t O[NT][NR], L[NR];  // L: the sum of p, in each register and lane of the column
    bool any[NR];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        M[nr] = limit[nr] = -INFINITY;
        room[nr] = GROW / sc[nr];
        bias[nr] = 0.0f;
        any[nr] = false;
        L[nr] = float4_t{0, 0, 0, 0};
#pragma unroll
        for (int dt = 0; dt < NT; ++dt) O[dt][nr] = float4_t{0, 0, 0, 0};
    }
    float4_t S[2][NR];
    // operand reads, half a step's at a time: the next half is on its way while
    // the matrix cores work on this one (left to itself, the compiler reads one
    // operand ahead and each product pair waits out the LDS)
    auto read_k = [&](half8_t (&f)[KS], int klds, int kb) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) f[ks] = *reinterpret_cast<const half8_t *>(smem + klds + kaddr[ks] + kb * 16 * T::RB);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto read_v = [&](half8_t (&f)[NT / 2], int vlds, int part) {
#pragma unroll
        for (int t = 0; t < NT / 2; ++t) {
            const int dt = part * (NT / 2) + t;
            const half4_t lo = read_transposed(smem + vlds + (vaddr ^ (dt * 32)));
            const half4_t hi = read_transposed(smem + vlds + (vaddr ^ (dt * 32)) + 16 * T::RB);
            f[t] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto scores = [&](const half8_t (&f)[KS], int kb) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) S[kb][nr] = float4_t{0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int q = NQ - 1; q >= 0; --q)
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
                    S[kb][nr] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[ks], qf[nr][q][ks], S[kb][nr], 0, 0, 0);
    };
    half8_t P[NR][NQ];
    auto softmax = [&](int j) {
        if (j + 32 > clear) {  // some keys are not for every row
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                uint32_t w;
                if (a.mask) {
                    w = mask_window(a.mask + (size_t)(s.start + tok[nr]) * a.words, a.words, s.n, j - s.len);
                } else {
                    const int left = s.len + tok[nr] + 1 - j;
                    w = left >= 32 ? 0xFFFFFFFFu : left > 0 ? (1u << left) - 1 : 0;
                }
                if (j1 - j < 32) w &= j1 > j ? (1u << (j1 - j)) - 1 : 0;
                any[nr] = any[nr] || w;
                w >>= 4 * g;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(w >> (16 * kb + e) & 1)) S[kb][nr][e] = -INFINITY;
            }
        } else {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) any[nr] = true;
        }
        float top[NR];  // of this lane's keys
        bool grow = false;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            top[nr] = S[0][nr][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top[nr] = fmaxf(top[nr], S[e >> 2][nr][e & 3]);
            grow = grow || top[nr] > limit[nr];
        }
        if (__any(grow)) {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                const float m = fmaxf(M[nr], column_max(top[nr]));
                const float nb = m == -INFINITY ? 0.0f : fmaf(-m, sc[nr], BASE);
                const float f = M[nr] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(nb - bias[nr]);
                M[nr] = m;
                limit[nr] = m + room[nr];
                bias[nr] = nb;
                L[nr] *= f;
#pragma unroll
                for (int dt = 0; dt < NT; ++dt) O[dt][nr] *= f;
            }
        }
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(S[e >> 2][nr][e & 3], sc[nr], bias[nr]));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                P[nr][0][e] = (_Float16)p[e];
                if constexpr (!HALF) P[nr][1][e] = (_Float16)(p[e] - (float)P[nr][0][e]);
            }
        }
    };
    auto values = [&](const half8_t (&f)[NT / 2], int part) {
#pragma unroll
        for (int t = 0; t < NT / 2; ++t)
#pragma unroll
            for (int q = NQ - 1; q >= 0; --q)
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
                    O[part * (NT / 2) + t][nr] =
                        __builtin_amdgcn_mfma_f32_16x16x32_f16(f[t], P[nr][q], O[part * (NT / 2) + t][nr], 0, 0, 0);
    };
    auto sums = [&] {
#pragma unroll
        for (int q = NQ - 1; q >= 0; --q)
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) L[nr] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, P[nr][q], L[nr], 0, 0, 0);
    };
    half8_t ka[KS], kb[KS], va[NT / 2], vb[NT / 2];

    if constexpr (SHARED) {
        for (int u = u0; u < u1; ++u) {
            dma_wait<0>();
            lds_barrier();  // the tile is there, and every wave is done with the other buffer
            if (u + 1 < u1) load_tile(u + 1);
            const int lds = (u & 1) * T::STAGE;
            read_k(ka, lds, 0);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int klds = lds + k * 32 * T::RB, vlds = klds + 64 * T::RB;
                read_k(kb, klds, 1);
                scores(ka, 0);
                scores(kb, 1);
                read_v(va, vlds, 0);
                softmax(u * 64 + k * 32);
                read_v(vb, vlds, 1);
                sums();
                values(va, 0);
                if (k == 0) read_k(ka, klds + 32 * T::RB, 0);
                values(vb, 1);
            }
        }
    } else {
        // loads younger than the K or V part waited for
        constexpr int YOUNGER = NL + (T::NS - 1) * 2 * NL;
        int lds = mine;
        for (int u = u0, j = j0 + wid * 32; u < u1; ++u, j += T::UNIT) {
            dma_wait<YOUNGER>();
            read_k(ka, lds, 0);
            read_k(kb, lds, 1);
            scores(ka, 0);
            scores(kb, 1);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the slot is refilled
            load(kp, left, lds);
            softmax(j);
            dma_wait<YOUNGER>();
            read_v(va, lds + 32 * T::RB, 0);
            read_v(vb, lds + 32 * T::RB, 1);
            sums();
            values(va, 0);
            values(vb, 1);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            load(vp, left, lds + 32 * T::RB);
            kp += turn;
            vp += turn;
            left -= T::UNIT;
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
        float z = l[nr] * 0.0f;
#pragma unroll
        for (int dt = 0; dt < NT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) z = fmaf(O[dt][nr][e], 0.0f, z);
        // (the largest score's p is 2^BASE at least if its product with sc rounds to within a bit)
        redo[nr] = live[nr] && (z != 0.0f || (any[nr] && !(l[nr] >= 32.0f)));
        if (redo[nr]) flag[row[nr] - r0] = flag[T::BM] = 1;
    }
    auto emit = [&](int t, int hd, int d, float4_t o, float m, float lsum) {
        const int64_t r = s.start + t;
        if (a.splits == 1) {
            const float inv = m == -INFINITY ? 0.0f : 1.0f / lsum;
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
                a.part_ml[part * 2 + 1] = lsum;
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
            float lsum = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float mw = ml[(w * T::BM + k) * 2];
                const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - m);
                lsum = fmaf(ml[(w * T::BM + k) * 2 + 1], f, lsum);
                o += *reinterpret_cast<const float4_t *>(join + (w * T::BM + k) * T::OS + d) * f;
            }
            const int t = r / group;
            emit(t, h * group + r - t * group, d, o, m, lsum);
        }
        lds_barrier();
    }
    if (!flag[T::BM]) return;
    RowScratch &sh = *reinterpret_cast<RowScratch *>(smem);
    for (int k = 0; k < T::BM; ++k) {
        if (!flag[k]) continue;  // (uniform)
        const int t = (r0 + k) / group, hd = h * group + r0 + k - t * group;
        float o, m, lsum;
        row_attention<D, HALF>(a, s, b, t, hd, j0, j1, sh, o, m, lsum);
        if (tid < D) {
            const int64_t r = s.start + t;
            if (a.splits == 1) {
                put<HALF>(a.out, r * a.ldo + (int64_t)hd * D + tid, m == -INFINITY ? 0.0f : o / lsum);
            } else {
                const int64_t part = (r * a.heads + hd) * a.splits + split;
                a.part_o[part * D + tid] = o;
                if (tid == 0) {
                    a.part_ml[part * 2] = m;
                    a.part_ml[part * 2 + 1] = lsum;
                }
            }
        }
    }
}

// Joins a row's splits: one wave a (row, query head), four values a lane, 64 /
// (D / 4) splits side by side and four such loads under way.
template <int D, bool HALF> __global__ __launch_bounds__(THREADS) void tree_join_kernel(const int32_t *row_start_p, const int32_t *cache_len_p,
                                                            const float *part_ml_p, const float *part_o_p, int heads_p,
                                                            int splits_p, int rows_p, int max_rows_p, int max_seq_p, int batch_p,
                                                            TreeAttnArgs args) {
    TreeAttnArgs a = args;
    a.row_start = row_start_p;
    a.cache_len = cache_len_p;
    a.heads = heads_p;
    a.splits = splits_p;
    a.rows = rows_p;
    a.max_rows = max_rows_p;
    a.max_seq = max_seq_p;
    a.batch = batch_p;
    constexpr int LANES = D / 4, SIDE = 64 / LANES;
    const int lane = threadIdx.x & 63, d = lane % LANES * 4, side = lane / LANES;
    const int x = blockIdx.x * WAVES + (threadIdx.x >> 6);
    const int hd = x % a.heads, bt = x / a.heads, t = bt % a.max_rows, b = bt / a.max_rows;
    if (b >= a.batch) return;
    const Seq s = sequence(a, b);
    if (t >= s.n) return;
    const int64_t r = s.start + t, part = (r * a.heads + hd) * a.splits;
    float4_t o = {0, 0, 0, 0};
    if (s.ok) {
        float m = -INFINITY, lw = 0.0f;
        if (lane < a.splits) {
            m = part_ml_p[(part + lane) * 2];
            lw = part_ml_p[(part + lane) * 2 + 1];
        }
        float top = m;
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);  // (nothing seen there: o = l = 0)
        lw *= f;
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) lw += __shfl_xor(lw, k);
        const float *p = part_o_p + part * D + d;
        for (int k = 0; k < a.splits; k += 4 * SIDE) {
            float4_t v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = k + u * SIDE + side;
                v[u] = i < a.splits ? *reinterpret_cast<const float4_t *>(p + (size_t)i * D) : float4_t{0, 0, 0, 0};
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float fk = __shfl(f, min(k + u * SIDE + side, 63));
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(v[u][e], fk, o[e]);
            }
        }
#pragma unroll
        for (int k = LANES; k < 64; k <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], k);
        const float inv = top == -INFINITY ? 0.0f : 1.0f / lw;
        o *= inv;
    } else {
        const float nan = __builtin_nanf("");
        o = float4_t{nan, nan, nan, nan};
    }
    if (side) return;
    const int64_t at = r * a.ldo + (int64_t)hd * D + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) put<HALF>(a.out, at + e, o[e]);
}

namespace {

constexpr int kSplits = 32;  // most (a lane of the joining wave each; 64 gained nothing and cost up to half more)
constexpr int64_t kBlocks = (1 << 24) - 1;  // of 256 threads in a launch

}  // namespace

// Rows of a block and splits.
//
// Up to 32 rows a kv head: blocks of 16 or 32 rows whose waves walk their own
// keys, one to a CU, bound by its reads; as many splits as fill the chip once.
// us over splits (16 / 8 heads of 128, fp32; call after call on one state, all
// sides in turn): one token at 32000, 8 blocks unsplit: 281 at 1, 30.8 at 16,
// 25.8 at 32; two trees of 16 rows over 16000, 16 blocks: 154 at 1, 32.4 at 16,
// 44.5 at 21. Where that leaves part of the chip idle, a few rounds of smaller
// blocks: 24 sequences of 3000 to 6000, 192 blocks: 80.0 at 1, 73.4 at 4, 74.6 at
// the rule's 5 (all of 6000: 91.5, 94.0 and 94.2, which the lengths, known only
// to the device, cannot tell apart); 40 of 1500 to 3000, 320 blocks: 68.5 at 1,
// 62.6 at 3. Not below 128 positions a split (one token at 1024: 11.7 at 1, 9.7
// at 8).
//
// More rows: blocks of 64 or 128, two to a CU. The model's constants, a turn of
// 64 positions at 0.78 us for 64 rows in fp16, 1.1 in fp32, 1.18 and 1.9 for 128,
// times the blocks on the CU, a quarter more for a block alone, 8 % for a tree's
// cache that two tiles read, were fitted to an earlier form of the kernel; a block
// alone now takes 0.77, 1.10, 1.15 and 1.81 a turn. A split call writes and reads
// its partial results (4 TB/s) and has one launch more (2.5 us). Both sides with
// the present kernel, the rule's choice first: 2000 rows behind 1200, fp16: 64
// rows unsplit 51.8, split 65.8, 128 rows 65.2 and 59.2 (fp32 74.1, 87.2, 102.5
// and 83.0); 4000 rows, fp16: 128 rows 84.2, 64 rows 87.9; 16 trees of 64 over
// 500: 14.3 unsplit, 24.2 in two; 8 trees of 40 over 8000: 128 rows 55.8, 64 rows
// 56.3 (fp32 74.0 and 78.3); three trees of 61 over 16000: 128 rows at 21 splits
// 52.0, where 64 rows at 10 take 46.7 (fp32 64.9 and 62.2).
TreePlan tree_attention_plan(int64_t rows, int heads, int kv_heads, int batch, int max_rows, int max_len, int head_dim,
                             bool half, bool chain) {
    const int64_t kv_rows = (int64_t)max_rows * (heads / kv_heads), most = ((int64_t)max_len + 127) / 128;
    auto blocks_of = [&](int bm) { return (kv_rows + bm - 1) / bm * batch * kv_heads; };
    if (kv_rows <= 32) {
        const int bm = kv_rows <= 16 ? 16 : 32;
        const int64_t base = blocks_of(bm);
        if (base < 1) return {bm, 1};
        int64_t k = 256 / base;
        if (k * base * 20 < 256 * 17) k = 1024 / base;
        k = k < most ? k : most;
        return {bm, (int)(k < 1 ? 1 : k < kSplits ? k : kSplits)};
    }
    TreePlan best{64, 1};
    double least = 1e30;
    for (int bm = 64; bm <= 128; bm *= 2) {
        const double turn = (bm == 64 ? (half ? 0.78 : 1.1) * (chain ? 1.0 : 1.08) : (half ? 1.18 : 1.9)) *
                            (head_dim == 64 ? 0.65 : 1.0);
        // the block that sees most, and the mean of a chain's
        const double all = max_len / 64.0, mean = chain ? all - (max_rows < max_len ? max_rows : max_len) / 128.0 : all;
        for (int k = 1; k <= kSplits && (k == 1 || k <= most); ++k) {
            const int64_t blocks = blocks_of(bm) * k;
            const double load = blocks <= 1536 ? (double)((blocks + 255) / 256) : (double)blocks / 256.0;  // of the fullest CU
            const double alone = all / k * turn * 1.25, shared = mean / k * turn * load;
            const double t = (alone > shared ? alone : shared) +
                             (k > 1 ? 2.5 + 8e-6 / 4.0 * (double)rows * heads * k * head_dim : 0.0);
            if (t < least) {
                least = t;
                best = {bm, k};
            }
        }
    }
    if (blocks_of(best.rows) * best.splits > kBlocks) best.splits = 1;
    return best;
}

bool tree_attention_fits(int64_t kv_rows, int kv_heads, int batch, int max_rows, int heads) {
    return (kv_rows + 15) / 16 * batch <= kBlocks / kv_heads && (int64_t)batch * max_rows <= kBlocks * WAVES / heads;
}

template <int D, bool HALF, int NR, bool SHARED, bool ONCE> static hipError_t launch_tile(const TreeAttnArgs &a, int tiles, hipStream_t st) {
    using T = Tile<D, NR, SHARED>;
    const unsigned grid = (unsigned)tiles * a.splits * a.batch * a.kv_heads;
    const hipError_t e = allow_lds<&tree_attention_kernel<D, HALF, NR, SHARED, ONCE>>(T::LDS);
    if (e != hipSuccess) return e;
    tree_attention_kernel<D, HALF, NR, SHARED, ONCE><<<grid, THREADS, T::LDS, st>>>(
        a.row_start, a.cache_len, a.q, a.kv_heads, a.heads, a.splits, a.rows, a.max_rows, a.max_seq, tiles, grid <= 512, a);
    return hipGetLastError();
}

template <int D, bool HALF> static hipError_t launch_d(const TreeAttnArgs &a, int bm, hipStream_t st) {
    const int tiles = (int)(((int64_t)a.max_rows * (a.heads / a.kv_heads) + bm - 1) / bm);
    // Keys and values that one block reads once go past the caches: always with few
    // rows; of shared tiles where together they are more than the caches keep
    // (us through them and past them, call after call on one state: 30 trees of 20
    // over 6000, 369 MB, fp16 138 and 118, fp32 145 and 123; 8 of 40 over 8000, 263
    // MB, 55 and 57, 76 and 76; but 1 of 64 over 16000, 66 MB: 25.7 and 28.6, 32.9
    // and 34.5).
    const bool once = tiles == 1 && (double)a.batch * a.kv_heads * a.max_len * D * 4 > 192e6;
    hipError_t e;
    if (bm == 16) e = launch_tile<D, HALF, 1, false, true>(a, tiles, st);
    else if (bm == 32) e = launch_tile<D, HALF, 2, false, true>(a, tiles, st);
    else if (bm == 64) e = once ? launch_tile<D, HALF, 1, true, true>(a, tiles, st) : launch_tile<D, HALF, 1, true, false>(a, tiles, st);
    else e = once ? launch_tile<D, HALF, 2, true, true>(a, tiles, st) : launch_tile<D, HALF, 2, true, false>(a, tiles, st);
    if (e != hipSuccess || a.splits == 1) return e;
    const unsigned waves = (unsigned)a.batch * a.max_rows * a.heads;
    tree_join_kernel<D, HALF><<<(waves + WAVES - 1) / WAVES, THREADS, 0, st>>>(
        a.row_start, a.cache_len, a.part_ml, a.part_o, a.heads, a.splits, a.rows, a.max_rows, a.max_seq, a.batch, a);
    return hipGetLastError();
}

hipError_t launch_tree_attention(const TreeAttnArgs &a, int head_dim, bool half, int block_rows, hipStream_t st) {
    if (head_dim == 128) return half ? launch_d<128, true>(a, block_rows, st) : launch_d<128, false>(a, block_rows, st);
    return half ? launch_d<64, true>(a, block_rows, st) : launch_d<64, false>(a, block_rows, st);
}

}  // namespace q3vl
