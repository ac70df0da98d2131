// long_attention.hip -- attention over long contexts: positions in 8-bit blocks
// and the fp16 rows behind them, all of them or a window of them with a few
// first ones. gfx950.
#include "q3vl_device.hpp"
#include "q3vl_kernels.hpp"
#include "q3vl_kv_blocks.hpp"

namespace q3vl {

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;

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

template <bool HALF> __device__ __forceinline__ void put(void *out, int64_t at, float v) {
    if (HALF) static_cast<uint16_t *>(out)[at] = f2h(v);
    else static_cast<float *>(out)[at] = v;
}

}  // namespace

// One workgroup a row and query head.
template <int D, bool HALF> __global__ __launch_bounds__(THREADS) void long_row_kernel(LongAttnArgs a) {
    __shared__ LongScratch sh;
    int x = blockIdx.x;
    const int head = x % a.heads;
    x /= a.heads;
    const int t = x % a.max_rows, b = x / a.max_rows, tid = threadIdx.x;
    const LongSeq s = long_sequence(a, b);
    if (t >= s.n) return;
    const int64_t at = (int64_t)(s.start + t) * a.ldo + (int64_t)head * D + tid;
    if (!s.ok) {
        if (tid < D) put<HALF>(a.out, at, __builtin_nanf(""));
        return;
    }
    const Turns<THREADS> turns = turns_of<THREADS>(a, s, s.len + (a.mask ? s.n : t + 1), window_from(a, s, t));
    float o, m, l;
    long_row<D, HALF, THREADS>(a, s, b, t, head, turns, 0, turns.count, sh, o, m, l);
    if (tid < D) put<HALF>(a.out, at, m == -INFINITY ? 0.0f : o / l);
}

hipError_t launch_long_attention(const LongAttnArgs &a, int head_dim, bool half, hipStream_t st) {
    const unsigned grid = (unsigned)a.batch * a.max_rows * a.heads;
    if (head_dim == 128) {
        if (half) long_row_kernel<128, true><<<grid, THREADS, 0, st>>>(a);
        else long_row_kernel<128, false><<<grid, THREADS, 0, st>>>(a);
    } else {
        if (half) long_row_kernel<64, true><<<grid, THREADS, 0, st>>>(a);
        else long_row_kernel<64, false><<<grid, THREADS, 0, st>>>(a);
    }
    return hipGetLastError();
}

}  // namespace q3vl
