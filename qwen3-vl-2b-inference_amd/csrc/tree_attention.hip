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

int tree_attention_splits(int64_t rows, int heads, int kv_heads, int batch, int max_rows, int max_len) { return 1; }

template <int D, bool HALF> __global__ __launch_bounds__(THREADS) void tree_attention_kernel(TreeAttnArgs a) {
    __shared__ RowScratch sh;
    const int head = blockIdx.x % a.heads, bt = blockIdx.x / a.heads;
    const int b = bt / a.max_rows, t = bt - b * a.max_rows;
    const Seq s = sequence(a, b);
    if (t >= s.n) return;
    float o = __builtin_nanf(""), m, l;
    if (s.ok) {
        row_attention<D, HALF>(a, s, b, t, head, 0, s.len + s.n, sh, o, m, l);
        o = m == -INFINITY ? 0.0f : o / l;
    }
    if (threadIdx.x < D) put<HALF>(a.out, (int64_t)(s.start + t) * a.ldo + (int64_t)head * D + threadIdx.x, o);
}

hipError_t launch_tree_attention(const TreeAttnArgs &a, int head_dim, bool half, hipStream_t st) {
    const unsigned grid = (unsigned)a.batch * (unsigned)a.max_rows * (unsigned)a.heads;
    if (head_dim == 128) {
        if (half) tree_attention_kernel<128, true><<<grid, THREADS, 0, st>>>(a);
        else tree_attention_kernel<128, false><<<grid, THREADS, 0, st>>>(a);
    } else {
        if (half) tree_attention_kernel<64, true><<<grid, THREADS, 0, st>>>(a);
        else tree_attention_kernel<64, false><<<grid, THREADS, 0, st>>>(a);
    }
    return hipGetLastError();
}

}  // namespace q3vl
