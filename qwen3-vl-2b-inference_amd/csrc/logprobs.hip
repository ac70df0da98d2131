// logprobs.hip -- what rows of logits say about given tokens: log probability,
// rank, entropy and the best alternatives. gfx950.
//
// One pass over the logits: per part of a row the running maximum m, the sum
// r = sum e^(x - m) over every value but the one maximum, the weighted sum
// t = sum e^(x - m) (x - m), and how many values stand ahead of the token; per
// sub-chunk of the row its maximum. Then, with s = 1 + r,
//   log p(x) = (x - m) - log1p(r),   H = log1p(r) - t / s.
// Leaving the maximum's own 1 out of r keeps log1p(r) exact to the last digits
// where one token has nearly all of the probability.
//
// The k best values lie in the k sub-chunks whose maxima come first (larger
// first, equal ones by place): each of k others ahead of a sub-chunk has a
// value ahead of all of its own. The second kernel picks those sub-chunks and
// reads them again, k of V / 256, instead of every block keeping a list.
#include "q3vl_device.hpp"
#include "q3vl_kernels.hpp"

namespace q3vl {

namespace {

constexpr int SUB = 256;          // values of a sub-chunk
constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float FAR = -300.0f;    // exponent (base 2) from which 2^x is 0 in fp32

typedef uint32_t lp_u32x4 __attribute__((ext_vector_type(4)));

// (maximum, sum of the rest, weighted sum in base 2) of some values
struct Sums {
    float m, r, t;
};

// 2^((lo - m) log2 e) for lo <= m, and its exponent, cut off where it is 0:
// keeps -inf (0 times infinity otherwise) out of t. m is finite here.
__device__ __forceinline__ float weight(float lo, float m, float &arg) {
    arg = fmaxf((lo - m) * LOG2E, FAR);
    return __builtin_amdgcn_exp2f(arg);
}

__device__ __forceinline__ Sums join(Sums a, Sums b) {
    Sums o;
    o.m = fmaxf(a.m, b.m);
    const float ref = fmaxf(o.m, -FLT_MAX);
    float ea, eb;
    const float wa = weight(a.m, ref, ea), wb = weight(b.m, ref, eb);
    // one of the two maxima stays out of the sum; the other enters it
    const bool a_top = a.m >= b.m;
    o.r = (a.r * wa + b.r * wb) + (a_top ? wb : wa);
    o.t = (fmaf(a.r, ea, a.t) * wa + fmaf(b.r, eb, b.t) * wb) + (a_top ? wb * eb : wa * ea);
    return o;
}

__device__ __forceinline__ Sums wave_join(Sums s) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) s = join(s, Sums{__shfl_xor(s.m, o), __shfl_xor(s.r, o), __shfl_xor(s.t, o)});
    return s;
}

// A value's place in the order: larger floats first, -0 as 0, NaN as -inf.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (!(x > -INFINITY)) x = -INFINITY;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
// ... with the place in the row: a key per value, the largest key ahead.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return (uint64_t)ordered(x) << 32 | (0xFFFFFFFFu - i); }
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o ^ (o & 0x80000000u ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

template <bool HALF> __device__ __forceinline__ float logit(const void *p, int64_t i) {
    return HALF ? h2f(static_cast<const uint16_t *>(p)[i]) : static_cast<const float *>(p)[i];
}

// Whether x stands ahead of the token's value xt at place t.
__device__ __forceinline__ bool ahead(float x, int i, float xt, int t) { return x > xt || (x == xt && i < t); }

}  // namespace

int logprob_subs(int V) { return (V + SUB - 1) / SUB; }

int logprob_parts(int M, int V) {
    const int subs = logprob_subs(V), most = (subs + WAVES - 1) / WAVES;
    const int want = (2048 + M - 1) / M;
    const int p = want < most ? want : most;
    return p < 1 ? 1 : p < kLogprobParts ? p : kLogprobParts;
}

template <bool HALF>
__global__ __launch_bounds__(THREADS) void logprob_scan_kernel(LogprobArgs a) {
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts, tid = threadIdx.x, lane = tid & 63;
    const void *x = HALF ? (const void *)(static_cast<const uint16_t *>(a.logits) + row * a.ld)
                         : (const void *)(static_cast<const float *>(a.logits) + row * a.ld);
    const int subs = (a.V + SUB - 1) / SUB;
    const int first = (int)((int64_t)subs * part / a.parts), last = (int)((int64_t)subs * (part + 1) / a.parts);
    const int t = a.tokens[row];
    const bool ok = t >= 0 && t < a.V;
    float xt = ok ? logit<HALF>(x, t) : 0.0f;
    if (!(xt > -INFINITY)) xt = -INFINITY;
    Sums s{-INFINITY, 0.0f, 0.0f};
    int n = 0;
    bool bad = false;
    for (int c = first + (tid >> 6); c < last; c += WAVES) {
        float best = -INFINITY;
#pragma unroll
        for (int u = 0; u < SUB / 64; ++u) {
            const int i = c * SUB + u * 64 + lane;
            if (i >= a.V) continue;
            const float raw = logit<HALF>(x, i);
            bad = bad || raw != raw;
            const float v = raw > -INFINITY ? raw : -INFINITY;
            n += ahead(v, i, xt, t);
            best = fmaxf(best, v);
            s = join(s, Sums{v, 0.0f, 0.0f});
        }
        if (a.k) {
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) best = fmaxf(best, __shfl_xor(best, o));
            if (lane == 0) a.sub_max[(size_t)row * subs + c] = best;
        }
    }
    if (bad) s.r = __builtin_nanf("");
    s = wave_join(s);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o);
    __shared__ float sh[WAVES][4];
    if (lane == 0) {
        sh[tid >> 6][0] = s.m;
        sh[tid >> 6][1] = s.r;
        sh[tid >> 6][2] = s.t;
        sh[tid >> 6][3] = __int_as_float(n);
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < WAVES; ++w) {
            s = join(s, Sums{sh[w][0], sh[w][1], sh[w][2]});
            n += __float_as_int(sh[w][3]);
        }
        float *o = a.part + ((size_t)row * a.parts + part) * 4;
        o[0] = s.m;
        o[1] = s.r;
        o[2] = s.t;
        o[3] = __int_as_float(n);
    }
}

template <bool HALF>
__global__ __launch_bounds__(THREADS) void logprob_finish_kernel(LogprobArgs a) {
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const void *x = HALF ? (const void *)(static_cast<const uint16_t *>(a.logits) + row * a.ld)
                         : (const void *)(static_cast<const float *>(a.logits) + row * a.ld);
    const int subs = (a.V + SUB - 1) / SUB;
    __shared__ float sh[WAVES][4];
    __shared__ uint64_t best[WAVES];
    Sums s{-INFINITY, 0.0f, 0.0f};
    int n = 0;
    for (int p = tid; p < a.parts; p += THREADS) {
        const float *o = a.part + ((size_t)row * a.parts + p) * 4;
        s = join(s, Sums{o[0], o[1], o[2]});
        n += __float_as_int(o[3]);
    }
    s = wave_join(s);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) n += __shfl_xor(n, o);
    if (lane == 0) {
        sh[tid >> 6][0] = s.m;
        sh[tid >> 6][1] = s.r;
        sh[tid >> 6][2] = s.t;
        sh[tid >> 6][3] = __int_as_float(n);
    }
    __syncthreads();
    s = Sums{sh[0][0], sh[0][1], sh[0][2]};
    n = __float_as_int(sh[0][3]);
    for (int w = 1; w < WAVES; ++w) {
        s = join(s, Sums{sh[w][0], sh[w][1], sh[w][2]});
        n += __float_as_int(sh[w][3]);
    }
    const float nan = __builtin_nanf("");
    const bool fine = s.m > -INFINITY && s.m < INFINITY;
    const float logs = fine ? log1pf(s.r) : nan;
    if (tid == 0) {
        const int t = a.tokens[row];
        const bool ok = t >= 0 && t < a.V;
        a.logprob[row] = ok ? (logit<HALF>(x, t) - s.m) - logs : nan;
        if (a.rank) a.rank[row] = ok ? n : -1;
        if (a.entropy) a.entropy[row] = logs - LN2 * s.t / (1.0f + s.r);
    }
    // the k best: the first key below the last one taken, k times
    uint64_t below = ~0ull;
    for (int j = 0; j < a.k; ++j) {
        uint64_t mine = 0;
        for (int c = tid >> 6; c < subs; c += WAVES) {
            if (key_of(a.sub_max[(size_t)row * subs + c], 0) < mine) continue;
            for (int i = c * SUB + lane; i < min(a.V, (c + 1) * SUB); i += 64) {
                const uint64_t key = key_of(logit<HALF>(x, i), i);
                if (key < below && key > mine) mine = key;
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)mine, o);
            mine = other > mine ? other : mine;
        }
        __syncthreads();
        if (lane == 0) best[tid >> 6] = mine;
        __syncthreads();
        below = best[0];
        for (int w = 1; w < WAVES; ++w) below = best[w] > below ? best[w] : below;
        if (tid == 0) {
            a.top_ids[(size_t)row * a.k + j] = (int32_t)index_of(below);
            a.top_logprobs[(size_t)row * a.k + j] = (value_of(below) - s.m) - logs;
        }
    }
}

hipError_t launch_token_logprobs(const LogprobArgs &a, bool half, hipStream_t st) {
    const unsigned grid = (unsigned)a.parts * (unsigned)a.M;
    if (half) logprob_scan_kernel<true><<<grid, THREADS, 0, st>>>(a);
    else logprob_scan_kernel<false><<<grid, THREADS, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (half) logprob_finish_kernel<true><<<a.M, THREADS, 0, st>>>(a);
    else logprob_finish_kernel<false><<<a.M, THREADS, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace q3vl
