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
// reads them again, k of V / 512, instead of every block keeping a list.
#include <type_traits>

#include "q3vl_device.hpp"
#include "q3vl_kernels.hpp"
#include "q3vl_mfma.hpp"

namespace q3vl {

namespace {

constexpr int SUB = 512;                             // values of a sub-chunk
constexpr int THREADS = 256, WAVES = THREADS / 64;   // of the scan
constexpr int FIN_WAVES = 8;                         // of the second kernel, with alternatives
constexpr float LOG2E = 1.4426950408889634f;
constexpr float FAR = -208.0f;    // x - m from which e^(x - m) is 0 in fp32
constexpr float TALL = 1e30f;     // a maximum up to which x - m is finite for every finite x (half a step of the
                                  // largest float is 2^103 = 1.01e31)

// v_max_f32 and v_min_f32 as they are, for operands that are no NaN: no
// instruction goes to quieting one first.
__device__ __forceinline__ float vmax(float a, float b) {
#if defined(__HIP_DEVICE_COMPILE__)
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
#else
    return a > b ? a : b;
#endif
}
__device__ __forceinline__ float vmin(float a, float b) {
#if defined(__HIP_DEVICE_COMPILE__)
    float r;
    asm("v_min_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
#else
    return a < b ? a : b;
#endif
}

// (maximum, sum of the rest, weighted sum) of some values
struct Sums {
    float m, r, t;
};

// e^d for d = lo - m, lo <= m. CUT: d cut off where the weight is 0, which
// keeps -inf (0 times infinity otherwise) out of t. Without it d has to be
// finite: d log2 e may overflow (d below -2.36e38, as of a mask of the type's
// lowest value), which makes the weight 0 and leaves d, that t takes, as it is.
// m is finite here.
template <bool CUT = true> __device__ __forceinline__ float weight(float lo, float m, float &d) {
    d = lo - m;
    if (CUT) d = fmaxf(d, FAR);
    return __builtin_amdgcn_exp2f(d * LOG2E);
}

__device__ __forceinline__ float lane_swap_max(float v) {
    v = row16_max(v);
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = vmax(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return vmax(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float lane_swap_sum(float v) {
    v += dpp_f(v, dpp_xor1);
    v += dpp_f(v, dpp_xor2);
    v += dpp_f(v, dpp_half_mirror);
    v += dpp_f(v, dpp_mirror);
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The 64 lanes' sums as one, in every lane: each scaled to the common maximum;
// every lane's own maximum enters r but one that is the common one.
__device__ __forceinline__ Sums wave_join(Sums s) {
    Sums o;
    o.m = lane_swap_max(s.m);
    const uint64_t top = __ballot(s.m == o.m);
    float d;
    const float w = weight(s.m, fmaxf(o.m, -FLT_MAX), d);
    const bool out = __lane_id() == (uint32_t)__builtin_ctzll(top | 1ull << 63);
    o.r = lane_swap_sum(fmaf(s.r, w, out ? 0.0f : w));
    o.t = lane_swap_sum(fmaf(fmaf(s.r, d, s.t), w, out ? 0.0f : w * d));
    return o;
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

// Sub-chunks lie on 16-byte boundaries, so a row may touch one more than its size asks for.
int logprob_subs(int V) { return (V + 7 + SUB - 1) / SUB; }

// Blocks a row. A turn of a wave is two sub-chunks; every wave but the last has
// as many turns as keep all rows' blocks to about 4096 or fewer (110 rows of
// 151936: 2 turns, 2090 blocks; 777: 8, 3885). With fewer than 4 x 4096 turns over
// all rows a wave has one (1 row 38 blocks, 61 rows 2318).
int logprob_parts(int M, int V) {
    const int64_t turns = (V + 7 + 2 * SUB - 1) / (2 * SUB);
    int64_t each = (turns * M + 2 * WAVES * 2048) / (WAVES * 4096);
    if (each < 1) each = 1;
    const int64_t p = (turns + WAVES * each - 1) / (WAVES * each);
    return (int)(p < kLogprobParts ? p : kLogprobParts);
}

// No fewer than m * logprob_parts(m, v) for any m <= M, v <= V: turns * m < WAVES
// 4096 each, so m * (turns / (WAVES each) + 1) stays below 4096 + m.
int64_t logprob_parts_most(int M, int V) {
    const int64_t all = (int64_t)M * logprob_parts(1, V), few = 4096 + (int64_t)M;
    return all < few ? all : few;
}

// A lane's 16 bytes of a row, values [i, i + VEC), -inf outside of [0, V);
// inside: the whole wave's piece lies in the row.
template <bool HALF> __device__ __forceinline__ u32x4 read_piece(const void *x, int i, int V, bool inside) {
    constexpr int VEC = HALF ? 8 : 4;
    const unsigned char *p = static_cast<const unsigned char *>(x) + (int64_t)i * (HALF ? 2 : 4);
    if (inside || (i >= 0 && i + VEC <= V)) return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
    u32x4 r;
    if constexpr (HALF) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = i + 2 * e;
            const uint32_t lo = k >= 0 && k < V ? static_cast<const uint16_t *>(x)[k] : 0xFC00u;
            const uint32_t hi = k + 1 >= 0 && k + 1 < V ? static_cast<const uint16_t *>(x)[k + 1] : 0xFC00u;
            r[e] = lo | hi << 16;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = i + e >= 0 && i + e < V ? static_cast<const uint32_t *>(x)[i + e] : 0xFF800000u;
    }
    return r;
}
template <bool HALF> __device__ __forceinline__ float piece_value(u32x4 r, int e) {
    return HALF ? h2f((uint16_t)(r[e >> 1] >> (16 * (e & 1)))) : __uint_as_float(r[e & 3]);
}

// Values before the row's first 16-byte boundary counted back to it.
template <bool HALF> __device__ __forceinline__ int row_offset(const void *x) {
    return HALF ? (int)((uintptr_t)x / 2 % 8) : (int)((uintptr_t)x / 4 % 4);
}

// A wave takes two sub-chunks a turn, 16 values a lane. The largest of them and
// of the lane's running maximum wins a tournament whose losers are exactly the
// values that enter the sum: one more instruction a value than a maximum alone.
// 209 VALU instructions a turn (13 a value of a lane): 777 rows of 151936 in fp16
// hold the VALU for 99 of 100 busy cycles, 48.9 us, where the reads need 36.5. 61
// rows in fp32: 10.6 us for 5.7 of reads, one turn a wave: 2318 blocks that each
// pay the token's load, two joins across lanes and a barrier for 16 values a lane.
template <bool HALF>
__global__ __launch_bounds__(THREADS) void logprob_scan_kernel(const void *logits_p, int64_t ld_p, const int32_t *tokens_p,
                                                              int parts_p, int V_p, int subs_max, LogprobArgs args) {
    LogprobArgs a = args;  // (the leading arguments arrive in registers)
    a.logits = logits_p;
    a.ld = ld_p;
    a.tokens = tokens_p;
    a.parts = parts_p;
    a.V = V_p;
    constexpr int VEC = HALF ? 8 : 4, U = 16 / VEC;  // values a load, loads a turn
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts, tid = threadIdx.x, lane = tid & 63;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const void *x = HALF ? (const void *)(static_cast<const uint16_t *>(a.logits) + row * a.ld)
                         : (const void *)(static_cast<const float *>(a.logits) + row * a.ld);
    const int off = row_offset<HALF>(x);
    const int turns = (a.V + off + 2 * SUB - 1) / (2 * SUB);
    const int first = (int)((int64_t)turns * part / a.parts), last = (int)((int64_t)turns * (part + 1) / a.parts);
    u32x4 raw[U];  // the turn's values, loaded a turn ahead
    auto load = [&](int c) {
        const int base = c * 2 * SUB - off;
        const bool inside = base >= 0 && base + 2 * SUB <= a.V;
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = read_piece<HALF>(x, base + (u * 64 + lane) * VEC, a.V, inside);
    };
    if (first + wid < last) load(first + wid);
    const int t = a.tokens[row];
    const bool ok = t >= 0 && t < a.V;
    float xt = ok ? logit<HALF>(x, t) : 0.0f;
    if (part == 0 && tid == 0) a.logprob[row] = ok ? xt : __builtin_nanf("");  // (for the second kernel)
    if (!(xt > -INFINITY)) xt = -INFINITY;
    Sums s{-INFINITY, 0.0f, 0.0f};
    float z = 0.0f;  // NaN once a NaN (or infinities of both signs) has been read
    int n = 0;
    for (int c = first + wid; c < last; c += WAVES) {
        const int base = c * 2 * SUB - off;
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[u][e] = piece_value<HALF>(raw[u], e);
        if (c + WAVES < last) load(c + WAVES);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e) z = fmaf(v[u][e], 0x1p-64f, z);
        if (__any(z != z)) {  // NaN as -inf (a signalling one would win the tournament)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[u][e] = v[u][e] > -INFINITY ? v[u][e] : -INFINITY;
        }
        // values ahead of the token: larger ones, and equal ones before it
        if (xt > -INFINITY) {
            if (base + 2 * SUB <= t) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) n += __builtin_popcountll(__ballot(v[u][e] >= xt));
            } else if (base > t) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) n += __builtin_popcountll(__ballot(v[u][e] > xt));
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        n += __builtin_popcountll(__ballot(ahead(v[u][e], base + (u * 64 + lane) * VEC + e, xt, t)));
            }
        } else {  // everything above -inf, and what stands with it before the token
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = base + (u * 64 + lane) * VEC + e;
                    n += __builtin_popcountll(__ballot(i >= 0 && i < a.V && (v[u][e] > -INFINITY || i < t)));
                }
        }
        float lose[16], win[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = v[2 * i / VEC][2 * i % VEC], q = v[2 * i / VEC][2 * i % VEC + 1];
            win[i] = vmax(p, q);
            lose[i] = vmin(p, q);
        }
        // (win: pairs in order, so halves of it are the turn's sub-chunks)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lose[8 + i] = vmin(win[2 * i], win[2 * i + 1]);
            win[i] = vmax(win[2 * i], win[2 * i + 1]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            lose[12 + i] = vmin(win[2 * i], win[2 * i + 1]);
            win[i] = vmax(win[2 * i], win[2 * i + 1]);
        }
        if (a.k) {
            const float m0 = lane_swap_max(win[0]), m1 = lane_swap_max(win[1]);
            if (lane < 2 && 2 * c + lane < subs_max) a.sub_max[(size_t)row * subs_max + 2 * c + lane] = lane ? m1 : m0;
        }
        lose[14] = vmin(win[0], win[1]);
        const float best = vmax(win[0], win[1]);
        lose[15] = vmin(best, s.m);
        const float m = vmax(best, s.m), ref = vmax(m, -FLT_MAX);
        if (__any(best > s.m)) {
            float d;
            const float w = weight(s.m, ref, d);
            s.t = fmaf(s.r, d, s.t) * w;
            s.r *= w;
            s.m = m;
        }
        float r[2] = {0.0f, 0.0f}, q[2] = {0.0f, 0.0f};
        auto add = [&](auto cut) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float d;
                const float w = weight<decltype(cut)::value>(lose[i], ref, d);
                r[i & 1] += w;
                q[i & 1] = fmaf(w, d, q[i & 1]);
            }
        };
        // (z is finite until a value was not; lose[15] is -inf in the first turn;
        // up to TALL the difference of two finite values is finite)
        if (__any(!(__builtin_fabsf(z) < INFINITY) || lose[15] == -INFINITY || ref > TALL)) add(std::true_type{});
        else add(std::false_type{});
        s.r += r[0] + r[1];
        s.t += q[0] + q[1];
    }
    if (z != z) s.r = z;
    s = wave_join(s);
    __shared__ float sh[WAVES][4];
    if (lane == 0) {
        sh[wid][0] = s.m;
        sh[wid][1] = s.r;
        sh[wid][2] = s.t;
        sh[wid][3] = __int_as_float(n);
    }
    __syncthreads();
    if (tid >= 64) return;
    const bool mine = lane < WAVES;
    s = wave_join(Sums{mine ? sh[lane & 3][0] : -INFINITY, mine ? sh[lane & 3][1] : 0.0f, mine ? sh[lane & 3][2] : 0.0f});
    if (lane == 0) {
        n = 0;
        for (int w = 0; w < WAVES; ++w) n += __float_as_int(sh[w][3]);
        float *o = a.part + ((size_t)row * a.parts + part) * 4;
        o[0] = s.m;
        o[1] = s.r;
        o[2] = s.t;
        o[3] = __int_as_float(ok ? n : -1);
    }
}

// The best keys that one wave has seen: up to 64 kept in order, and room for a
// push of 64 more. A key's rank is how many of the others are larger (keys are
// distinct), found by broadcasting each; once k are kept, what is not above the
// last of them is not taken up.
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

struct Best {
    uint64_t *buf;  // LDS, 128
    int k, n;
    uint64_t floor;

    __device__ void sort() {
        const int lane = __lane_id();
        wave_lds_sync();
        const uint64_t p = lane < n ? buf[lane] : 0, q = lane + 64 < n ? buf[lane + 64] : 0;
        int rp = 0, rq = 0;
        // (absent keys are 0, larger than none)
        if (n <= 64) {
            for (int i = 0; i < n; i += 8)
#pragma unroll
                for (int u = 0; u < 8; ++u) rp += from_lane(p, i + u) > p;
        } else {
            for (int i = 0; i < 64; i += 4)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint64_t o = from_lane(p, i + u), w = from_lane(q, i + u);
                    rp += (o > p) + (w > p);
                    rq += (o > q) + (w > q);
                }
        }
        wave_lds_sync();
        if (lane < n && rp < k) buf[rp] = p;
        if (lane + 64 < n && rq < k) buf[rq] = q;
        n = min(n, k);
        wave_lds_sync();
        if (n == k) {
            const uint64_t last = from_lane(buf[k - 1], 0);
            floor = last > floor ? last : floor;
        }
    }
    // A sort each time that 32 came after the k kept ones, or else each value
    // taken up would cost one where k is 64; before that where a push might not fit.
    __device__ __forceinline__ void push(uint64_t key, bool take) {
        take = take && key > floor;
        uint64_t m = __ballot(take);
        if (!m) return;
        if (n + __builtin_popcountll(m) > 128) {
            sort();
            take = take && key > floor;
            m = __ballot(take);
            if (!m) return;
        }
        if (take) buf[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0))] = key;
        n += __builtin_popcountll(m);
        if (n >= 64 && n - k >= 32) sort();
    }
};

// LDS of the second kernel.
struct FinishLds {
    uint64_t buf[FIN_WAVES][128];
    uint64_t list[FIN_WAVES * kLogprobTop];  // of all waves, what can be among the first k
    uint64_t out[kLogprobTop];               // the first k in order
    int rank[FIN_WAVES * kLogprobTop];
    int count[FIN_WAVES];
    int n;
};

// The waves' lists as one, in sh.out; how many there are (k at most). The
// largest of the waves' own k-th keys bounds the answer's from below. So does
// the smallest of their k/8-th keys (rounded up: together they have k that are
// no smaller), which leaves fewer candidates: `wide`, where every value of a row
// was one (us a call at k = 64: 67 rows of 32000 86 -> 73, 323 of 3812 70 -> 58;
// elsewhere few are left anyway and it costs 0.6 to 0.8). A candidate's
// comparisons are spread over the waves.
__device__ int merge(Best &best, FinishLds &sh, int wid, bool mine, bool wide) {
    const int lane = __lane_id(), tid = threadIdx.x, k = best.k;
    if (mine) {
        best.sort();
        if (lane == 0) sh.count[wid] = best.n;
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    if (mine) {
        uint64_t bound = lane < FIN_WAVES && sh.count[lane] == k ? sh.buf[lane][k - 1] : 0;
#pragma unroll
        for (int o = 1; o < FIN_WAVES; o <<= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)bound, o);
            bound = other > bound ? other : bound;
        }
        bound = from_lane(bound, 0);
        if (wide) {
            const int kk = (k + FIN_WAVES - 1) / FIN_WAVES;
            uint64_t low = lane >= FIN_WAVES ? ~0ull : sh.count[lane] >= kk ? sh.buf[lane][kk - 1] : 0;
#pragma unroll
            for (int o = 1; o < FIN_WAVES; o <<= 1) {
                const uint64_t other = __shfl_xor((unsigned long long)low, o);
                low = other < low ? other : low;
            }
            low = from_lane(low, 0);
            bound = low > bound ? low : bound;
        }
        const bool take = lane < best.n && best.buf[lane] >= bound;
        const uint64_t m = __ballot(take);  // (lists are in order: a leading run)
        int at = 0;
        if (lane == 0 && m) at = atomicAdd(&sh.n, __builtin_popcountll(m));
        at = __builtin_amdgcn_readfirstlane(at);
        if (take) {
            sh.list[at + lane] = best.buf[lane];
            sh.rank[at + lane] = 0;
        }
    }
    __syncthreads();
    const int n = sh.n;
    if (mine) {
        for (int c = lane; c < n; c += 64) {
            const uint64_t key = sh.list[c];
            int r = 0;
            for (int i = wid; i < n; i += 4 * FIN_WAVES) {
                uint64_t o[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) o[u] = sh.list[min(i + u * FIN_WAVES, n - 1)];
#pragma unroll
                for (int u = 0; u < 4; ++u) r += i + u * FIN_WAVES < n && o[u] > key;
            }
            if (r) atomicAdd(&sh.rank[c], r);
        }
    }
    __syncthreads();
    if (mine)
        for (int c = tid; c < n; c += 64 * FIN_WAVES)
            if (sh.rank[c] < k) sh.out[sh.rank[c]] = sh.list[c];
    __syncthreads();
    return min(n, k);
}

// One block a row: a wave joins the parts' sums; eight others (TOP) find the
// alternatives.
template <bool HALF, bool TOP>
__global__ __launch_bounds__(TOP ? 64 * (FIN_WAVES + 1) : 64) void logprob_finish_kernel(
    const void *logits_p, int64_t ld_p, const float *sub_max_p, const float *part_p, float *logprob_p, int parts_p, int V_p,
    int k_p, int subs_max, LogprobArgs args) {
    LogprobArgs a = args;
    a.logits = logits_p;
    a.ld = ld_p;
    a.logprob = logprob_p;
    a.parts = parts_p;
    a.V = V_p;
    a.k = k_p;
    constexpr int VEC = HALF ? 8 : 4, PER = SUB / (64 * VEC);
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const void *x = HALF ? (const void *)(static_cast<const uint16_t *>(a.logits) + row * a.ld)
                         : (const void *)(static_cast<const float *>(a.logits) + row * a.ld);
    const float nan = __builtin_nanf("");
    __shared__ float whole[2];
    if (wid == (TOP ? FIN_WAVES : 0)) {
        const float xt = a.logprob[row];  // the token's value, from the scan
        Sums s{-INFINITY, 0.0f, 0.0f};
        int n = 0;  // below 0: no such token
        for (int p = 0; p < a.parts; p += 64) {
            Sums q{-INFINITY, 0.0f, 0.0f};
            int c = 0;
            if (p + lane < a.parts) {
                const float4_t o = *reinterpret_cast<const float4_t *>(part_p + ((size_t)row * a.parts + p + lane) * 4);
                q = Sums{o[0], o[1], o[2]};
                c = __float_as_int(o[3]);
            }
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) c += __shfl_xor(c, o);
            n += c;
            q = wave_join(q);
            if (p == 0) s = q;
            else s = wave_join(Sums{lane == 0 ? s.m : lane == 1 ? q.m : -INFINITY, lane == 0 ? s.r : lane == 1 ? q.r : 0.0f,
                                    lane == 0 ? s.t : lane == 1 ? q.t : 0.0f});
        }
        const float logs = s.m > -INFINITY && s.m < INFINITY ? log1pf(s.r) : nan;
        if (lane == 0) {
            whole[0] = s.m;
            whole[1] = logs;
            a.logprob[row] = (xt - s.m) - logs;
            if (a.rank) a.rank[row] = n < 0 ? -1 : n;
            if (a.entropy) a.entropy[row] = logs - s.t / (1.0f + s.r);
        }
    }
    if constexpr (TOP) {
        __shared__ FinishLds sh;
        const bool mine = wid < FIN_WAVES;
        const int off = row_offset<HALF>(x), subs = (a.V + off + SUB - 1) / SUB;
        Best best{sh.buf[mine ? wid : 0], a.k, 0, 0};
        if (mine)
            for (int c = wid * 64; c < subs; c += 64 * FIN_WAVES) {
                const int i = c + lane;
                best.push(i < subs ? key_of(sub_max_p[(size_t)row * subs_max + i], i) : 0, i < subs);
            }
        const int chunks = merge(best, sh, wid, mine, false);
        if (mine) {
            // values below the k-th sub-chunk's maximum have k others ahead of them
            const uint64_t bound = chunks == a.k ? sh.out[a.k - 1] & ~0xFFFFFFFFull : 0;
            best = Best{sh.buf[wid], a.k, 0, 0};
            // (one float comparison a value first: few values pass. -inf: all do)
            const float least = bound ? value_of(bound) : -INFINITY;
            const bool all = !(least > -INFINITY);
            constexpr int AHEAD = 4;  // sub-chunks under way
            for (int c = wid; c < chunks; c += AHEAD * FIN_WAVES) {
                u32x4 raw[AHEAD][PER];
                int base[AHEAD];
#pragma unroll
                for (int g = 0; g < AHEAD; ++g) {
                    if (c + g * FIN_WAVES >= chunks) break;  // (uniform)
                    base[g] = (int)index_of(sh.out[c + g * FIN_WAVES]) * SUB - off;
#pragma unroll
                    for (int u = 0; u < PER; ++u) raw[g][u] = read_piece<HALF>(x, base[g] + (u * 64 + lane) * VEC, a.V, false);
                }
#pragma unroll
                for (int g = 0; g < AHEAD; ++g) {
                    if (c + g * FIN_WAVES >= chunks) break;
#pragma unroll
                    for (int u = 0; u < PER; ++u)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float v = piece_value<HALF>(raw[g][u], e);
                            if (!__any(all || v >= least)) continue;
                            const int i = base[g] + (u * 64 + lane) * VEC + e;
                            const uint64_t key = key_of(v, i);
                            best.push(key, key >= bound && i >= 0 && i < a.V);
                        }
                }
            }
        }
        merge(best, sh, wid, mine, chunks < a.k);
        if (wid == 0 && lane < a.k) {
            const uint64_t key = sh.out[lane];
            a.top_ids[(size_t)row * a.k + lane] = (int32_t)index_of(key);
            a.top_logprobs[(size_t)row * a.k + lane] = (value_of(key) - whole[0]) - whole[1];
        }
    }
}

template <bool HALF> static hipError_t launch_half(const LogprobArgs &a, hipStream_t st) {
    const int subs = logprob_subs(a.V);
    logprob_scan_kernel<HALF><<<(unsigned)a.parts * (unsigned)a.M, THREADS, 0, st>>>(a.logits, a.ld, a.tokens, a.parts, a.V, subs, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.k)
        logprob_finish_kernel<HALF, true><<<a.M, 64 * (FIN_WAVES + 1), 0, st>>>(a.logits, a.ld, a.sub_max, a.part, a.logprob,
                                                                               a.parts, a.V, a.k, subs, a);
    else
        logprob_finish_kernel<HALF, false><<<a.M, 64, 0, st>>>(a.logits, a.ld, a.sub_max, a.part, a.logprob, a.parts, a.V, a.k,
                                                              subs, a);
    return hipGetLastError();
}

hipError_t launch_token_logprobs(const LogprobArgs &a, bool half, hipStream_t st) {
    return half ? launch_half<true>(a, st) : launch_half<false>(a, st);
}

}  // namespace q3vl
