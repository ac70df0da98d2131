// verify.hip -- drafted tokens judged against the target's probabilities by
// rejection sampling, along chains and trees. gfx950.
//
// With p the target's probabilities after a row and q those that its children
// were drawn from, a rejected child leaves max(r - q, 0) / sum of the
// distribution r that it was tested against. From r = p this is
//   r = max(p - c q, 0) / Z,  Z = sum max(p - c q, 0),  c' = c + Z,
// as max(max(p - c q, 0) / Z - q, 0) = max(p - (c + Z) q, 0) / Z: one number c
// stands for any number of rejections. Nothing that a row decides depends on
// another row: every row decides at once, and the path is followed after.
//
// In 64 bits throughout: the choices are comparisons, and every implementation
// of their definition should come to the same one.
//
// Rows are cut into chunks, one wave each. The first kernel leaves a chunk's
// maximum m_c and sum of e^((x - m_c) / T). From these a workgroup a row joins m
// and the whole sum, tests the row's children and, if the row is decided, finds
// the chunk in which the cumulated sums pass the row's number and the value in
// it. A row whose child is rejected waits for a round: its chunks' sums of max(p
// - c q, 0), by all workgroups again, then the next test. So each logit is read
// once, or once more for each rejection. Two rounds are launched; a row that they
// leave open goes on by itself, a workgroup for all its chunks, which costs most
// where trees have many children a row. us a call with 1, 2, 4 and 6 rounds, values
// as below: 16 chains of 8 rows 43, 47, 55, 63; 8 trees of 16 rows 102, 53, 60, 68; 3
// trees of 61 rows, with up to nine children, 212, 171, 113, 103 (with 2, the last
// step alone 126).
//
// us at 151936 values, fp32: the sums of 83 rows 15.5, of 164 24 (4.2 TB/s: 64-bit
// conversions and products, 71 of 100 busy cycles in vector instructions), a step
// 6 to 8 (its chain of loads: lengths, parents and tokens, logits, the chunk), a round
// of which two rows in five have a part 12, the path 3 to 4. All tests and the
// choice in one workgroup a row took 545 for the 83.
#include "q3vl_device.hpp"
#include "q3vl_kernels.hpp"

namespace q3vl {

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int SMALL = 9, LARGE = 11;  // chunks of 2^9 or 2^11 values

// 2^(z / 32) for z <= 0: z = n + f, |f| <= 1/2, 2^(n / 32) from a table of the 32
// fractions, and 2^(f / 32) by the polynomial of degree 5 that takes its values at
// the Chebyshev nodes (1.4e-16 off, relatively). Without the table the degree is
// 11: 164 rows' sums 26.0 us for 24.0.
__constant__ double kFractions[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924, 1.1387886347566916,
    1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332, 1.2968395546510096,
    1.3252366431597413, 1.3542555469368927, 1.383909881963832, 1.4142135623730951, 1.4451808069770467, 1.4768261459394993,
    1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.6457554781539649, 1.681792830507429,
    1.7186192981224779, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103, 1.9152065613971474,
    1.9571441241754002};
__device__ __forceinline__ void fill_table(double *table) {  // (a barrier follows)
    if (threadIdx.x < 32) table[threadIdx.x] = kFractions[threadIdx.x];
}
__device__ __forceinline__ double exp2_64(double z, const double *table) {
    z = fmax(z, -64000.0);  // (0 then: a double's least is 2^-1074)
    const double n = __builtin_rint(z), f = z - n;
    const int i = (int)n;
    double r = 3.9737266313166245e-11;
    r = fma(r, f, 9.1726164981598514e-09);
    r = fma(r, f, 1.6938509724215757e-06);
    r = fma(r, f, 0.00023459619819720339);
    r = fma(r, f, 0.02166084939249829);
    r = fma(r, f, 1.0);
    return __builtin_ldexp(r * table[i & 31], i >> 5);
}
// e^((x - m) / T), with per = 32 log2 e / T
struct Weight {
    double per, top;
    const double *table;
    __device__ __forceinline__ Weight(float m, double p, const double *t) : per(p), top(m), table(t) {}
    __device__ __forceinline__ double operator()(float x) const { return exp2_64(((double)x - top) * per, table); }
};
__device__ __forceinline__ double draft_of(float q) { return q > 0.0f ? (double)q : 0.0; }

// A lane's value from the lane `ctrl` says, 0 where there is none or `rows` (of 16
// lanes, a bit each) leaves it out: data-parallel moves, an eighth of the latency
// of an exchange through LDS.
template <int ctrl, int rows> __device__ __forceinline__ double moved(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, ctrl, rows, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), ctrl, rows, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double v) {  // inclusive
    v += moved<0x111, 0xF>(v);  // from 1, 2, 4, 8 lanes before in the row
    v += moved<0x112, 0xF>(v);
    v += moved<0x114, 0xF>(v);
    v += moved<0x118, 0xF>(v);
    v += moved<0x142, 0xA>(v);  // lane 15 of the row before, to rows 1 and 3
    v += moved<0x143, 0xC>(v);  // lane 31, to rows 2 and 3
    return v;
}
__device__ __forceinline__ double lane_value(double v, int lane) {  // (lane uniform)
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double v) { return lane_value(wave_scan(v), 63); }
__device__ __forceinline__ float wave_max(float v) {
    v = row16_max(v);
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// (rows may begin anywhere)
typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h4_any __attribute__((ext_vector_type(4), aligned(2)));

// Values of a row from `i` on, four and every `step` again; behind its end `rest`.
template <bool HALF, int PER> __device__ __forceinline__ void load_values(const void *x, int i, int step, int V, float rest, float (&v)[PER]) {
#pragma unroll
    for (int k = 0; k < PER; k += 4, i += step) {
        if (i + 4 <= V) {
            if constexpr (HALF) {
                const h4_any r = *reinterpret_cast<const h4_any *>(static_cast<const uint16_t *>(x) + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[k + e] = h2f(r[e]);
            } else {
                const f4_any r = *reinterpret_cast<const f4_any *>(static_cast<const float *>(x) + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[k + e] = r[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[k + e] = i + e < V ? (HALF ? h2f(static_cast<const uint16_t *>(x)[i + e]) : static_cast<const float *>(x)[i + e]) : rest;
        }
    }
}
template <bool HALF> __device__ __forceinline__ const void *row_of(const VerifyArgs &a, int r) {
    return HALF ? (const void *)(static_cast<const uint16_t *>(a.logits) + (size_t)r * a.ld)
                : (const void *)(static_cast<const float *>(a.logits) + (size_t)r * a.ld);
}
template <bool HALF> __device__ __forceinline__ float value_of(const void *x, int i) {
    return HALF ? h2f(static_cast<const uint16_t *>(x)[i]) : static_cast<const float *>(x)[i];
}

// EACH values of a row from `i` on; behind its end `rest`.
template <bool HALF, int EACH> __device__ __forceinline__ void load_few(const void *x, int i, int V, float rest, float (&v)[EACH]) {
    if constexpr (EACH % 4 == 0) {
        load_values<HALF, EACH>(x, i, 4, V, rest, v);
    } else {
#pragma unroll
        for (int k = 0; k < EACH; ++k) v[k] = i + k < V ? value_of<HALF>(x, i + k) : rest;
    }
}

// (a row's chunks by wave: -1 past the last)
__device__ __forceinline__ int chunk_of(const VerifyArgs &a, int &r) {
    const int blocks = (a.chunks + WAVES - 1) / WAVES;
    r = blockIdx.x / blocks;
    const int c = (blockIdx.x - r * blocks) * WAVES + (threadIdx.x >> 6);
    return c < a.chunks ? c : -1;
}

constexpr int OPEN = -2;  // taken[] of a row that waits for a round's sums

}  // namespace

// One wave a chunk of a row: its maximum (+inf: a NaN or +inf in it) and the sum
// of its weights.
template <bool HALF, int SHIFT> __global__ __launch_bounds__(THREADS) void verify_sums_kernel(VerifyArgs a) {
    constexpr int PER = (1 << SHIFT) / 64;
    __shared__ double table[32];
    const int lane = threadIdx.x & 63;
    int r;
    const int c = chunk_of(a, r);
    float v[PER];
    // (a wave past the last chunk reads nothing: from 0 on, of a row of none)
    load_values<HALF, PER>(row_of<HALF>(a, r), (max(c, 0) << SHIFT) + lane * 4, 256, c < 0 ? 0 : a.V, -INFINITY, v);
    fill_table(table);
    __syncthreads();
    if (c < 0) return;
    float m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        bad = bad || !(v[k] < INFINITY);
        m = fmaxf(m, v[k]);
    }
    m = wave_max(m);
    bad = __any(bad);
    double s = 0.0;
    if (m > -INFINITY && !bad) {
        const Weight w(m, a.per, table);
#pragma unroll
        for (int k = 0; k < PER; ++k) s += w(v[k]);
    }
    s = wave_sum(s);
    if (lane == 0) {
        a.chunk_top[(size_t)r * a.chunks + c] = bad ? INFINITY : m;
        a.chunk_sum[(size_t)r * a.chunks + c] = s;
    }
}

// A round: of the rows that wait, the chunk's sum of max(e - c q, 0).
template <bool HALF, int SHIFT> __global__ __launch_bounds__(THREADS) void verify_round_kernel(VerifyArgs a, int round) {
    constexpr int PER = (1 << SHIFT) / 64;
    __shared__ double table[32];
    const int lane = threadIdx.x & 63;
    int r;
    const int chunk = chunk_of(a, r);
    if (a.taken[r] != OPEN) return;  // (the whole workgroup)
    fill_table(table);
    __syncthreads();
    if (chunk < 0) return;
    const VerifyRow s = a.state[r];
    float v[PER], q[PER];
    load_values<HALF, PER>(row_of<HALF>(a, r), (chunk << SHIFT) + lane * 4, 256, a.V, -INFINITY, v);
    load_values<false, PER>(a.draft + (size_t)r * a.ldp, (chunk << SHIFT) + lane * 4, 256, a.V, 0.0f, q);
    const Weight w(s.m, a.per, table);
    double z = 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k) z += fmax(w(v[k]) - s.c * draft_of(q[k]), 0.0);
    z = wave_sum(z);
    if (lane == 0) a.round_sum[((size_t)round * a.rows + r) * a.chunks + chunk] = z;
}

// One workgroup a row, behind the sums (round 0) or a round: taken[row], the
// child that stays (-1: none, OPEN: one was rejected and its sums are not there),
// and pick[row], the token after the row if the path ends there. In the last
// step no row stays open: further sums are made here, chunk by chunk.
template <bool HALF, int SHIFT> __global__ __launch_bounds__(THREADS) void verify_step_kernel(VerifyArgs a, int round) {
    constexpr int PER = (1 << SHIFT) / 64, EACH = (1 << SHIFT) / THREADS;
    __shared__ double sums[WAVES], table[32];
    __shared__ uint64_t kids[kDraftRows / 64];
    __shared__ int token[kDraftRows];                       // of the children
    __shared__ float accept[kDraftRows], logit[kDraftRows], draft[kDraftRows];
    __shared__ int seq, first_at[WAVES], last_at[WAVES];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (round > 0 && a.taken[r] != OPEN) return;
    const void *x = row_of<HALF>(a, r);

    // what does not depend on anything: loads under way together
    const float *top = a.chunk_top + (size_t)r * a.chunks;
    const double *sum = a.chunk_sum + (size_t)r * a.chunks;
    constexpr int HELD = 5;  // chunks that a lane keeps (a row of up to 320; others are read again)
    float tops[HELD];
    double held[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int c = lane + 64 * k;
        tops[k] = c < a.chunks ? top[c] : -INFINITY;
        held[k] = c < a.chunks ? sum[c] : 0.0;
    }
    const double number = (double)a.sample_u[r];
    int found_seq = -1;
    for (int b = tid; b < a.batch; b += THREADS)
        if (a.row_start[b] <= r && r < a.row_start[b + 1]) found_seq = b;
    fill_table(table);
    if (tid == 0) seq = -1;
    __syncthreads();
    if (found_seq >= 0) atomicMax(&seq, found_seq);
    __syncthreads();

    // ---- its sequence and its children there
    const int start = seq < 0 ? r : max(a.row_start[seq], 0);
    const int n = seq < 0 ? 0 : min(min(a.row_start[seq + 1], a.rows) - start, a.max_rows), t = r - start;
    float m = -INFINITY;  // (+inf where the row cannot be judged)
#pragma unroll
    for (int k = 0; k < HELD; ++k) m = fmaxf(m, tops[k]);
    for (int c = lane + 64 * HELD; c < a.chunks; c += 64) m = fmaxf(m, top[c]);
    m = wave_max(m);
    if (t >= n || !(m > -INFINITY && m < INFINITY)) {
        if (tid == 0) {
            a.pick[r] = -1;
            a.taken[r] = -1;
        }
        return;
    }
    const int words = (n + 63) >> 6;
    for (int w = wave; w < words; w += WAVES) {
        const int i = w * 64 + lane;
        const int at = start + min(i, n - 1), tok = a.tokens[at];
        const float u = a.draft ? a.accept_u[at] : 0.0f;
        const bool kid = i < n && i > t && a.parents[at] == t && tok >= 0 && tok < a.V;
        if (kid) {
            token[i] = tok;
            if (a.draft) {
                accept[i] = u;
                logit[i] = value_of<HALF>(x, tok);
                draft[i] = a.draft[(size_t)r * a.ldp + tok];
            }
        }
        const uint64_t bits = __ballot(kid);
        if (lane == 0) kids[w] = bits;
    }

    // ---- the sum of its weights (each wave for itself, in one order)
    const Weight weight(m, a.per, table);
    double total = 0.0;
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        if (64 * k >= a.chunks) break;
        held[k] *= weight(tops[k]);
        total += held[k];
    }
    for (int c = lane + 64 * HELD; c < a.chunks; c += 64) total += sum[c] * weight(top[c]);
    total = wave_sum(total);
    __syncthreads();

    // ---- the tests
    int taken = -1, pick = -1;
    double c = 0.0, z = total;  // times the sum of weights
    const double *left = nullptr;  // the chunks' sums of max(e - c q, 0) (null: of e)
    if (a.draft) {
        int rejected = 0;
        auto join = [&](const double *p) {
            double v = 0.0;
            for (int i = lane; i < a.chunks; i += 64) v += p[i];
            left = p;
            return wave_sum(v);
        };
        int from = 0;  // the first child not tested yet
        if (round > 0) {
            const VerifyRow s = a.state[r];
            c = s.c;
            from = s.child + 1;
            rejected = round;
            z = join(a.round_sum + ((size_t)(round - 1) * a.rows + r) * a.chunks);
        }
        for (int w = from >> 6; w < words && taken < 0; ++w) {
            uint64_t k = kids[w];
            if (w == from >> 6) k &= ~0ull << (from & 63);
            for (; k; k &= k - 1) {
                const int child = w * 64 + __ffsll((unsigned long long)k) - 1;
                const double q = draft_of(draft[child]), e = weight(logit[child]), rest = rejected ? fmax(e - c * q, 0.0) : e;
                if ((double)accept[child] * q * z < rest) {
                    taken = child;
                    break;
                }
                c += z;
                ++rejected;
                if (rejected <= a.rounds) {
                    __syncthreads();  // (every wave has read what the round before left)
                    if (tid == 0) {
                        a.state[r] = VerifyRow{c, m, child};
                        a.taken[r] = OPEN;
                    }
                    return;
                }
                double *own = a.round_sum + ((size_t)a.rounds * a.rows + r) * a.chunks;
                for (int i = wave; i < a.chunks; i += WAVES) {
                    float v[PER], p[PER];
                    load_values<HALF, PER>(x, (i << SHIFT) + lane * 4, 256, a.V, -INFINITY, v);
                    load_values<false, PER>(a.draft + (size_t)r * a.ldp, (i << SHIFT) + lane * 4, 256, a.V, 0.0f, p);
                    double s = 0.0;
#pragma unroll
                    for (int j = 0; j < PER; ++j) s += fmax(weight(v[j]) - c * draft_of(p[j]), 0.0);
                    s = wave_sum(s);
                    if (lane == 0) own[i] = s;
                }
                __syncthreads();  // (of this workgroup's own stores too)
                z = join(own);
                __syncthreads();
            }
        }
        if (!(z > 0.0)) {  // nothing is left of p: p itself
            c = 0.0;
            z = total;
            left = nullptr;
        }
    }

    // ---- the token by the inverse of the cumulated weights
    if (taken < 0) {
        const double want = number * z;
        double before = 0.0, ahead = 0.0;  // sums of earlier chunks: than the next 64, than the one chosen
        int chunk = -1, last = 0;
        double last_ahead = 0.0;
        auto look = [&](int base, double v) {  // at 64 chunks' sums
            const double run = wave_scan(v);
            const uint64_t over = __ballot(v > 0.0 && before + run > want), some = __ballot(v > 0.0);
            const int at = over ? __ffsll((unsigned long long)over) - 1 : some ? 63 - __clzll((long long)some) : 0;
            const double prior = before + (at ? lane_value(run, at - 1) : 0.0);
            if (over) {
                chunk = base + at;
                ahead = prior;
            } else if (some) {
                last = base + at;
                last_ahead = prior;
            }
            before += lane_value(run, 63);
        };
        if (!left) {
#pragma unroll
            for (int k = 0; k < HELD; ++k)
                if (chunk < 0 && 64 * k < a.chunks) look(64 * k, held[k]);
        }
        for (int base = left ? 0 : 64 * HELD; base < a.chunks && chunk < 0; base += 64) {
            const int i = base + lane;
            look(base, i < a.chunks ? (left ? left[i] : sum[i] * weight(top[i])) : 0.0);
        }
        if (chunk < 0) {  // (the numbers' last bits)
            chunk = last;
            ahead = last_ahead;
        }
        // EACH values in a row a thread
        const int first = (chunk << SHIFT) + tid * EACH;
        float v[EACH], p[EACH];
        load_few<HALF, EACH>(x, first, a.V, -INFINITY, v);
        if (c > 0.0) load_few<false, EACH>(a.draft + (size_t)r * a.ldp, first, a.V, 0.0f, p);
        double w[EACH], mine = 0.0;
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            w[k] = weight(v[k]);
            if (c > 0.0) w[k] = fmax(w[k] - c * draft_of(p[k]), 0.0);
            mine += w[k];
        }
        const double run = wave_scan(mine);
        if (lane == 63) sums[wave] = run;
        __syncthreads();
        double at = ahead + (run - mine);
        for (int v = 0; v < wave; ++v) at += sums[v];
        int found = INT_MAX, some = -1;
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            at += w[k];
            if (w[k] > 0.0) {
                some = first + k;
                if (at > want && found == INT_MAX) found = first + k;
            }
        }
        // (the values ascend with the lanes and waves)
        const uint64_t over = __ballot(found != INT_MAX), any = __ballot(some >= 0);
        if (lane == 0) {
            first_at[wave] = INT_MAX;
            last_at[wave] = -1;
        }
        if (over && lane == __ffsll((unsigned long long)over) - 1) first_at[wave] = found;
        if (any && lane == 63 - __clzll((long long)any)) last_at[wave] = some;
        __syncthreads();
        int last_value = -1;
        pick = INT_MAX;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            pick = min(pick, first_at[w]);
            last_value = max(last_value, last_at[w]);
        }
        if (pick == INT_MAX) pick = last_value;
        if (!a.draft)  // the first child that has the token
            for (int w = 0; w < words && taken < 0; ++w)
                for (uint64_t k = kids[w]; k; k &= k - 1) {
                    const int child = w * 64 + __ffsll((unsigned long long)k) - 1;
                    if (token[child] == pick) {
                        taken = child;
                        break;
                    }
                }
    }
    if (tid == 0) {
        a.pick[r] = pick;
        a.taken[r] = taken;
    }
}

// One wave a sequence follows its path.
__global__ __launch_bounds__(64) void verify_path_kernel(VerifyArgs a) {
    __shared__ int taken[kDraftRows];
    const int b = blockIdx.x, lane = threadIdx.x;
    const int start = min(max(a.row_start[b], 0), a.rows), end = min(max(a.row_start[b + 1], start), a.rows);
    const int n = min(end - start, a.max_rows);
    for (int i = lane; i < n; i += 64) taken[i] = a.taken[start + i];
    __syncthreads();
    int32_t *path = a.path + (size_t)b * a.max_rows;
    int count = 0, at = n > 0 ? 0 : -1, last = -1;
    while (at >= 0) {
        if (lane == 0) path[count] = at;
        ++count;
        last = at;
        const int to = taken[at];
        at = to > at && to < n ? to : -1;  // (a row that no sequence claimed holds anything)
    }
    for (int i = count + lane; i < a.max_rows; i += 64) path[i] = -1;
    if (lane == 0) {
        a.accepted[b] = count;
        a.next[b] = last < 0 ? -1 : a.pick[start + last];
    }
}

// Chunks of 2^11 values where those of all rows fill the chip (a wave each, 16 a
// CU), else of 2^9.
int verify_shift(int64_t rows, int64_t V) { return rows * ((V + 2047) >> 11) >= 4096 ? LARGE : SMALL; }
int verify_chunks(int64_t rows, int64_t V) {
    const int s = verify_shift(rows, V);
    return (int)((V + (1 << s) - 1) >> s);
}
// The most (row, chunk) pairs of up to `rows` rows of up to V values: small
// chunks are taken up to four times 4095 of them.
int64_t verify_pairs_most(int64_t rows, int64_t V) {
    const int64_t large = rows * ((V + 2047) >> 11), small = rows * ((V + 511) >> 9);
    const int64_t s = small < 4 * 4095 ? small : 4 * 4095;
    return large > s ? large : s;
}

template <bool HALF, int SHIFT> static hipError_t launch(const VerifyArgs &a, hipStream_t st) {
    const unsigned grid = (unsigned)a.rows * ((a.chunks + WAVES - 1) / WAVES);
    verify_sums_kernel<HALF, SHIFT><<<grid, THREADS, 0, st>>>(a);
    verify_step_kernel<HALF, SHIFT><<<a.rows, THREADS, 0, st>>>(a, 0);
    for (int round = 0; round < a.rounds; ++round) {
        verify_round_kernel<HALF, SHIFT><<<grid, THREADS, 0, st>>>(a, round);
        verify_step_kernel<HALF, SHIFT><<<a.rows, THREADS, 0, st>>>(a, round + 1);
    }
    return hipGetLastError();
}

hipError_t launch_verify_drafts(const VerifyArgs &a, bool half, hipStream_t st) {
    if (a.rows) {
        const bool large = verify_shift(a.rows, a.V) == LARGE;
        const hipError_t e = half ? (large ? launch<true, LARGE>(a, st) : launch<true, SMALL>(a, st))
                                  : (large ? launch<false, LARGE>(a, st) : launch<false, SMALL>(a, st));
        if (e != hipSuccess) return e;
    }
    verify_path_kernel<<<a.batch, 64, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace q3vl
