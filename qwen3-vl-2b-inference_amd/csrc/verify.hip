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
#include "q3vl_device.hpp"
#include "q3vl_kernels.hpp"

namespace q3vl {

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr double FAR = -700.0;  // (x - m) / T below which a weight is 0

struct Scratch {
    double sum[WAVES];
    float top[WAVES];
    int bad[WAVES];
    int at[WAVES];
    uint64_t kids[kDraftRows / 64];
    int child;
};

__device__ __forceinline__ double block_sum(double v, Scratch &sh) {
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) v += __shfl_xor(v, k);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.sum[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < WAVES; ++w) s += sh.sum[w];
    return s;
}

template <bool HALF> struct Row {
    const void *x;
    const float *q;  // or null
    float m;
    double inv_t;
    __device__ __forceinline__ float logit(int i) const {
        return HALF ? h2f(static_cast<const uint16_t *>(x)[i]) : static_cast<const float *>(x)[i];
    }
    __device__ __forceinline__ double e(int i) const {  // p times its sum
        const double d = ((double)logit(i) - (double)m) * inv_t;
        return d >= FAR ? exp(d) : 0.0;
    }
    __device__ __forceinline__ double draft(int i) const {
        const float v = q[i];
        return v > 0.0f ? (double)v : 0.0;
    }
    // p - c q, times p's sum
    __device__ __forceinline__ double w(int i, double c) const {
        double v = e(i);
        if (c > 0.0) v = fmax(v - c * draft(i), 0.0);
        return v;
    }
};

}  // namespace

// One workgroup a row: pick[row] the token after it if the path ends there,
// taken[row] the child that stays (-1: none).
template <bool HALF> __global__ __launch_bounds__(THREADS) void verify_row_kernel(VerifyArgs a) {
    __shared__ Scratch sh;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // the row's sequence
    int b = 0;
    {
        int lo = 0, hi = a.batch;  // the last b with row_start[b] <= r
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (a.row_start[mid] <= r) lo = mid;
            else hi = mid;
        }
        b = lo;
    }
    const int start = max(a.row_start[b], 0), end = min(max(a.row_start[b + 1], start), a.rows);
    const int n = min(end - start, a.max_rows), t = r - start;
    if (t < 0 || t >= n) return;
    Row<HALF> row;
    row.x = HALF ? (const void *)(static_cast<const uint16_t *>(a.logits) + (size_t)r * a.ld)
                 : (const void *)(static_cast<const float *>(a.logits) + (size_t)r * a.ld);
    row.q = a.draft ? a.draft + (size_t)r * a.ldp : nullptr;
    row.inv_t = a.inv_t;
    float top = -INFINITY;
    bool bad = false;
    for (int i = tid; i < a.V; i += THREADS) {
        const float x = row.logit(i);
        bad = bad || !(x < INFINITY);
        top = fmaxf(top, x);
    }
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
    const bool any_bad = __any(bad);
    if (lane == 0) {
        sh.top[wave] = top;
        sh.bad[wave] = any_bad;
    }
    __syncthreads();
    bad = false;
    for (int w = 0; w < WAVES; ++w) {
        top = fmaxf(top, sh.top[w]);
        bad = bad || sh.bad[w];
    }
    if (bad || top == -INFINITY) {
        if (tid == 0) {
            a.pick[r] = -1;
            a.taken[r] = -1;
        }
        return;
    }
    row.m = top;
    const uint64_t kid = __ballot(tid < n && tid > t && a.parents[start + min(tid, n - 1)] == t);
    if (lane == 0) sh.kids[wave] = kid;
    double s = 0.0;
    for (int i = tid; i < a.V; i += THREADS) s += row.e(i);
    const double total = block_sum(s, sh);  // (its barriers stand between kids' write and reads too)
    double c = 0.0, z = total;              // c and Z, times p's sum
    int taken = -1;
    if (row.q) {
        for (int w = 0; w < WAVES && taken < 0; ++w)
            for (uint64_t k = sh.kids[w]; k; k &= k - 1) {
                const int child = w * 64 + __ffsll((unsigned long long)k) - 1;
                const int tok = a.tokens[start + child];
                if (tok < 0 || tok >= a.V) continue;
                if ((double)a.accept_u[start + child] * row.draft(tok) * z < row.w(tok, c)) {
                    taken = child;
                    break;
                }
                c += z;
                s = 0.0;
                for (int i = tid; i < a.V; i += THREADS) s += row.w(i, c);
                z = block_sum(s, sh);
            }
        if (!(z > 0.0)) {
            c = 0.0;
            z = total;
        }
    }
    int pick = -1;
    if (taken < 0) {
        // the token by the inverse of the cumulated weights, chunk by chunk
        const double want = (double)a.sample_u[r] * z;
        double before = 0.0;
        int last = -1;  // the last value with a weight
        for (int base = 0; base < a.V && pick < 0; base += THREADS) {
            const int i = base + tid;
            const double v = i < a.V ? row.w(i, c) : 0.0;
            double run = v;  // inclusive within the wave
#pragma unroll
            for (int k = 1; k < 64; k <<= 1) {
                const double o = __shfl_up(run, k);
                if (lane >= k) run += o;
            }
            __syncthreads();
            if (lane == 63) sh.sum[wave] = run;
            __syncthreads();
            double ahead = before;
            for (int w = 0; w < WAVES; ++w) {
                if (w < wave) ahead += sh.sum[w];
                before += sh.sum[w];
            }
            const uint64_t over = __ballot(v > 0.0 && ahead + run > want), some = __ballot(v > 0.0);
            __syncthreads();
            if (lane == 0) {
                sh.at[wave] = over ? base + wave * 64 + __ffsll((unsigned long long)over) - 1 : -1;
                sh.bad[wave] = some ? base + wave * 64 + 63 - __clzll((long long)some) : -1;
            }
            __syncthreads();
            for (int w = WAVES - 1; w >= 0; --w) {
                if (sh.at[w] >= 0) pick = sh.at[w];
                last = max(last, sh.bad[w]);
            }
        }
        if (pick < 0) pick = last;
        if (!row.q) {
            for (int w = 0; w < WAVES && taken < 0; ++w)
                for (uint64_t k = sh.kids[w]; k; k &= k - 1) {
                    const int child = w * 64 + __ffsll((unsigned long long)k) - 1;
                    if (a.tokens[start + child] == pick) {
                        taken = child;
                        break;
                    }
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
    const int b = blockIdx.x, lane = threadIdx.x;
    const int start = min(max(a.row_start[b], 0), a.rows), end = min(max(a.row_start[b + 1], start), a.rows);
    const int n = min(end - start, a.max_rows);
    int32_t *path = a.path + (size_t)b * a.max_rows;
    int count = 0, at = n > 0 ? 0 : -1, next = -1;
    while (at >= 0) {
        if (lane == 0) path[count] = at;
        ++count;
        next = a.pick[start + at];
        const int to = a.taken[start + at];
        at = to > at && to < n ? to : -1;  // (a row that no sequence claimed holds anything)
    }
    for (int i = count + lane; i < a.max_rows; i += 64) path[i] = -1;
    if (lane == 0) {
        a.accepted[b] = count;
        a.next[b] = next;
    }
}

hipError_t launch_verify_drafts(const VerifyArgs &a, bool half, hipStream_t st) {
    if (a.rows) {
        if (half) verify_row_kernel<true><<<a.rows, THREADS, 0, st>>>(a);
        else verify_row_kernel<false><<<a.rows, THREADS, 0, st>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    verify_path_kernel<<<a.batch, 64, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace q3vl
