// rows.hip -- what a step over several rows of tokens needs ahead of its
// attention: the plan of its drafts, and the head norms with the rotary
// position and the cache stores. gfx950.
#include "q3vl_device.hpp"
#include "q3vl_kernels.hpp"

namespace q3vl {

// ---------------------------------------------------------------- draft plan
// One block per sequence, and one for the rows behind the last. Row t's mask
// is its own bit and its ancestors'. Pointer doubling: with up[t] an ancestor
// of t (at first its parent) and mask[t] holding the ancestors from t to just
// above up[t], one turn sets mask[t] |= mask[up[t]], up[t] = up[up[t]], so
// ceil(log2(depth + 1)) turns do. up is -1 past a root and -2 past a parent
// that no row can have, which its descendants inherit.
//
// up is double-buffered; the masks are not: a turn that reads mask[up[t]]
// after its owner's update finds more ancestors of t in it, never others, and
// never fewer than the old mask had. Depth is the mask's bit count less one.
__global__ __launch_bounds__(1024) void draft_plan_kernel(const int32_t *parents, const int32_t *row_start,
                                                          const int32_t *cache_len, const int32_t *pos_delta,
                                                          int batch, int rows, int max_rows, int max_seq,
                                                          uint64_t *mask, int words, int32_t *pos, int64_t *slots) {
    extern __shared__ __align__(16) unsigned char smem[];
    const int b = blockIdx.x, tid = threadIdx.x, nt = blockDim.x;
    const int start = min(max(row_start[b], 0), rows);
    if (b == batch) {  // rows that hold no token
        for (int r = start + tid; r < rows; r += nt) {
            pos[r] = -1;
            slots[r] = -1;
        }
        for (size_t i = (size_t)start * words + tid; i < (size_t)rows * words; i += nt) mask[i] = 0;
        return;
    }
    const int end = min(max(row_start[b + 1], start), rows);
    const int n = min(end - start, max_rows);
    const int wn = (n + 63) >> 6;  // words that n rows can set
    uint64_t *m = reinterpret_cast<uint64_t *>(smem);                        // [n][wn]
    int16_t *up = reinterpret_cast<int16_t *>(smem + (size_t)n * wn * 8);  // [2][n]
    for (int t = tid; t < n; t += nt) {
        const int p = parents[start + t];
        up[t] = (int16_t)(p >= -1 && p < t ? p : -2);
    }
    for (int i = tid; i < n * wn; i += nt) {
        const int t = i / wn, w = i - t * wn;
        m[i] = w == t >> 6 ? 1ull << (t & 63) : 0;
    }
    for (int turn = 0;; turn ^= 1) {
        const int16_t *u = up + turn * n;
        int16_t *next = up + (turn ^ 1) * n;
        int more = 0;
        __syncthreads();  // up and the masks of the last turn are written
        for (int t = tid; t < n; t += nt) {
            const int p = u[t], q = p >= 0 ? u[p] : p;
            next[t] = (int16_t)q;
            more |= q >= 0;
        }
        for (int i = tid; i < n * wn; i += nt) {
            const int t = i / wn, w = i - t * wn, p = u[t];
            if (p >= 0 && w <= p >> 6) m[i] |= m[p * wn + w];
        }
        if (!__syncthreads_or(more)) {
            up = next;
            break;
        }
    }
    // (past the last turn's barrier: every mask is whole)
    const int len = cache_len[b];
    const int64_t base = (int64_t)len + (pos_delta ? pos_delta[b] : 0);
    for (int t = tid; t < end - start; t += nt) {
        const size_t r = (size_t)start + t;
        int64_t at = -2, slot = -1;
        if (t < n && up[t] == -1 && len >= 0 && (int64_t)len + t < max_seq) {
            at = base - 1;
            for (int w = 0; w < wn; ++w) at += __popcll(m[t * wn + w]);
            if (at < 0 || at > 0x7fffffff) at = -2;
            else slot = (int64_t)b * max_seq + len + t;
        }
        pos[r] = (int32_t)at;
        slots[r] = slot;
        for (int w = 0; w < words; ++w) mask[r * words + w] = slot >= 0 && w < wn ? m[t * wn + w] : 0;
    }
}

hipError_t launch_draft_plan(const int32_t *parents, const int32_t *row_start, const int32_t *cache_len,
                             const int32_t *pos_delta, int batch, int rows, int max_rows, int max_seq, uint64_t *mask,
                             int words, int32_t *pos, int64_t *slots, hipStream_t st) {
    const int n = max_rows < rows ? max_rows : rows;
    const size_t lds = (size_t)n * ((n + 63) / 64) * 8 + (size_t)n * 4;
    static_assert(kDraftRows * (kDraftRows / 64) * 8 + kDraftRows * 4 <= 160 * 1024, "LDS");
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(draft_plan_kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    const int threads = n <= 64 ? 64 : n <= 256 ? 256 : 1024;
    draft_plan_kernel<<<batch + 1, threads, lds, st>>>(parents, row_start, cache_len, pos_delta, batch, rows, n, max_seq,
                                                       mask, words, pos, slots);
    return hipGetLastError();
}

// ------------------------------------------------- head norms, rotation, cache
// Four lanes a head: lane j of the quad holds x[8m + 2j] and x[8m + 2j + 1] for
// m = 0 .. D/8 - 1. The reference's sum of squares (8 chains, chain c over
// x[c], x[c+8], ..., folded left to right) then runs as two chains a lane with
// no exchange before the fold, and the pair (x_i, x_{i + D/2}) that the
// rotation mixes lies in one lane. A wave takes 16 heads of one row, counted q,
// k, v.
#define Q3VL_QUADB(v, j) \
    __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), (j) * 0x55, 0xF, 0xF, true))

template <int D, bool HALF, bool AXES3>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkRopeArgs a) {
    constexpr int M = D / 8, MH = M / 2;
    const int lane = threadIdx.x & 63, j = lane & 3;
    const int per_row = (a.heads + 2 * a.kv_heads + 15) >> 4;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t row = unit / per_row;
    if (row >= a.rows) return;
    const int head = (int)(unit - row * per_row) * 16 + (lane >> 2);
    if (head >= a.heads + 2 * a.kv_heads) return;  // (whole quads)
    const int32_t *pr = a.pos + row * (AXES3 ? 3 : 1);
    const int p0 = pr[0];
    if (p0 == -1) return;
    bool ok = p0 >= 0 && p0 < a.table_rows;
    int p1 = p0, p2 = p0;
    if constexpr (AXES3) {
        p1 = pr[1];
        p2 = pr[2];
        ok = ok && p1 >= 0 && p1 < a.table_rows && p2 >= 0 && p2 < a.table_rows;
    }
    const int64_t slot = a.slots[row];
    const bool kept = ok && slot >= 0 && slot < (int64_t)a.batch * a.max_seq;
    const bool is_q = head < a.heads, is_k = !is_q && head < a.heads + a.kv_heads;
    const int h = is_q ? head : head - a.heads - (is_k ? 0 : a.kv_heads);
    const size_t at = kept ? (size_t)(slot / a.max_seq) * a.seq_stride + (size_t)h * a.head_stride +
                                 (size_t)(slot % a.max_seq) * a.row_stride
                           : 0;
    const float *x = (is_q ? a.q + row * a.ldq : is_k ? a.k + row * a.ldk : a.v + row * a.ldv) + (size_t)h * D + 2 * j;
    if (!is_q && !kept) return;
    float2 v[M];
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] = make_float2(x[8 * m], x[8 * m + 1]);
    if (!is_q && !is_k) {
        uint16_t *o = a.v_cache + at + 2 * j;
#pragma unroll
        for (int m = 0; m < M; ++m) *reinterpret_cast<uint32_t *>(o + 8 * m) = f2h(v[m].x) | (uint32_t)f2h(v[m].y) << 16;
        return;
    }
    const int8_t *w = is_q ? a.q_w : a.k_w;
    const float *ws = is_q ? a.q_s : a.k_s;
    float c0 = 0.0f, c1 = 0.0f;
#pragma unroll
    for (int m = 0; m < M; ++m) {
        c0 = fmaf(v[m].x, v[m].x, c0);
        c1 = fmaf(v[m].y, v[m].y, c1);
    }
    float ss = Q3VL_QUADB(c0, 0) + Q3VL_QUADB(c1, 0);
    ss = (ss + Q3VL_QUADB(c0, 1)) + Q3VL_QUADB(c1, 1);
    ss = (ss + Q3VL_QUADB(c0, 2)) + Q3VL_QUADB(c1, 2);
    ss = (ss + Q3VL_QUADB(c0, 3)) + Q3VL_QUADB(c1, 3);
    const float inv = rcp_rn(sqrt_rn(ss * (1.0f / D) + a.eps));
    auto turn = [&](float lo, float hi, int i, float &olo, float &ohi) {
        int p = p0;
        if constexpr (AXES3) {
            if (a.interleaved) {
                const int ax = i % 3;
                p = ax == 1 && i < 3 * a.sec1 ? p1 : ax == 2 && i < 3 * a.sec2 ? p2 : p0;
            } else {
                p = i < a.sec0 ? p0 : i < a.sec0 + a.sec1 ? p1 : p2;
            }
        }
        const float c = ok ? a.cos[(size_t)p * (D / 2) + i] : __builtin_nanf("");
        const float s = ok ? a.sin[(size_t)p * (D / 2) + i] : __builtin_nanf("");
        const float y = (float)w[i] * ((ws[i / a.gs] * inv) * lo);
        const float z = (float)w[i + D / 2] * ((ws[(i + D / 2) / a.gs] * inv) * hi);
        olo = fmaf(y, c, -(z * s));
        ohi = fmaf(y, s, z * c);
    };
#pragma unroll
    for (int m = 0; m < MH; ++m) {
        const int i = 8 * m + 2 * j;
        float2 lo, hi;
        turn(v[m].x, v[m + MH].x, i, lo.x, hi.x);
        turn(v[m].y, v[m + MH].y, i + 1, lo.y, hi.y);
        v[m] = lo;
        v[m + MH] = hi;
    }
    if (is_q && !HALF) {
        float *o = static_cast<float *>(a.q_out) + row * a.ldo + (size_t)h * D + 2 * j;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            o[8 * m] = v[m].x;
            o[8 * m + 1] = v[m].y;
        }
    } else {
        uint16_t *o = is_q ? static_cast<uint16_t *>(a.q_out) + row * a.ldo + (size_t)h * D + 2 * j : a.k_cache + at + 2 * j;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            o[8 * m] = f2h(v[m].x);
            o[8 * m + 1] = f2h(v[m].y);
        }
    }
}

hipError_t launch_qk_norm_rope(const QkRopeArgs &a, int head_dim, bool half, int axes, hipStream_t st) {
    const int64_t per_row = (a.heads + 2 * a.kv_heads + 15) / 16;
    const unsigned grid = (unsigned)((a.rows * per_row + 3) / 4);
    auto go = [&](auto kernel) {
        kernel<<<grid, 256, 0, st>>>(a);
        return hipGetLastError();
    };
    if (head_dim == 128) {
        if (axes == 3) return half ? go(qk_norm_rope_kernel<128, true, true>) : go(qk_norm_rope_kernel<128, false, true>);
        return half ? go(qk_norm_rope_kernel<128, true, false>) : go(qk_norm_rope_kernel<128, false, false>);
    }
    if (axes == 3) return half ? go(qk_norm_rope_kernel<64, true, true>) : go(qk_norm_rope_kernel<64, false, true>);
    return half ? go(qk_norm_rope_kernel<64, true, false>) : go(qk_norm_rope_kernel<64, false, false>);
}

}  // namespace q3vl
