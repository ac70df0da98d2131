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
//
// Bound by latency: 8 sequences of 32 rows 4.2 us, 96 of 500 8.9 us.
__global__ __launch_bounds__(1024) void draft_plan_kernel(const int32_t *parents, const int32_t *row_start,
                                                          const int32_t *cache_len, const int32_t *pos_delta,
                                                          int batch, int rows, int max_rows, int max_seq,
                                                          uint64_t *mask, int words, int32_t *pos, int64_t *slots) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int more[16];  // per turn: whether some row has ancestors left
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
    const int end = min(max(row_start[b + 1], start), rows), len = cache_len[b];
    const int64_t base = (int64_t)len + (pos_delta ? pos_delta[b] : 0);
    const int n = min(end - start, max_rows);
    const int wn = (n + 63) >> 6;  // words that n rows can set
    const int ws = wn > 1 ? 32 - __builtin_clz(wn - 1) : 0, wm = (1 << ws) - 1;  // (row, word) items by shifts
    uint64_t *m = reinterpret_cast<uint64_t *>(smem);                        // [n][wn]
    int16_t *up = reinterpret_cast<int16_t *>(smem + (size_t)n * wn * 8);  // [2][n]
    if (tid < 16) more[tid] = 0;
    for (int t = tid; t < n; t += nt) {
        const int p = parents[start + t];
        up[t] = (int16_t)(p >= -1 && p < t ? p : -2);
    }
    for (int i = tid; i < n << ws; i += nt) {
        const int t = i >> ws, w = i & wm;
        if (w < wn) m[t * wn + w] = w == t >> 6 ? 1ull << (t & 63) : 0;
    }
    __syncthreads();
    for (int turn = 0;; ++turn) {  // (12 at most: each doubles what is covered)
        const int16_t *u = up + (turn & 1) * n;
        int16_t *next = up + (~turn & 1) * n;
        bool again = false;
        for (int t = tid; t < n; t += nt) {
            const int p = u[t], q = p >= 0 ? u[p] : p;
            next[t] = (int16_t)q;
            again = again || q >= 0;
        }
        for (int i = tid; i < n << ws; i += nt) {
            const int t = i >> ws, w = i & wm, p = u[t];
            if (p >= 0 && w <= p >> 6) m[t * wn + w] |= m[p * wn + w];
        }
        if (again) more[turn] = 1;
        __syncthreads();
        if (!more[turn]) {
            up = next;
            break;
        }
    }
    // (past the last turn's barrier: every mask is whole)
    int16_t *done = up == reinterpret_cast<int16_t *>(m + (size_t)n * wn) ? up + n : up - n;  // (the other buffer)
    for (int t = tid; t < end - start; t += nt) {
        int64_t at = -2, slot = -1;
        if (t < n && up[t] == -1 && len >= 0 && (int64_t)len + t < max_seq) {
            at = base - 1;
            for (int w = 0; w <= t >> 6; ++w) at += __popcll(m[t * wn + w]);
            if (at < 0 || at > 0x7fffffff) at = -2;
            else slot = (int64_t)b * max_seq + len + t;
        }
        pos[start + t] = (int32_t)at;
        slots[start + t] = slot;
        if (t < n) done[t] = slot >= 0;
    }
    __syncthreads();
    const int64_t left = (int64_t)(end - start) * words;
    uint64_t *out = mask + (size_t)start * words;
    if (words == wn && n == end - start && ws >= 0 && wm + 1 == wn) {  // a row's words are what LDS holds
        for (int i = tid; i < n << ws; i += nt) out[i] = done[i >> ws] ? m[i] : 0;
        return;
    }
    for (int64_t i = tid; i < left; i += nt) {
        const int t = (int)(i / words), w = (int)(i - (int64_t)t * words);
        out[i] = t < n && w < wn && done[t] ? m[t * wn + w] : 0;
    }
}

hipError_t launch_draft_plan(const int32_t *parents, const int32_t *row_start, const int32_t *cache_len,
                             const int32_t *pos_delta, int batch, int rows, int max_rows, int max_seq, uint64_t *mask,
                             int words, int32_t *pos, int64_t *slots, hipStream_t st) {
    const int n = max_rows < rows ? max_rows : rows;
    const size_t lds = (size_t)n * ((n + 63) / 64) * 8 + (size_t)n * 4;
    constexpr int most = kDraftRows * (kDraftRows / 64) * 8 + kDraftRows * 4;
    static_assert(most <= 160 * 1024, "LDS");
    if (lds > 64 * 1024) {
        const hipError_t e = allow_lds<&draft_plan_kernel>(most);
        if (e != hipSuccess) return e;
    }
    const int threads = n <= 64 ? 64 : n <= 256 ? 256 : 1024;
    draft_plan_kernel<<<batch + 1, threads, lds, st>>>(parents, row_start, cache_len, pos_delta, batch, rows, n, max_seq,
                                                       mask, words, pos, slots);
    return hipGetLastError();
}

// ------------------------------------------------- head norms, rotation, cache
// Four lanes a head: lane j of the quad holds x[16 q + 4 j + e], q = 0 .. D/16 -
// 1, e = 0 .. 3, so that a quad reads and writes 64 bytes in one piece, and the
// pair (x_i, x_{i + D/2}) that the rotation mixes lies in one lane. A wave takes
// 16 heads of one row, counted q, k, v.
//
// The sum of squares keeps the reference's order (chain c = 0 .. 7 over x[c],
// x[c + 8], ..., folded left to right): lanes j and j ^ 2 each hold half of the
// same four chains, exchange their values and run all of them.
//
// Bound by HBM: 8 D bytes a query head in and out, 6 D a key or value head.
// 4999 rows of 16 + 8 + 8 heads with three positions: 29.3 us again and again,
// 37.8 a call on other data each time; pairs of two values a lane (32-byte
// pieces, no exchange) took 65.8 where this took 28.4.
#define Q3VL_QUADP(v, ctrl) \
    __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), ctrl, 0xF, 0xF, true))

typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));      // rows of any stride
typedef uint16_t h4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint16_t h4_row __attribute__((ext_vector_type(4)));

template <int D, bool HALF, bool AXES3>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const float *q_p, const float *k_p, const float *v_p,
                                                           const int32_t *pos_p, const int64_t *slots_p, int heads_p,
                                                           int kv_heads_p, int gs_p, int rows_p, QkRopeArgs args) {
    QkRopeArgs a = args;  // (the leading arguments arrive in registers)
    a.q = q_p;
    a.k = k_p;
    a.v = v_p;
    a.pos = pos_p;
    a.slots = slots_p;
    a.heads = heads_p;
    a.kv_heads = kv_heads_p;
    a.gs = gs_p;
    a.rows = rows_p;
    constexpr int Q = D / 16, QH = Q / 2;
    __shared__ __align__(16) float wsh[2][D], ssh[2][D];  // norm weights and their scales, q and k
    const int lane = threadIdx.x & 63, j = lane & 3;
    const int per_row = (a.heads + 2 * a.kv_heads + 15) >> 4;
    const int64_t units = a.rows * per_row, stride = (int64_t)gridDim.x * 4;
    int64_t unit = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (threadIdx.x < D) {
        const int d = threadIdx.x, g = d / a.gs;
        wsh[0][d] = (float)a.q_w[d];
        wsh[1][d] = (float)a.k_w[d];
        ssh[0][d] = a.q_s[g];
        ssh[1][d] = a.k_s[g];
    }
    int axes[QH];  // AXES3: this lane's frequencies' axes, two bits each
    if constexpr (AXES3) {
#pragma unroll
        for (int q = 0; q < QH; ++q) {
            axes[q] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 16 * q + 4 * j + e, r = i % 3;
                const int ax = a.interleaved ? (r == 1 && i < 3 * a.sec1 ? 1 : r == 2 && i < 3 * a.sec2 ? 2 : 0)
                                             : (i < a.sec0 ? 0 : i < a.sec0 + a.sec1 ? 1 : 2);
                axes[q] |= ax << (2 * e);
            }
        }
    }
    __syncthreads();
    for (; unit < units; unit += stride) {
        const int64_t row = (uint32_t)unit / (uint32_t)per_row;  // (units fit 31 bits)
        const int head = (int)(unit - row * per_row) * 16 + (lane >> 2);
        const int32_t *pr = a.pos + row * (AXES3 ? 3 : 1);
        const int p0 = pr[0];
        if (p0 == -1 || head >= a.heads + 2 * a.kv_heads) continue;  // (whole quads)
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
        if (!is_q && !kept) continue;
        const int h = is_q ? head : head - a.heads - (is_k ? 0 : a.kv_heads);
        const float *x = (is_q ? a.q + row * a.ldq : is_k ? a.k + row * a.ldk : a.v + row * a.ldv) + (size_t)h * D + 4 * j;
        float v[Q][4];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const f4_any r = *reinterpret_cast<const f4_any *>(x + 16 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] = r[e];
        }
        if (is_q || is_k) {
            // the rotation's factors (a NaN row where a position is past the tables)
            float c[QH][4], n[QH][4];
#pragma unroll
            for (int q = 0; q < QH; ++q) {
                const int i = 16 * q + 4 * j;
                if constexpr (AXES3) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int ax = axes[q] >> (2 * e) & 3, p = ok ? (ax == 0 ? p0 : ax == 1 ? p1 : p2) : 0;
                        c[q][e] = a.cos[(size_t)p * (D / 2) + i + e];
                        n[q][e] = a.sin[(size_t)p * (D / 2) + i + e];
                    }
                } else {
                    const size_t at = (size_t)(ok ? p0 : 0) * (D / 2) + i;
                    const f4_any rc = *reinterpret_cast<const f4_any *>(a.cos + at), rn = *reinterpret_cast<const f4_any *>(a.sin + at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        c[q][e] = rc[e];
                        n[q][e] = rn[e];
                    }
                }
            }
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const bool upper = j >= 2;  // holds the odd elements of its chains
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float o = Q3VL_QUADP(v[q][e], 0x4E);  // quad_perm [2,3,0,1]
                    const float first = upper ? o : v[q][e], second = upper ? v[q][e] : o;
                    sum[e] = fmaf(first, first, sum[e]);
                    sum[e] = fmaf(second, second, sum[e]);
                }
            float ss = Q3VL_QUADP(sum[0], 0x00);
#pragma unroll
            for (int e = 1; e < 4; ++e) ss = ss + Q3VL_QUADP(sum[e], 0x00);
#pragma unroll
            for (int e = 0; e < 4; ++e) ss = ss + Q3VL_QUADP(sum[e], 0x55);
            float inv = rcp_rn(sqrt_rn(ss * (1.0f / D) + a.eps));
            if (!ok) inv = __builtin_nanf("");
            const float *w = wsh[is_q ? 0 : 1] + 4 * j, *ws = ssh[is_q ? 0 : 1] + 4 * j;
#pragma unroll
            for (int q = 0; q < QH; ++q) {
                const float4 wl = *reinterpret_cast<const float4 *>(w + 16 * q), wh = *reinterpret_cast<const float4 *>(w + 16 * q + D / 2);
                const float4 sl = *reinterpret_cast<const float4 *>(ws + 16 * q), sh = *reinterpret_cast<const float4 *>(ws + 16 * q + D / 2);
                const float wle[4] = {wl.x, wl.y, wl.z, wl.w}, whe[4] = {wh.x, wh.y, wh.z, wh.w};
                const float sle[4] = {sl.x, sl.y, sl.z, sl.w}, she[4] = {sh.x, sh.y, sh.z, sh.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = wle[e] * ((sle[e] * inv) * v[q][e]);
                    const float z = whe[e] * ((she[e] * inv) * v[q + QH][e]);
                    v[q][e] = fmaf(y, c[q][e], -(z * n[q][e]));
                    v[q + QH][e] = fmaf(y, n[q][e], z * c[q][e]);
                }
            }
        }
        if (is_q && !HALF) {
            float *o = static_cast<float *>(a.q_out) + row * a.ldo + (size_t)h * D + 4 * j;
#pragma unroll
            for (int q = 0; q < Q; ++q) *reinterpret_cast<f4_any *>(o + 16 * q) = f4_any{v[q][0], v[q][1], v[q][2], v[q][3]};
        } else if (is_q) {
            uint16_t *o = static_cast<uint16_t *>(a.q_out) + row * a.ldo + (size_t)h * D + 4 * j;
#pragma unroll
            for (int q = 0; q < Q; ++q)
                *reinterpret_cast<h4_any *>(o + 16 * q) = h4_any{f2h(v[q][0]), f2h(v[q][1]), f2h(v[q][2]), f2h(v[q][3])};
        } else {
            // (slots mostly fit 32 bits, whose division is a fraction of the 64-bit one)
            const uint64_t seq = slot <= 0xFFFFFFFFll ? (uint32_t)slot / (uint32_t)a.max_seq : (uint64_t)slot / (uint32_t)a.max_seq;
            uint16_t *o = (is_k ? a.k_cache : a.v_cache) + seq * a.seq_stride + (size_t)h * a.head_stride +
                          ((size_t)slot - seq * (uint32_t)a.max_seq) * a.row_stride + 4 * j;
#pragma unroll
            for (int q = 0; q < Q; ++q)
                *reinterpret_cast<h4_row *>(o + 16 * q) = h4_row{f2h(v[q][0]), f2h(v[q][1]), f2h(v[q][2]), f2h(v[q][3])};
        }
    }
}

hipError_t launch_qk_norm_rope(const QkRopeArgs &a, int head_dim, bool half, int axes, hipStream_t st) {
    const int64_t per_row = (a.heads + 2 * a.kv_heads + 15) / 16, blocks = (a.rows * per_row + 3) / 4;
    const unsigned grid = (unsigned)(blocks < 2048 ? blocks : 2048);  // eight a CU, each its share
    auto go = [&](auto kernel) {
        kernel<<<grid, 256, 0, st>>>(a.q, a.k, a.v, a.pos, a.slots, a.heads, a.kv_heads, a.gs, (int)a.rows, a);
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
