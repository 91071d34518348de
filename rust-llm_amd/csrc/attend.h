// Attention of new tokens over the paged cache (include/rl_mixers.h).
#pragma once
#include "kv_cache.h"

namespace rl {

struct AttendArgs {
    CacheArgs cache;
    const void *q;
    void *out;
    float *lse;
    uint64_t q_row, q_head, out_row, out_head;
    const int32_t *starts, *lens, *pages;
    uint32_t rows, seqs, q_heads, table_width, window, most_rows, max_len;
    float scale;
};

// The sequence that a query row belongs to: the last that starts at or before it
// (empty ones share their start with the next).
__device__ inline uint32_t sequence_of(const int32_t *starts, uint32_t seqs, uint32_t row) {
    if (!starts) return row;
    uint32_t lo = 0, hi = seqs;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if ((uint32_t)starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

constexpr uint32_t ATTEND_THREADS = 256;

// One workgroup a query row and head: a thread a token for the scores, a thread a
// value column for the sums, one pass with the running maximum and sum.
template <typename T, int FMT>
__global__ void __launch_bounds__(ATTEND_THREADS) k_attend_rows(AttendArgs a) {
    __shared__ float qs[256], ps[ATTEND_THREADS], red[ATTEND_THREADS / 64];
    __shared__ int bad;
    const uint32_t tid = threadIdx.x, row = blockIdx.x / a.q_heads, qh = blockIdx.x - row * a.q_heads;
    const uint32_t dim = a.cache.dim, head = qh / (a.q_heads / a.cache.heads), page = a.cache.page;
    const uint32_t s = sequence_of(a.starts, a.seqs, row);
    const uint32_t first = a.starts ? a.starts[s] : s, n = a.starts ? a.starts[s + 1] - first : 1;
    const int64_t len = a.lens[s], at = len - n + (row - first);
    const int64_t end = at + 1 > 0 ? at + 1 : 0, begin = a.window && end > a.window ? end - a.window : 0;
    T *out = (T *)a.out + row * a.out_row + qh * a.out_head;
    if (tid == 0) bad = n > a.most_rows || len > a.max_len || (end > 0 && (uint64_t)(end - 1) / page >= a.table_width);
    if (tid < dim) qs[tid] = (float)((const T *)a.q + row * a.q_row + qh * a.q_head)[tid] * a.scale;
    __syncthreads();
    // Read between barriers only, so that every thread leaves the loop in the same round.
    bool stop = bad;
    __syncthreads();
    float top = -INFINITY, total = 0.0f, sum = 0.0f;
    for (int64_t t0 = begin; !stop && t0 < end; t0 += ATTEND_THREADS) {
        const int64_t t = t0 + tid;
        const uint32_t count = (uint32_t)(end - t0 < ATTEND_THREADS ? end - t0 : ATTEND_THREADS);
        float x = -INFINITY;
        if (tid < count) {
            const int32_t p = a.pages[(uint64_t)s * a.table_width + t / page];
            if (p < 0 || (uint64_t)p >= a.cache.slots / page) bad = 1;
            else {
                const uint64_t v = cache_vector(a.cache, (uint64_t)p * page + t % page, head);
                x = 0.0f;
                for (uint32_t d = 0; d < dim; d += 8) {
                    float k[8];
                    if constexpr (FMT == RL_F16) load_f32((const half_t *)a.cache.keys + v * dim + d, true, k);
                    else if constexpr (FMT == RL_BF16) load_f32((const bhalf_t *)a.cache.keys + v * dim + d, true, k);
                    else decode8<FMT>(*(const uint2 *)((const uint8_t *)a.cache.keys + v * dim + d), k);
#pragma unroll
                    for (int j = 0; j < 8; j++) x += qs[d + j] * k[j];
                }
                if constexpr (FMT == RL_I8 || FMT == RL_F8) x *= a.cache.key_steps[v];
            }
        }
        float m = group_max<64>(x);
        if (tid % 64 == 0) red[tid / 64] = m;
        __syncthreads();
        stop = bad;
        if (stop) break;
        m = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), top);
        const float keep = top == -INFINITY ? 0.0f : expf(top - m);
        const float p = tid < count ? expf(x - m) : 0.0f;
        ps[tid] = p;
        const float part = group_sum<64>(p);
        __syncthreads();
        if (tid % 64 == 0) red[tid / 64] = part;
        __syncthreads();
        total = total * keep + (red[0] + red[1] + red[2] + red[3]);
        top = m;
        if (tid < dim) {
            sum *= keep;
            for (uint32_t j = 0; j < count; j++) {
                const int64_t u = t0 + j;
                const uint64_t v = cache_vector(
                    a.cache, (uint64_t)a.pages[(uint64_t)s * a.table_width + u / page] * page + u % page, head);
                float x1;
                if constexpr (FMT == RL_F16) x1 = (float)((const half_t *)a.cache.values)[v * dim + tid];
                else if constexpr (FMT == RL_BF16) x1 = (float)((const bhalf_t *)a.cache.values)[v * dim + tid];
                else {
                    float w[8];
                    decode8<FMT>(make_uint2(((const uint8_t *)a.cache.values)[v * dim + tid], 0), w);
                    x1 = w[0] * a.cache.value_steps[v];
                }
                sum += ps[j] * x1;
            }
        }
        __syncthreads();
    }
    if (tid < dim) out[tid] = (T)(stop ? NAN : end == begin ? 0.0f : sum / total);
    if (tid == 0 && a.lse)
        a.lse[(uint64_t)row * a.q_heads + qh] = stop ? NAN : end == begin ? -INFINITY : top + logf(total);
}

}  // namespace rl
