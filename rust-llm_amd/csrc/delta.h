// The gated delta rule (include/rl_mixers.h), one token after the other.
#pragma once
#include "mix_types.h"

namespace rl {

struct DeltaArgs {
    const void *q, *k, *v;
    void *out;
    uint64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
    const float *g, *beta;
    uint64_t g_row, beta_row;
    float *states;
    uint64_t state_slots;
    const int32_t *slots_in, *slots_out, *starts;
    uint32_t rows, seqs, key_heads, value_heads, key_dim, value_dim;
    float scale, eps; // eps < 0: q and k as they are
    uint32_t wide;    // whether q, k, v and out are aligned for 16-byte accesses
};

constexpr uint32_t DELTA_WAVES = 4;

// Where a sequence's rows begin, within the call's rows whatever `starts` holds.
__device__ inline uint32_t first_row(const DeltaArgs &a, uint32_t s) {
    return a.starts ? (uint32_t)min(max(a.starts[s], 0), (int)a.rows) : s;
}

// Sum over the lanes Q apart, which hold one column quad.
template <int Q>
__device__ inline float quad_sum(float x) {
    x += rotate16<8>(x);
    x += rotate16<4>(x);
    if (Q == 2) x += rotate16<2>(x);
    return rows_sum(x);
}

// A wave holds 4 Q columns of one head's state in registers (16, or 8 where 16
// leave SIMDs idle and the chain of a step counts): a column does not
// depend on the others, so a state splits over as many waves as it has column
// groups and no wave waits for another. Lane l has the columns 4 (l % Q) .. + 4 of
// the rows R (l / Q) .. + R; the two products with the state are summed over the
// 64 / Q lanes of a column, in registers. A step's inputs are loaded while the one
// before is computed; their norms, roots and e^g are formed at its own start. For single
// tokens bound by HBM (the state is
// read and written once): 64 sequences of 32 heads of 128 x 128 take 63.5 us, 4.2
// TB/s. For several by the chain of a step, two reductions over the wave: 9 rows of
// one sequence 11.9 us, about 1 us a row.
template <typename T, int R, int Q>
__global__ void __launch_bounds__(64 * DELTA_WAVES) k_delta_steps(DeltaArgs a) {
    const uint32_t lane = threadIdx.x % 64, col0 = (blockIdx.y * DELTA_WAVES + threadIdx.x / 64) * 4 * Q;
    const uint32_t s = blockIdx.x / a.value_heads, head = blockIdx.x - s * a.value_heads;
    if (col0 >= a.value_dim) return;
    const uint32_t key_head = head / (a.value_heads / a.key_heads);
    const uint32_t col = col0 + 4 * (lane % Q), row0 = R * (lane / Q);
    const uint32_t begin = first_row(a, s), end = first_row(a, s + 1);
    const int32_t in = a.slots_in[s], to = a.slots_out[s];
    const uint64_t size = (uint64_t)a.key_dim * a.value_dim;
    const bool here = row0 + R <= a.key_dim; // else none of the lane's rows: key_dim is a multiple of 16, so of R
    float k[R], q[R], v[4], g = 0.0f, beta = 0.0f;
    auto fetch = [&](uint32_t t) {
#pragma unroll
        for (int j = 0; j < R; j++) k[j] = q[j] = 0.0f;
        if (here) {
            load_f32((const T *)a.k + t * a.k_row + key_head * a.k_head + row0, a.wide, k);
            load_f32((const T *)a.q + t * a.q_row + key_head * a.q_head + row0, a.wide, q);
        }
        load_f32((const T *)a.v + t * a.v_row + head * a.v_head + col, a.wide, v);
        g = a.g[t * a.g_row + head];
        beta = a.beta[t * a.beta_row + head];
    };
    if (begin < end) fetch(begin);
    vec<float, 4> S[R];
    const float fill = in >= 0 && here ? NAN : 0.0f;
#pragma unroll
    for (int j = 0; j < R; j++) S[j] = fill;
    if (in >= 0 && (uint64_t)in < a.state_slots && here) {
        const float *src = a.states + ((uint64_t)in * a.value_heads + head) * size + (uint64_t)row0 * a.value_dim + col;
#pragma unroll
        for (int j = 0; j < R; j++) S[j] = *(const vec<float, 4> *)(src + (uint64_t)j * a.value_dim);
    }
    for (uint32_t t = begin; t < end; t++) {
        float kc[R], qc[R], vc[4], kn = 1.0f, qn = a.scale;
        const float keep = expf(g), b = beta;
        if (a.eps >= 0.0f) {
            float kk = 0.0f, qq = 0.0f;
#pragma unroll
            for (int j = 0; j < R; j++) kk = fmaf(k[j], k[j], kk), qq = fmaf(q[j], q[j], qq);
            kn = 1.0f / sqrtf(quad_sum<Q>(kk) + a.eps);
            qn = a.scale / sqrtf(quad_sum<Q>(qq) + a.eps);
        }
#pragma unroll
        for (int j = 0; j < R; j++) kc[j] = k[j] * kn, qc[j] = q[j] * qn;
#pragma unroll
        for (int c = 0; c < 4; c++) vc[c] = v[c];
        if (t + 1 < end) fetch(t + 1);
        float p[4] = {}, o[4] = {};
#pragma unroll
        for (int j = 0; j < R; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                S[j][c] *= keep;
                p[c] = fmaf(S[j][c], kc[j], p[c]);
            }
#pragma unroll
        for (int c = 0; c < 4; c++) p[c] = b * (vc[c] - quad_sum<Q>(p[c]));
#pragma unroll
        for (int j = 0; j < R; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                S[j][c] = fmaf(kc[j], p[c], S[j][c]);
                o[c] = fmaf(S[j][c], qc[j], o[c]);
            }
#pragma unroll
        for (int c = 0; c < 4; c++) o[c] = quad_sum<Q>(o[c]);
        if (lane < Q) store_f32((T *)a.out + t * a.out_row + head * a.out_head + col, a.wide, o);
    }
    if (to < 0 || (uint64_t)to >= a.state_slots || !here) return;
    float *dst = a.states + ((uint64_t)to * a.value_heads + head) * size + (uint64_t)row0 * a.value_dim + col;
#pragma unroll
    for (int j = 0; j < R; j++) *(vec<float, 4> *)(dst + (uint64_t)j * a.value_dim) = S[j];
}

}  // namespace rl
