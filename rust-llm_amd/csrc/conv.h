// The short causal convolution (include/rl_mixers.h).
//
//   y[t][c] = act(bias[c] + sum_j w[j][c] x[t - W + 1 + j][c])
//
// A wave takes 512 channels (16-bit types; 256 of f32) of a run of rows and keeps the
// W - 1 rows before the current one in registers: a row is read once but for the W - 1
// that a run reads again of the one before. The rows before a sequence's first are its
// state; the run with the first row reads it and also writes the new one, so a slot may
// be read and written by one call.
//
// Bound by HBM for long prompts (8192 rows of 8192 bf16 channels, width 4: 52 us, 5.1
// TB/s, 44.3 again over the same rows; rows not aligned to 16 bytes 60.2), below that by
// the instructions of
// a wave, some 500 cycles a row, of which the exponential and the reciprocal of the
// activation are a third. Weights are loaded as vectors: one by one, lanes 32 bytes apart,
// they took twice the time of all the rows (88 us for the same, 16.5 for 1024 rows
// where it is 9.0 now).
#pragma once
#include "row_blocks.h"

namespace rl {

struct ConvArgs {
    const void *x;
    void *out;
    uint64_t x_row, out_row;
    const float *weight, *bias; // [W][channels], [channels]
    void *states;               // [slots][W - 1][channels]
    uint64_t state_slots;
    const int32_t *slots_in, *slots_out, *starts;
    uint32_t rows, seqs, channels;
    uint32_t columns; // waves that a row takes
    RowBlocks runs;   // at least W - 1 rows
};

constexpr uint32_t CONV_MAX_WIDTH = 8, CONV_LANES = 64;

// y / (1 + e^-y). f32 outputs get the rounding of y log2 e back, which is all that e^-y would lose.
template <typename T>
__device__ inline float silu(float y) {
    constexpr float L = 1.44269504088896341f, LOW = 1.92596299e-8f, LN2 = 0.693147180559945309f;
    const float p = y * -L;
    float e = __builtin_amdgcn_exp2f(p);
    if constexpr (sizeof(T) == 4) {
        const float rest = fmaf(y, -L, -p) - y * LOW;
        if (fabsf(rest) < 1.0f && e < INFINITY) e = fmaf(e, rest * LN2, e);
        return y / (1.0f + e);
    } else
        return y * __builtin_amdgcn_rcpf(1.0f + e);
}

// WIDE: a lane's V channels are one 16-byte vector; else they are 64 apart.
template <typename T, int W, bool WIDE, bool SILU>
__global__ void __launch_bounds__(CONV_LANES) k_conv(ConvArgs a) {
    constexpr int V = WIDE ? 16 / sizeof(T) : 4, AHEAD = 4;
    using Raw = vec<T, V>;
    const uint32_t block = blockIdx.x / a.columns, column = blockIdx.x - block * a.columns, lane = threadIdx.x;
    const RowBlock r = find_block(a.starts, a.rows, a.seqs, a.runs, block);
    if (!r.used) return;
    const auto channel = [&](int i) { return column * 64 * V + (WIDE ? lane * V + i : lane + 64 * i); };
    if (channel(0) >= a.channels) return;
    const auto load = [&](const T *row) {
        Raw v;
        if constexpr (WIDE) v = *(const Raw *)(row + channel(0));
        else
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = row[min(channel(i), a.channels - 1)];
        return v;
    };
    const auto store = [&](T *row, const Raw &v) {
        if constexpr (WIDE) *(Raw *)(row + channel(0)) = v;
        else
#pragma unroll
            for (int i = 0; i < V; i++)
                if (channel(i) < a.channels) row[channel(i)] = v[i];
    };
    const auto state = [&](int32_t slot, int j) { return (T *)a.states + ((uint64_t)(uint32_t)slot * (W - 1) + j) * a.channels; };
    const auto none = [&](float x) {
        Raw v;
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = (T)x;
        return v;
    };
    const uint32_t t0 = r.block * a.runs.size, count = min(r.rows - t0, a.runs.size); // t0 is 0 where there are no rows
    const T *x = (const T *)a.x + (uint64_t)r.begin * a.x_row;
    const int32_t in = t0 ? -1 : a.slots_in[r.seq];
    // What the sequence's state holds in row j.
    const auto before = [&](int j) {
        if (in < 0) return none(0.0f);
        return (uint64_t)in < a.state_slots ? load(state(in, j)) : none(NAN);
    };
    Raw ahead[AHEAD], history[W - 1];
    if (count) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++) ahead[u] = load(x + (uint64_t)(t0 + min((uint32_t)u, count - 1)) * a.x_row);
    }
#pragma unroll
    for (int j = 0; j < W - 1; j++) history[j] = t0 ? load(x + (uint64_t)(t0 - (W - 1) + j) * a.x_row) : before(j);
    float w[W][V], bias[V];
    const auto weights = [&](const float *from, float *to) {
        if constexpr (WIDE)
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const f32x4 v = *(const f32x4 *)(from + channel(i));
#pragma unroll
                for (int k = 0; k < 4; k++) to[i + k] = v[k];
            }
        else
#pragma unroll
            for (int i = 0; i < V; i++) to[i] = from[min(channel(i), a.channels - 1)];
    };
    weights(a.bias, bias);
#pragma unroll
    for (int j = 0; j < W; j++) weights(a.weight + (uint64_t)j * a.channels, w[j]);
    if (!t0) {
        const int32_t to = a.slots_out[r.seq];
        if (to >= 0 && (uint64_t)to < a.state_slots) {
            // The last W - 1 of the old state's rows and the sequence's. Row rows + j of the two; all are loaded before the
            // first is written.
            Raw next[W - 1];
#pragma unroll
            for (int j = 0; j < W - 1; j++) {
                if (r.rows + j >= W - 1) next[j] = load(x + (uint64_t)(r.rows + j - (W - 1)) * a.x_row);
                else next[j] = before(r.rows + j);
            }
#pragma unroll
            for (int j = 0; j < W - 1; j++) store(state(to, j), next[j]);
        }
    }
    float window[W - 1 + AHEAD][V];
#pragma unroll
    for (int j = 0; j < W - 1; j++)
#pragma unroll
        for (int i = 0; i < V; i++) window[j][i] = (float)history[j][i];
    T *out = (T *)a.out + (uint64_t)(r.begin + t0) * a.out_row;
    for (uint32_t u0 = 0; u0 < count; u0 += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
#pragma unroll
            for (int i = 0; i < V; i++) window[W - 1 + u][i] = (float)ahead[u][i];
        if (u0 + AHEAD < count) {
#pragma unroll
            for (int u = 0; u < AHEAD; u++)
                ahead[u] = load(x + (uint64_t)(t0 + min(u0 + AHEAD + u, count - 1)) * a.x_row);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            if (u0 + u >= count) break;
            Raw v;
#pragma unroll
            for (int i = 0; i < V; i++) {
                float y = bias[i];
#pragma unroll
                for (int j = 0; j < W; j++) y = fmaf(w[j][i], window[u + j][i], y);
                v[i] = (T)(SILU ? silu<T>(y) : y);
            }
            store(out + (uint64_t)(u0 + u) * a.out_row, v);
        }
#pragma unroll
        for (int j = 0; j < W - 1; j++)
#pragma unroll
            for (int i = 0; i < V; i++) window[j][i] = window[AHEAD + j][i];
    }
}

}  // namespace rl
