// The selective state space scan (include/rl_mixers.h).
//
//   D = softplus(dt + bias);  h[n] <- 2^(D a2[n]) h[n] + D x b[n];  y = sum_n c[n] h[n]
//
// with a2 = a log2(e). All f32. A channel does not depend on the others.
#pragma once
#include "conv.h"

namespace rl {

struct ScanArgs {
    const void *x, *dt, *z, *b, *c; // z may be null
    void *out;
    uint64_t x_row, dt_row, z_row, b_row, b_group, c_row, c_group, out_row;
    const float *a2, *skip, *bias; // [channels][state], [channels], [channels]
    float *states;                 // [slots][channels][state]
    uint64_t state_slots;
    const int32_t *slots_in, *slots_out, *starts;
    uint32_t rows, seqs, channels, groups, state;
    uint32_t per;      // channels of a group
    uint32_t softplus; // whether steps are softplus(dt + bias), else dt + bias
    uint32_t wide;     // whether four values of b and c are one aligned vector
    uint32_t columns;  // workgroups that a row (prompts: a piece) takes
    RowBlocks pieces;  // prompts: tokens of a piece, 0 for whole sequences
    // Pieces of sequences that have several: ends[slot] is a state as the lanes hold it, steps[slot][channel] the sum of a
    // piece's steps. A sequence's slots begin at scan_slot; slot 0 of a sequence has its first state and piece i's end from
    // zeros is in slot i + 1.
    float *ends, *steps;
};

constexpr uint32_t SCAN_THREADS = 256, SCAN_WAVES = 4;

// The first slot of a sequence of more rows than a piece has; it needs one slot a piece, which are at most twice as many as
// whole pieces lie between its first row and the next sequence's.
__device__ inline uint64_t scan_slot(uint32_t begin, RowBlocks pieces) { return 2 * (uint64_t)split_by(begin, pieces.size, pieces.inv).x; }
inline uint64_t scan_slots(uint64_t pieces) { return 2 * pieces + 2; } // of a call of that many whole pieces

// ln(1 + e^v), to f32's precision for every v: 0 for the lowest ones and -infinity, NaN for NaN.
__device__ inline float soft_plus(float v) {
    constexpr float L = 1.44269504088896341f, LOW = 1.92596299e-8f, LN2 = 0.693147180559945309f;
    const float m = -fabsf(v), p = m * L;
    // The rounding of m L is brought back while e^m is a normal number; below, m L may be infinite and its rounding with it.
    const float e = __builtin_amdgcn_exp2f(p), t = p > -126.0f ? fmaf(e, (fmaf(m, L, -p) + m * LOW) * LN2, e) : e;
    // ln(1 + t) by the rounded sum u and what the rounding took, at most 2^-24: ln(u) + (1 + t - u) / u. The last division
    // by 1 to 2 is left out, which costs at most a unit in the last place.
    const float u = 1.0f + t;
    return fmaxf(v, 0.0f) + fmaf(__builtin_amdgcn_logf(u), LN2, t - (u - 1.0f));
}

template <typename T>
__device__ inline float scan_step(const ScanArgs &a, T dt, float bias) {
    const float v = (float)dt + bias;
    return a.softplus ? soft_plus(v) : v;
}

// Single tokens and short runs. L lanes hold a channel, four state values each, so
// states move as whole vectors. Bound by HBM, the state in and out: 64 sequences of
// 5120 channels of 16 take 13.0 us over inputs that change, 3.4 TB/s.
template <typename T, int L>
__global__ void __launch_bounds__(SCAN_THREADS) k_scan_steps(ScanArgs a) {
    const uint32_t s = blockIdx.x / a.columns, column = blockIdx.x - s * a.columns, lane = threadIdx.x % 64;
    const uint32_t ch = column * (SCAN_THREADS / L) + threadIdx.x / L, n0 = 4 * (lane % L);
    const bool here = ch < a.channels && n0 < a.state;
    const uint32_t channel = min(ch, a.channels - 1), at = n0 < a.state ? n0 : 0, group = channel / a.per;
    uint32_t begin = s, end = s + 1;
    if (a.starts) {
        begin = (uint32_t)min(max(a.starts[s], 0), (int32_t)a.rows);
        end = (uint32_t)min(max(a.starts[s + 1], 0), (int32_t)a.rows);
    }
    const int32_t in = a.slots_in[s], to = a.slots_out[s];
    const auto state = [&](int32_t slot) { return a.states + ((uint64_t)(uint32_t)slot * a.channels + channel) * a.state + at; };
    f32x4 h = {0, 0, 0, 0};
    if (in >= 0) {
        if ((uint64_t)in < a.state_slots) h = *(const f32x4 *)state(in);
        else h = f32x4{NAN, NAN, NAN, NAN};
    }
    f32x4 a2 = *(const f32x4 *)(a.a2 + (uint64_t)channel * a.state + at);
    if (!here) h = a2 = f32x4{0, 0, 0, 0};
    const float bias = a.bias[channel], skip = a.skip[channel];
    T x{}, dt{}, z{};
    float b[4] = {}, c[4] = {};
    auto fetch = [&](uint64_t t) {
        x = ((const T *)a.x)[t * a.x_row + channel];
        dt = ((const T *)a.dt)[t * a.dt_row + channel];
        if (a.z) z = ((const T *)a.z)[t * a.z_row + channel];
        load_f32((const T *)a.b + t * a.b_row + group * a.b_group + at, a.wide, b);
        load_f32((const T *)a.c + t * a.c_row + group * a.c_group + at, a.wide, c);
    };
    if (begin < end) fetch(begin);
    for (uint32_t t = begin; t < end; t++) {
        const float step = scan_step(a, dt, bias), xt = (float)x, zt = (float)z, drive = step * xt;
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            h[i] = fmaf(__builtin_amdgcn_exp2f(step * a2[i]), h[i], drive * b[i]);
            y = fmaf(h[i], c[i], y);
        }
        if (!here) y = 0.0f;
        if (t + 1 < end) fetch(t + 1);
        y = fmaf(skip, xt, group_sum<L>(y));
        if (a.z) y *= silu<T>(zt);
        if (here && n0 == 0) ((T *)a.out)[(uint64_t)t * a.out_row + channel] = (T)y;
    }
    if (to >= 0 && (uint64_t)to < a.state_slots && here) *(f32x4 *)state(to) = h;
}

// Prompts. L lanes hold a channel, S state values each: a step's softplus, gate and
// sums are formed once for S of them. A workgroup takes 256 / L channels of a group
// through a piece of one sequence; b and c of the next tokens are staged in LDS in f32
// and read by all. Where a call has too few channels to fill the device its sequences
// go in pieces: SCAN_ENDS leaves what each but the last does to a state of zeros,
// and the pass with the outputs makes each piece's first state of those before it.
// Bound by instructions: while a CU has waves its vector units issue without a pause.
// A wave's instruction takes them 4 cycles, an exponential 8. 8192 tokens of 5120
// channels of 16: 64 and 90 million instructions in the two passes and 12 and 15 million
// exponentials and logarithms among them, 140 and 201 us at 2.1 GHz. A token, channel
// and state value has 5 or 6 of these slots, two thirds of all; the others are softplus,
// gates, sums and loads. 24 prompts of up to 701 tokens, 1536 channels of 32 in f32:
// 59 and 88 us, of which instructions 46 and 68; CUs that are done wait for the last.
enum ScanPass { SCAN_ENDS, SCAN_OUTPUTS };

template <typename T, int S, int L, ScanPass PASS>
__global__ void __launch_bounds__(SCAN_THREADS) k_scan(ScanArgs a) {
    constexpr int N = S * L, TILE = N <= 64 ? 16 : 4, U = 8 < TILE ? 8 : TILE; // tokens staged at a time, tokens ahead
    constexpr bool OUT = PASS == SCAN_OUTPUTS;
    constexpr int SIDES = OUT ? 2 : 1, QUADS = TILE * SIDES * N / 4, EACH = (QUADS + SCAN_THREADS - 1) / SCAN_THREADS;
    __shared__ __attribute__((aligned(16))) float staged[2][TILE][SIDES][N];
    const uint32_t block = blockIdx.x / a.columns, column = blockIdx.x - block * a.columns, tid = threadIdx.x;
    RowBlock r;
    const bool whole = a.pieces.size == 0; // sequences
    if (whole) {
        r.seq = block, r.block = 0, r.begin = block, r.rows = 1;
        if (a.starts) {
            r.begin = (uint32_t)min(max(a.starts[block], 0), (int32_t)a.rows);
            r.rows = max(min(max(a.starts[block + 1], 0), (int32_t)a.rows) - (int32_t)r.begin, 0);
        }
    } else {
        r = find_block(a.starts, a.rows, a.seqs, a.pieces, block);
        if (!r.used) return;
    }
    const uint32_t t0 = r.block * a.pieces.size, count = whole ? r.rows : min(r.rows - t0, a.pieces.size);
    const bool several = count < r.rows, last = t0 + count == r.rows;
    if (!OUT && last) return;
    const uint32_t tiles = a.columns / a.groups; // of a group
    const uint32_t group = column / tiles, ch = (column - group * tiles) * (SCAN_THREADS / L) + tid / L;
    const bool mine = ch < a.per;
    const uint32_t channel = group * a.per + min(ch, a.per - 1), n0 = S * (tid % L);
    // A state as the lanes of a workgroup hold it, quads of all lanes side by side.
    const auto end_at = [&](uint64_t slot, int i) {
        return a.ends + (((slot * a.columns + column) * (S / 4) + i / 4) * SCAN_THREADS + tid) * 4;
    };
    const auto state = [&](int32_t slot) { return a.states + ((uint64_t)(uint32_t)slot * a.channels + channel) * a.state; };
    const uint64_t slot0 = whole ? 0 : scan_slot(r.begin, a.pieces);
    float h[S], a2[S];
#pragma unroll
    for (int i = 0; i < S; i += 4) {
        const bool in = n0 + i < a.state; // state is a multiple of 4
        const f32x4 v = *(const f32x4 *)(a.a2 + (uint64_t)channel * a.state + (in ? n0 + i : 0));
#pragma unroll
        for (int j = 0; j < 4; j++) a2[i + j] = in ? v[j] : 0.0f, h[i + j] = 0.0f;
    }
    if (t0 == 0 && (!OUT || !several)) {
        const int32_t from = a.slots_in[r.seq];
        if (from >= 0) {
#pragma unroll
            for (int i = 0; i < S; i += 4) {
                const bool in = n0 + i < a.state;
                f32x4 v = {NAN, NAN, NAN, NAN};
                if ((uint64_t)from < a.state_slots) v = *(const f32x4 *)(state(from) + (in ? n0 + i : 0));
#pragma unroll
                for (int j = 0; j < 4; j++) h[i + j] = in ? v[j] : 0.0f;
            }
        }
        if (!OUT) { // kept for the second pass, when the slot may be written
#pragma unroll
            for (int i = 0; i < S; i += 4) {
                *(f32x4 *)end_at(slot0, i) = f32x4{h[i], h[i + 1], h[i + 2], h[i + 3]};
#pragma unroll
                for (int j = 0; j < 4; j++) h[i + j] = 0.0f;
            }
        }
    }
    if (OUT && several) {
        for (uint32_t p = 0; p <= r.block; p++) {
            const float sum = p ? a.steps[(slot0 + p) * a.channels + channel] : 0.0f;
#pragma unroll
            for (int i = 0; i < S; i += 4) {
                const f32x4 v = *(const f32x4 *)end_at(slot0 + p, i);
#pragma unroll
                for (int j = 0; j < 4; j++) h[i + j] = p ? fmaf(__builtin_amdgcn_exp2f(sum * a2[i + j]), h[i + j], v[j]) : v[j];
            }
        }
    }
    const float bias = a.bias[channel], skip = a.skip[channel];
    const uint64_t row0 = r.begin + t0;
    const T *xs = (const T *)a.x + row0 * a.x_row + channel, *dts = (const T *)a.dt + row0 * a.dt_row + channel;
    const T *zs = (const T *)a.z + (a.z ? row0 * a.z_row + channel : 0);
    T *out = (T *)a.out + row0 * a.out_row + channel;
    const T *sides[2] = {(const T *)a.b + row0 * a.b_row + group * a.b_group, (const T *)a.c + row0 * a.c_row + group * a.c_group};
    float stage[EACH][4];
    // Quads tid, tid + 256, .. of the tile's b (and c); what is past the state or the piece is zero.
    auto fetch = [&](uint32_t t) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const uint32_t q = tid + e * SCAN_THREADS, n = q % (N / 4) * 4, side = q / (N / 4) % SIDES, token = t + q / (N / 4) / SIDES;
#pragma unroll
            for (int j = 0; j < 4; j++) stage[e][j] = 0.0f;
            if (q < QUADS && n < a.state && token < count)
                load_f32(sides[side] + (uint64_t)token * (side ? a.c_row : a.b_row) + n, a.wide, stage[e]);
        }
    };
    auto put = [&](int buffer) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const uint32_t q = tid + e * SCAN_THREADS;
            if (q < QUADS) *(f32x4 *)(&staged[buffer][0][0][0] + q * 4) = f32x4{stage[e][0], stage[e][1], stage[e][2], stage[e][3]};
        }
    };
    T x[U], dt[U], z[U];
    auto ahead = [&](uint32_t t) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint64_t at = min(t + u, count - 1);
            x[u] = xs[at * a.x_row], dt[u] = dts[at * a.dt_row];
            if (OUT && a.z) z[u] = zs[at * a.z_row];
        }
    };
    float total = 0.0f;
    if (count) {
        fetch(0);
        ahead(0);
        put(0);
    }
    __syncthreads();
    for (uint32_t t = 0; t < count; t += TILE) {
        const int buffer = t / TILE % 2;
        const bool more = t + TILE < count;
        if (more) fetch(t + TILE);
#pragma unroll
        for (int u0 = 0; u0 < TILE; u0 += U) {
            float xt[U], step[U], zt[U];
#pragma unroll
            for (int u = 0; u < U; u++) xt[u] = (float)x[u], step[u] = scan_step(a, dt[u], bias), zt[u] = OUT && a.z ? (float)z[u] : 0.0f;
            if (t + u0 + U < count) ahead(t + u0 + U);
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (t + u0 + u >= count) break;
                const float *bs = staged[buffer][u0 + u][0] + n0, *cs = staged[buffer][u0 + u][SIDES - 1] + n0;
                const float drive = step[u] * xt[u];
                float y = 0.0f;
#pragma unroll
                for (int i = 0; i < S; i += 4) {
                    const f32x4 b = *(const f32x4 *)(bs + i), c = *(const f32x4 *)(cs + i);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        h[i + j] = fmaf(__builtin_amdgcn_exp2f(step[u] * a2[i + j]), h[i + j], drive * b[j]);
                        if (OUT) y = fmaf(h[i + j], c[j], y);
                    }
                }
                if constexpr (OUT) {
                    y = fmaf(skip, xt[u], group_sum<L>(y));
                    if (a.z) y *= silu<T>(zt[u]);
                    if (mine && n0 == 0) out[(uint64_t)(t + u0 + u) * a.out_row] = (T)y;
                } else
                    total += step[u];
            }
        }
        if (more) put(1 - buffer);
        __syncthreads();
    }
    if constexpr (!OUT) {
        const uint64_t slot = slot0 + r.block + 1;
#pragma unroll
        for (int i = 0; i < S; i += 4) *(f32x4 *)end_at(slot, i) = f32x4{h[i], h[i + 1], h[i + 2], h[i + 3]};
        if (mine && n0 == 0) a.steps[slot * a.channels + channel] = total;
    } else if (last) {
        const int32_t to = a.slots_out[r.seq];
        if (to >= 0 && (uint64_t)to < a.state_slots && mine) {
#pragma unroll
            for (int i = 0; i < S; i += 4)
                if (n0 + i < a.state) *(f32x4 *)(state(to) + n0 + i) = f32x4{h[i], h[i + 1], h[i + 2], h[i + 3]};
        }
    }
}

// Launches for one element type (scan_*.hip, one unit a type).
template <typename T>
void launch_scan_steps(const ScanArgs &a, hipStream_t s);
template <typename T>
void launch_scan(const ScanArgs &a, hipStream_t s);

// Lanes that hold a channel of `state` values, `each` a lane: a power of two.
inline uint32_t scan_lanes(uint32_t state, uint32_t each) {
    uint32_t lanes = 1;
    while (lanes * each < state) lanes *= 2;
    return lanes;
}
// State values a lane of k_scan.
inline uint32_t scan_each(uint32_t state) { return state <= 8 ? 8 : 16; }

#ifdef RL_SCAN_UNIT
template <typename T>
void launch_scan_steps(const ScanArgs &a, hipStream_t s) {
    const uint32_t lanes = scan_lanes(a.state, 4);
    auto kern = lanes == 1 ? k_scan_steps<T, 1> : lanes == 2 ? k_scan_steps<T, 2> : lanes == 4 ? k_scan_steps<T, 4>
              : lanes == 8 ? k_scan_steps<T, 8> : lanes == 16 ? k_scan_steps<T, 16> : lanes == 32 ? k_scan_steps<T, 32>
                                                                                       : k_scan_steps<T, 64>;
    hipLaunchKernelGGL(kern, dim3(a.seqs * a.columns), dim3(SCAN_THREADS), 0, s, a);
}

template <typename T, int S, int L>
void launch_scan_of(const ScanArgs &a, hipStream_t s) {
    const dim3 grid((a.pieces.size ? row_block_count(a.rows, a.seqs, a.pieces.size) : a.seqs) * a.columns);
    if (a.pieces.size) hipLaunchKernelGGL((k_scan<T, S, L, SCAN_ENDS>), grid, dim3(SCAN_THREADS), 0, s, a);
    hipLaunchKernelGGL((k_scan<T, S, L, SCAN_OUTPUTS>), grid, dim3(SCAN_THREADS), 0, s, a);
}

template <typename T>
void launch_scan(const ScanArgs &a, hipStream_t s) {
    if (a.state <= 8) return launch_scan_of<T, 8, 1>(a, s);
    switch (scan_lanes(a.state, 16)) {
    case 1: return launch_scan_of<T, 16, 1>(a, s);
    case 2: return launch_scan_of<T, 16, 2>(a, s);
    case 4: return launch_scan_of<T, 16, 4>(a, s);
    case 8: return launch_scan_of<T, 16, 8>(a, s);
    default: return launch_scan_of<T, 16, 16>(a, s);
    }
}
#endif

}  // namespace rl
