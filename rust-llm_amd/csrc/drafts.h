// Verification of drafted tokens (include/rl_drafts.h).
//
// Every workgroup of a sequence finds for itself how many drafts are accepted (a gather
// of 64 drafts at a time), which names the one row, or pair of rows, to draw from. Dense
// rows: a workgroup a chunk of 4096 tokens sums what can be drawn of it; the last to
// arrive finds the chunk that the draw falls into and goes through it once more. Sums
// are f64 (products and differences of f32 values are exact there, or nearly), and their
// order does not depend on how workgroups arrive. Bound by HBM for many sequences, one
// row of each side: 64 of 248320 tokens 29 us, 4.4 TB/s. For few by the chain of loads
// (starts, drafted token, two gathers, a chunk, the arrival, the chunk sums, a chunk
// again): 9.4 us for one of 151936. Lists: a workgroup a sequence, the same chain without
// the arrival, 7.8 us for 64 of up to 8 drafts and 64 entries.
#pragma once
#include "mix_types.h"
#include "rl_drafts.h"

namespace rl {

struct DraftArgs {
    rl_probs target, draft; // draft.probs null: q is 1 at the drafted token
    const int32_t *drafted, *starts;
    const float *uniforms, *draws;
    int32_t *accepted, *tokens;
    uint32_t vocab, drafts, seqs, chunks;
    uint32_t per, groups; // chunks of a workgroup, workgroups of a sequence
    double *sums;      // [seq][chunk]
    uint32_t *arrived; // [seq], zero between calls
};

constexpr uint32_t DRAFT_THREADS = 256, DRAFT_WAVES = 4, DRAFT_CHUNK = 4096, DRAFT_EACH = DRAFT_CHUNK / DRAFT_THREADS;
constexpr uint32_t DRAFT_PER = 8; // chunks of a workgroup at most
constexpr uint32_t LIST_EACH = 4, LIST_CHUNK = DRAFT_THREADS * LIST_EACH, LIST_TILE = 1024;
constexpr int DRAFT_STORED = 0x0F70; // s_waitcnt vmcnt(0)

__device__ inline float positive(float p) { return p > 0.0f && p < INFINITY ? p : 0.0f; }
__device__ inline double probability(float p) { return (double)positive(p); }

// What the running sum has to pass. A draw of 1 or more or NaN passes none, also where rounding brings a running sum above
// the total.
__device__ inline double draft_border(float draw, double total) { return draw < 1.0f ? fmax((double)draw * total, 0.0) : INFINITY; }

// Inclusive sums over the wave in lane order.
__device__ inline double wave_scan(double x) {
    const uint32_t lane = threadIdx.x % 64;
#pragma unroll
    for (uint32_t d = 1; d < 64; d *= 2) {
        const double y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}

// The sum of the threads before this one, and of all, in thread order. `waves` is shared and free again after the next
// barrier.
__device__ inline double block_scan(double x, double *waves, double &all) {
    const uint32_t wave = threadIdx.x / 64;
    const double upto = wave_scan(x);
    __syncthreads();
    if (threadIdx.x % 64 == 63) waves[wave] = upto;
    __syncthreads();
    double before = 0.0;
    all = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < DRAFT_WAVES; w++) {
        if (w == wave) before = all;
        all += waves[w];
    }
    return before + (upto - x);
}

// The smallest of the threads' numbers.
__device__ inline uint32_t block_min(uint32_t x, uint32_t *waves) {
#pragma unroll
    for (uint32_t d = 32; d; d /= 2) x = min(x, (uint32_t)__shfl_xor((int)x, d));
    __syncthreads();
    if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = x;
    __syncthreads();
    return min(min(waves[0], waves[1]), min(waves[2], waves[3]));
}

constexpr uint32_t DRAFT_NONE = 0xFFFFFFFFu;

// The first of the block's entries, a run of N a thread, at which the running sum from `base` on passes `border`; the last
// above zero if none does, DRAFT_NONE without any.
template <uint32_t N>
__device__ inline uint32_t block_pick(const double (&left)[N], double base, double border, double *waves, uint32_t *mins) {
    double sum = 0.0, all;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) sum += left[i];
    double run = base + block_scan(sum, waves, all);
    uint32_t first = DRAFT_NONE, last = DRAFT_NONE; // `last` counts down, for the smallest
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
        run += left[i];
        if (!(left[i] > 0.0)) continue;
        const uint32_t at = threadIdx.x * N + i;
        if (run > border && first == DRAFT_NONE) first = at;
        last = ~(at + 1);
    }
    first = block_min(first, mins);
    if (first != DRAFT_NONE) return first;
    last = block_min(last, mins);
    return last == DRAFT_NONE ? DRAFT_NONE : ~last - 1;
}

struct DraftSpan {
    uint32_t begin, count; // the sequence's drafts, within the call's whatever `starts` holds
};
__device__ inline DraftSpan draft_span(const DraftArgs &a, uint32_t s) {
    const int32_t n = (int32_t)a.drafts, b = min(max(a.starts[s], 0), n), e = min(max(a.starts[s + 1], 0), n);
    return {(uint32_t)b, (uint32_t)max(e - b, 0)};
}

// What the sequence's outputs are, by all threads of a workgroup.
__device__ inline void draft_write(const DraftArgs &a, uint32_t s, const DraftSpan &d, uint32_t accepted, int32_t token) {
    if (threadIdx.x == 0) a.accepted[s] = (int32_t)accepted;
    for (uint32_t i = threadIdx.x; i <= d.count; i += DRAFT_THREADS)
        a.tokens[(uint64_t)d.begin + s + i] = i < accepted ? a.drafted[d.begin + i] : i == accepted ? token : -1;
}

// WIDE: rows are aligned for 16-byte loads.
template <bool WIDE>
__global__ void __launch_bounds__(DRAFT_THREADS) k_drafts(DraftArgs a) {
    __shared__ double waves[DRAFT_WAVES], sums[(1u << 21) / DRAFT_CHUNK], parts[DRAFT_PER][DRAFT_WAVES];
    __shared__ uint32_t mins[DRAFT_WAVES];
    __shared__ bool last;
    const uint32_t s = blockIdx.x / a.groups, first = (blockIdx.x - s * a.groups) * a.per, tid = threadIdx.x, lane = tid % 64;
    const DraftSpan d = draft_span(a, s);
    const float draw = a.draws[s];
    uint32_t accepted = d.count;
    for (uint32_t i0 = 0; i0 < d.count; i0 += 64) {
        const uint32_t i = i0 + lane;
        bool fine = true;
        if (i < d.count) {
            const uint32_t token = (uint32_t)a.drafted[d.begin + i];
            fine = false;
            if (token < a.vocab) {
                const double p = probability(a.target.probs[((uint64_t)d.begin + s + i) * a.target.row_stride + token]);
                const double q = a.draft.probs ? probability(a.draft.probs[((uint64_t)d.begin + i) * a.draft.row_stride + token]) : 1.0;
                fine = (double)a.uniforms[d.begin + i] * q < p;
            }
        }
        const uint64_t refused = __ballot(!fine);
        if (refused) {
            accepted = i0 + (uint32_t)__ffsll((unsigned long long)refused) - 1;
            break;
        }
    }
    const bool rejected = accepted < d.count;
    const float *p = a.target.probs + ((uint64_t)d.begin + s + accepted) * a.target.row_stride;
    const float *q = rejected && a.draft.probs ? a.draft.probs + ((uint64_t)d.begin + accepted) * a.draft.row_stride : nullptr;
    const uint32_t one = rejected && !a.draft.probs ? (uint32_t)a.drafted[d.begin + accepted] : a.vocab; // q is 1 there
    // Four tokens' probabilities, zeros past the vocabulary, and what can be drawn of them.
    const auto load4 = [&](uint32_t v, bool less, f32x4 &x, f32x4 &y) {
        x = y = f32x4{0, 0, 0, 0};
        if (WIDE && v + 4 <= a.vocab) {
            x = *(const f32x4 *)(p + v);
            if (less && q) y = *(const f32x4 *)(q + v);
        } else
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
                if (v + i < a.vocab) {
                    x[i] = p[v + i];
                    if (less && q) y[i] = q[v + i];
                }
    };
    const auto left4 = [&](uint32_t v, bool less, f32x4 x, f32x4 y, double *left) {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const double from = probability(x[i]), take = less && v + i == one ? 1.0 : probability(y[i]);
            left[i] = from > take ? from - take : 0.0;
        }
    };
    // The wave's part of a chunk's sum. The next chunk is on its way while one is added.
    constexpr uint32_t QUADS = DRAFT_EACH / 4;
    f32x4 x[QUADS], y[QUADS];
    const auto load_chunk = [&](uint32_t c, bool less) {
#pragma unroll
        for (uint32_t j = 0; j < QUADS; j++) load4(c * DRAFT_CHUNK + (j * DRAFT_THREADS + tid) * 4, less, x[j], y[j]);
    };
    const auto add_chunk = [&](uint32_t c, bool less) { // of what was loaded
        double sum = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < QUADS; j++) {
            double left[4];
            left4(c * DRAFT_CHUNK + (j * DRAFT_THREADS + tid) * 4, less, x[j], y[j], left);
            sum += (left[0] + left[1]) + (left[2] + left[3]);
        }
        return sum;
    };
    const uint32_t end = min(first + a.per, a.chunks);
    load_chunk(first, true);
    for (uint32_t c = first; c < end; c++) {
        double sum = add_chunk(c, true);
        if (c + 1 < end) load_chunk(c + 1, true);
#pragma unroll
        for (uint32_t d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
        if (lane == 0) parts[c - first][tid / 64] = sum;
    }
    __syncthreads();
    const auto chunk_total = [&](uint32_t i) { return (parts[i][0] + parts[i][1]) + (parts[i][2] + parts[i][3]); };
    if (a.groups > 1) {
        if (tid < end - first)
            __hip_atomic_store((uint64_t *)(a.sums + (uint64_t)s * a.chunks + first + tid),
                               __builtin_bit_cast(uint64_t, chunk_total(tid)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (tid == 0) { // of the wave that has stored them all
            __builtin_amdgcn_s_waitcnt(DRAFT_STORED);
            last = atomicAdd(a.arrived + s, 1u) == a.groups - 1;
            if (last) __hip_atomic_store(a.arrived + s, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); // ready for the next call
        }
        __syncthreads();
        if (!last) return;
    }
    for (uint32_t c = tid; c < a.chunks; c += DRAFT_THREADS)
        sums[c] = a.groups > 1 ? __builtin_bit_cast(double, __hip_atomic_load((const uint64_t *)(a.sums + (uint64_t)s * a.chunks + c),
                                                                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
                               : chunk_total(c);
    __syncthreads();
    int32_t token = -1;
    for (uint32_t less = 2; less-- > 0;) { // from max(p - q, 0), and from p where that has nothing
        if (!less) {
            for (uint32_t c = 0; c < a.chunks; c++) {
                double all;
                load_chunk(c, false);
                block_scan(add_chunk(c, false), waves, all);
                if (tid == 0) sums[c] = all;
            }
            __syncthreads();
        }
        // The chunk: sums of two chunks a thread, 512 at most.
        constexpr uint32_t PER = (1u << 21) / DRAFT_CHUNK / DRAFT_THREADS;
        double part[PER], all, total;
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) part[i] = tid * PER + i < a.chunks ? sums[tid * PER + i] : 0.0;
        double sum = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) sum += part[i];
        block_scan(sum, waves, total);
        if (!(total > 0.0)) continue;
        const double border = draft_border(draw, total);
        const uint32_t c = block_pick(part, 0.0, border, waves, mins);
        // The sum of the chunks before it.
        double before = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < PER; i++)
            if (tid * PER + i < c) before += part[i];
        block_scan(before, waves, all);
        double left[DRAFT_EACH];
#pragma unroll
        for (uint32_t j = 0; j < QUADS; j++) load4(c * DRAFT_CHUNK + tid * DRAFT_EACH + 4 * j, less, x[j], y[j]);
#pragma unroll
        for (uint32_t j = 0; j < QUADS; j++) left4(c * DRAFT_CHUNK + tid * DRAFT_EACH + 4 * j, less, x[j], y[j], left + 4 * j);
        token = (int32_t)(c * DRAFT_CHUNK + block_pick(left, all, border, waves, mins));
        break;
    }
    draft_write(a, s, d, accepted, token);
}

// Candidate lists. Targets' entries in chunks of 1024, four a thread, each compared with
// every entry of the draft's list, which passes by in LDS: the time grows with the
// product of the two lengths, and with lists of up to some hundred entries is one
// chain of loads.
__global__ void __launch_bounds__(DRAFT_THREADS) k_drafts_lists(DraftArgs a) {
    __shared__ double waves[DRAFT_WAVES];
    __shared__ uint32_t mins[DRAFT_WAVES], refused;
    __shared__ uint2 tile[LIST_TILE]; // id and probability
    const uint32_t s = blockIdx.x, tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const DraftSpan d = draft_span(a, s);
    const float draw = a.draws[s];
    const auto kept = [](const rl_probs &x, uint64_t row) { return (uint32_t)min(min((uint64_t)x.kept[row], x.row_stride), (uint64_t)1 << 31); };
    // A token's probability in a list, by a wave. The first 64 entries are loaded before it is known how many there are.
    struct Head {
        uint32_t id, n;
        float p;
    };
    const auto head = [&](const rl_probs &x, uint64_t row) {
        const uint64_t at = row * x.row_stride + min((uint64_t)lane, x.row_stride - 1);
        return Head{x.ids[at], kept(x, row), x.probs[at]};
    };
    const auto of = [&](const rl_probs &x, uint64_t row, const Head &h, uint32_t token) {
        uint64_t where = __ballot(lane < h.n && h.id == token);
        if (where) return probability(__shfl(h.p, (int)__ffsll((unsigned long long)where) - 1));
        for (uint32_t j0 = 64; j0 < h.n; j0 += 64) {
            const uint32_t j = j0 + lane;
            where = __ballot(j < h.n && x.ids[row * x.row_stride + j] == token);
            if (where) return probability(x.probs[row * x.row_stride + j0 + (uint32_t)__ffsll((unsigned long long)where) - 1]);
        }
        return 0.0;
    };
    if (tid == 0) refused = d.count;
    __syncthreads();
    for (uint32_t i0 = wave; i0 < d.count; i0 += 2 * DRAFT_WAVES) { // two drafts at a time, up to the wave's first refused one
        Head target[2], draft[2] = {};
        uint32_t token[2];
        float u[2];
#pragma unroll
        for (uint32_t k = 0; k < 2; k++) {
            const uint64_t i = min(i0 + k * DRAFT_WAVES, d.count - 1);
            target[k] = head(a.target, d.begin + s + i);
            if (a.draft.probs) draft[k] = head(a.draft, d.begin + i);
            token[k] = (uint32_t)a.drafted[d.begin + i], u[k] = a.uniforms[d.begin + i];
        }
        bool fine = true;
#pragma unroll
        for (uint32_t k = 0; k < 2; k++) {
            const uint32_t i = i0 + k * DRAFT_WAVES;
            if (!fine || i >= d.count) break;
            const double p = of(a.target, (uint64_t)d.begin + s + i, target[k], token[k]);
            const double q = a.draft.probs ? of(a.draft, (uint64_t)d.begin + i, draft[k], token[k]) : 1.0;
            fine = (double)u[k] * q < p;
            if (!fine && lane == 0) atomicMin(&refused, i);
        }
        if (!fine) break;
    }
    __syncthreads();
    const uint32_t accepted = refused;
    const bool rejected = accepted < d.count;
    const uint64_t row = (uint64_t)d.begin + s + accepted, from = (uint64_t)d.begin + accepted;
    const float *probs = a.target.probs + row * a.target.row_stride;
    const uint32_t *ids = a.target.ids + row * a.target.row_stride;
    const uint32_t n = kept(a.target, row), others = rejected && a.draft.probs ? kept(a.draft, from) : 0;
    const uint32_t one = rejected && !a.draft.probs ? (uint32_t)a.drafted[d.begin + accepted] : 0;
    // The first entries are loaded before it is known how many there are.
    uint32_t id0[LIST_EACH];
    float p0[LIST_EACH];
#pragma unroll
    for (uint32_t i = 0; i < LIST_EACH; i++) {
        const uint64_t j = min((uint64_t)tid * LIST_EACH + i, a.target.row_stride - 1);
        id0[i] = ids[j], p0[i] = probs[j];
    }
    uint2 entry{};
    if (rejected && a.draft.probs) {
        const uint64_t at = from * a.draft.row_stride + min((uint64_t)tid, a.draft.row_stride - 1);
        entry = make_uint2(a.draft.ids[at], __float_as_uint(a.draft.probs[at]));
    }
    double left[LIST_EACH];
    // What can be drawn of the entries from `at` on, a run a thread.
    const auto fill = [&](uint32_t at, bool less) {
        uint32_t id[LIST_EACH];
        float take[LIST_EACH];
#pragma unroll
        for (uint32_t i = 0; i < LIST_EACH; i++) {
            const uint32_t j = at + tid * LIST_EACH + i;
            left[i] = j < n ? probability(at ? probs[j] : p0[i]) : 0.0;
            id[i] = j >= n ? 0 : at ? ids[j] : id0[i];
            take[i] = less && rejected && !a.draft.probs && id[i] == one ? 1.0f : 0.0f;
        }
        for (uint32_t j0 = 0; less && j0 < others; j0 += LIST_TILE) {
            const uint32_t m = min(others - j0, LIST_TILE);
            __syncthreads();
            for (uint32_t j = tid; j < m; j += DRAFT_THREADS) {
                uint2 x = entry;
                if (j0 + j != tid) {
                    const uint64_t at = from * a.draft.row_stride + j0 + j;
                    x = make_uint2(a.draft.ids[at], __float_as_uint(a.draft.probs[at]));
                }
                tile[j] = make_uint2(x.x, __float_as_uint(positive(__uint_as_float(x.y))));
            }
            __syncthreads();
#pragma unroll 8
            for (uint32_t j = 0; j < m; j++) {
                const uint2 x = tile[j];
#pragma unroll
                for (uint32_t i = 0; i < LIST_EACH; i++) take[i] = x.x == id[i] ? __uint_as_float(x.y) : take[i];
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < LIST_EACH; i++) left[i] = left[i] > (double)take[i] ? left[i] - (double)take[i] : 0.0;
    };
    int32_t token = -1;
    for (uint32_t less = 2; less-- > 0;) {
        double total = 0.0, all;
        for (uint32_t at = 0; at < n; at += LIST_CHUNK) {
            fill(at, less);
            double sum = 0.0;
#pragma unroll
            for (uint32_t i = 0; i < LIST_EACH; i++) sum += left[i];
            block_scan(sum, waves, all);
            total += all;
        }
        if (!(total > 0.0)) continue;
        const double border = draft_border(draw, total);
        double base = 0.0;
        uint32_t final = DRAFT_NONE; // the last that can be drawn so far
        for (uint32_t at = 0; at < n; at += LIST_CHUNK) {
            if (n > LIST_CHUNK) fill(at, less);
            double sum = 0.0;
#pragma unroll
            for (uint32_t i = 0; i < LIST_EACH; i++) sum += left[i];
            block_scan(sum, waves, all);
            if (all > 0.0) {
                const uint32_t i = block_pick(left, base, border, waves, mins);
                final = at + i;
                // base + all passes the border, or the next chunk's first does, or none does: then the last stands.
                if (base + all > border) break;
            }
            base += all;
        }
        token = (int32_t)ids[final];
        break;
    }
    draft_write(a, s, d, accepted, token);
}

}  // namespace rl
