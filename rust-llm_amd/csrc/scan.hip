// C ABI of the selective state space scan (include/rl_mixers.h); the kernels are in
// scan.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>
#include <string>

#include "mix_args.h"
#include "scan.h"

using namespace rl;

struct rl_scan {
    int device = 0;
    uint32_t max_rows = 0, max_seqs = 0, channels = 0, groups = 0, state = 0;
    uint32_t columns = 0; // workgroups of k_scan that a row takes
    uint64_t slots = 0;   // pieces' ends that there is room for
    float *a2 = nullptr;  // [channels][state], then skip, then bias
    float *ends = nullptr, *steps = nullptr;
    ~rl_scan() {
        (void)hipFree(a2);
        (void)hipFree(ends);
        (void)hipFree(steps);
    }
};

namespace {

// k_scan_steps or k_scan: the first has a quarter of the state values a lane, so a shorter way in and out, but forms each
// softplus and gate four times as often. It is taken for sequences of up to SCAN_FEW tokens, and up to SCAN_SHORT while
// the call's tokens are no more than SCAN_WORK waves together (each a token of 64 lanes). us, steps / other, 5120 channels
// of 16 bf16: one sequence of 8 tokens 5.8 / 7.4, of 32 15.8 / 17.1; 8 of 8 7.9 / 8.1; 16 of 4 7.2 / 8.6, of 8 10.6 / 10.0,
// of 16 18.1 / 14.5; 64 of 2 12.9 / 16.3, of 4 18.5 / 17.9, of 8 30.3 / 21.1; 256 of 2 41.0 / 50.2, of 4 65 / 53.
constexpr uint32_t SCAN_FEW = 3, SCAN_SHORT = 32, SCAN_WORK = 36864;
// Workgroups that pieces are made for, the fewest tokens of one, and the most pieces of a sequence: a piece's first state is
// made of the ends of all before it.
constexpr uint64_t SCAN_FILL = 1024, SCAN_MOST = 64;
constexpr uint32_t SCAN_LEAST = 16;

// Tokens of a piece, 0 for whole sequences. A token takes a wave 0.42 us (its loads, a softplus, 16 exponentials in a row,
// its output), and the device 0.25 us for each round of a wave a SIMD; pieces take each token twice, 1.8 times the work, and
// a second launch. us, whole / in pieces, 5120 channels of 16 bf16: one sequence of 33 tokens 19.1 / 18.6, 64 30.7 / 20.2,
// 128 52.3 / 22.4; 16 of 33 26.6 / 39.0, of 128 88.4 / 97.4 in pieces of 64 and 16.
// Both rules over nine kinds of channels (8 to 256 state values, bf16 and f32, 1024 to 5120 of them) and 1 to 64 sequences of 4
// to 2048 tokens, 176 calls: 3 % longer than with the best of the two kernels and pieces of 16 to 256, on average; at most 30 %
// (four of 1000 tokens, 1024 channels of 256, us, whole / in pieces 615 / 474; 2048 of 128 521 / 432).
uint32_t piece_size(uint64_t rows, uint64_t most, uint64_t seqs, uint32_t columns) {
    const uint64_t size = std::max({(uint64_t)SCAN_LEAST, (most + SCAN_MOST - 1) / SCAN_MOST, (rows * columns + SCAN_FILL - 1) / SCAN_FILL});
    const double simds = 1024.0, round = 0.25 * SCAN_WAVES * columns / simds;
    const double whole = most * std::max(0.42, round * seqs);
    const double pieces = 8.0 + std::max(1.8 * round * rows, 2 * 0.42 * size + 0.1 * most / size);
    return pieces < whole ? (uint32_t)size : 0;
}

}  // namespace

extern "C" {

int rl_scan_create(int device, uint32_t max_rows, uint32_t max_seqs, uint32_t channels, uint32_t groups,
                   uint32_t state_dim, const float *a, const float *skip, const float *dt_bias, rl_scan **out) {
    if (!out) return fail(RL_ERR_ARGUMENT, "out is null");
    *out = nullptr;
    if (!a) return fail(RL_ERR_ARGUMENT, "a is null");
    if (max_rows == 0 || max_seqs == 0 || channels == 0 || groups == 0 || channels % groups)
        return fail(RL_ERR_ARGUMENT, "max_rows and max_seqs must be positive, channels a multiple of groups");
    if (state_dim < 4 || state_dim > 256 || state_dim % 4)
        return fail(RL_ERR_ARGUMENT, "state_dim must be a multiple of 4, from 4 to 256");
    if (channels > 1u << 20 || max_rows > MAX_ROWS || max_seqs > MAX_ROWS)
        return fail(RL_ERR_CAPACITY, "more than 2^20 channels, or max_rows or max_seqs above 2^23");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select device " + std::to_string(device));
    auto *h = new (std::nothrow) rl_scan();
    if (!h) return fail(RL_ERR_CAPACITY, "out of host memory");
    h->device = device;
    h->max_rows = max_rows, h->max_seqs = max_seqs, h->channels = channels, h->groups = groups, h->state = state_dim;
    const uint32_t each = scan_each(state_dim), per = SCAN_THREADS / scan_lanes(state_dim, each);
    h->columns = groups * ((channels / groups + per - 1) / per);
    // Pieces of a call are no more than its rows have, nor than fill the device.
    h->slots = scan_slots(std::min<uint64_t>(max_rows / SCAN_LEAST, SCAN_FILL / h->columns + 1));
    const size_t size = (size_t)channels * state_dim, all = size + 2 * (size_t)channels;
    float *laid = new (std::nothrow) float[all];
    if (!laid) {
        delete h;
        return fail(RL_ERR_CAPACITY, "out of host memory");
    }
    for (size_t i = 0; i < size; i++) laid[i] = (float)(a[i] * 1.4426950408889634);
    for (uint32_t c = 0; c < channels; c++) {
        laid[size + c] = skip ? skip[c] : 0.0f;
        laid[size + channels + c] = dt_bias ? dt_bias[c] : 0.0f;
    }
    hipError_t e = hipMalloc(&h->a2, all * sizeof(float));
    if (e == hipSuccess) e = hipMemcpy(h->a2, laid, all * sizeof(float), hipMemcpyHostToDevice);
    delete[] laid;
    if (e == hipSuccess) e = hipMalloc(&h->ends, h->slots * h->columns * SCAN_THREADS * each * sizeof(float));
    if (e == hipSuccess) e = hipMalloc(&h->steps, h->slots * channels * sizeof(float));
    if (e != hipSuccess) {
        delete h;
        return hip_fail(e, "rl_scan_create");
    }
    *out = h;
    return RL_OK;
}

void rl_scan_destroy(rl_scan *scan) {
    if (!scan) return;
    DeviceGuard guard(scan->device);
    delete scan;
}

int rl_scan_rows(rl_scan *h, const rl_heads *x, const rl_heads *dt, const rl_heads *z, const rl_heads *b, const rl_heads *c,
                 const rl_heads *out, float *states, uint64_t state_slots, const int32_t *slots_in, const int32_t *slots_out,
                 const int32_t *starts, uint32_t rows, uint32_t seqs, int softplus, uint32_t most_rows, void *stream) {
    if (!h) return fail(RL_ERR_ARGUMENT, "scan is null");
    CHECK_HEADS(x, "x", false);
    CHECK_HEADS(dt, "dt", false);
    if (z) CHECK_HEADS(z, "z", false);
    CHECK_HEADS(b, "b", false);
    CHECK_HEADS(c, "c", false);
    CHECK_HEADS(out, "out", true);
    for (const rl_heads *t : {x, dt, z ? z : x, out})
        if (t->heads != 1 || t->dim != h->channels)
            return fail(RL_ERR_ARGUMENT, "x, dt, z and out must be one head of the handle's channels");
    for (const rl_heads *t : {b, c})
        if (t->heads != h->groups || t->dim != h->state)
            return fail(RL_ERR_ARGUMENT, "b and c must have the handle's groups and state_dim");
    for (const rl_heads *t : {dt, z ? z : x, b, c, out})
        if (t->dtype != x->dtype) return fail(RL_ERR_ARGUMENT, "the tensors of a call have one type");
    for (const rl_heads *t : {x, dt, z ? z : x})
        if (rows > 1 && t->data == out->data && t->row_stride != out->row_stride)
            return fail(RL_ERR_ARGUMENT, "in place needs the same strides");
    if (rows && (out->data == b->data || out->data == c->data)) return fail(RL_ERR_ARGUMENT, "out must not be b or c");
    if (!starts && seqs != rows) return fail(RL_ERR_ARGUMENT, "without starts there is one row a sequence");
    if (rows && !seqs) return fail(RL_ERR_ARGUMENT, "rows without a sequence");
    if (rows > h->max_rows) return fail(RL_ERR_CAPACITY, "rows above the handle's max_rows");
    if (seqs > h->max_seqs) return fail(RL_ERR_CAPACITY, "seqs above the handle's max_seqs");
    if (seqs == 0) return RL_OK;
    if (!slots_in || !slots_out) return fail(RL_ERR_ARGUMENT, "slots_in and slots_out must be device pointers");
    if (state_slots && !states) return fail(RL_ERR_ARGUMENT, "states must be a device pointer");
    if ((uintptr_t)states % 16) return fail(RL_ERR_ARGUMENT, "states must be aligned to 16 bytes");
    DeviceGuard guard(h->device);
    if (!guard.ok) return fail(RL_ERR_DEVICE, "cannot select the handle's device");
    ScanArgs a{};
    a.x = x->data, a.dt = dt->data, a.z = z ? z->data : nullptr, a.b = b->data, a.c = c->data, a.out = out->data;
    a.x_row = x->row_stride, a.dt_row = dt->row_stride, a.z_row = z ? z->row_stride : 0;
    a.b_row = b->row_stride, a.b_group = b->head_stride, a.c_row = c->row_stride, a.c_group = c->head_stride;
    a.out_row = out->row_stride;
    a.a2 = h->a2, a.skip = h->a2 + (size_t)h->channels * h->state, a.bias = a.skip + h->channels;
    a.states = states, a.state_slots = state_slots;
    a.slots_in = slots_in, a.slots_out = slots_out, a.starts = starts;
    a.rows = rows, a.seqs = seqs, a.channels = h->channels, a.groups = h->groups, a.state = h->state;
    a.per = h->channels / h->groups;
    a.softplus = softplus != 0;
    a.wide = wide(b) && wide(c);
    a.ends = h->ends, a.steps = h->steps;
    const uint32_t most = !starts ? 1 : most_rows ? std::min(most_rows, rows) : rows;
    const uint32_t lanes = scan_lanes(h->state, 4);
    const bool steps = most <= SCAN_FEW || (most <= SCAN_SHORT && (uint64_t)rows * h->channels * lanes / 64 <= SCAN_WORK);
    if (steps) {
        const uint32_t per = SCAN_THREADS / lanes;
        a.columns = (h->channels + per - 1) / per;
    } else {
        a.columns = h->columns;
        const uint32_t size = piece_size(rows, most, seqs, h->columns);
        if (size) a.pieces = row_blocks(size);
    }
    const uint64_t blocks = (uint64_t)(steps || !a.pieces.size ? seqs : row_block_count(rows, seqs, a.pieces.size)) * a.columns;
    if (blocks > MAX_ROWS) return fail(RL_ERR_CAPACITY, "too many sequences times channels in a call");
    with_type(x->dtype, [&](auto t) {
        if (steps) launch_scan_steps<decltype(t)>(a, static_cast<hipStream_t>(stream));
        else launch_scan<decltype(t)>(a, static_cast<hipStream_t>(stream));
    });
    return launched("rl_scan_rows launch");
}

}  // extern "C"
